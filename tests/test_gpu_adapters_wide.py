"""Low-rank adapters (csrc/adapters.hip): blocks of 32 rows and of several times 256 columns, ranks that need most of the LDS, calls without adapters."""
import ctypes as C

import pytest
import torch

import nuvec_amd as nv
from nuvec_amd import _lib
from tests.test_gpu_adapters import TYPES, check, ints, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rank", [0, 16, 200])
def test_no_adapters_and_no_operands_of_theirs(dtype, rank):
    """The entry point with 0 adapters: y's bits, x, the weights and the workspace absent."""
    for rows, n in ((1, 64), (40, 300), (2100, 4000)):
        y = torch.randn(rows, n, device="cuda").to(dtype)
        ids, out = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.empty_like(y)
        d = _lib.AdaptersDescC({torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}[dtype], rank, rows, 4096, n, 0, 4096, n, n)
        lib, p = _lib.load(), lambda t: C.c_void_p(t.data_ptr())
        nv.ops._init(y)
        assert lib.nvq_apply_adapters_workspace_bytes(C.byref(d)) == 0
        _lib.check(lib.nvq_apply_adapters(C.byref(d), None, None, None, None, p(ids), p(y), p(out), None, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        assert torch.equal(out, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n,rank,count", [
    (2048, 96, 4096, 16, 3), (2049, 130, 4096 + 70, 12, 5), (2100, 640, 7001, 32, 4), (2048, 33, 6912, 100, 2), (2081, 64, 2500, 240, 3), (2100, 70, 7000, 256, 3),
    (4099, 257, 300, 17, 9), (2300, 64, 63, 1, 2)])
def test_blocks_of_thirty_two_rows(dtype, rows, k, n, rank, count):
    """One, two and three times 256 columns a block, the last ones ragged; adapters that change with every row and in runs, rows without one; in place of y."""
    y, x, adapters = make(rows, k, n, rank, count, dtype)
    g = torch.Generator().manual_seed(rows)
    for ids in (torch.randint(-1, count, (rows,), generator=g).to(torch.int32).cuda(),
                torch.repeat_interleave(ints([0, -1, count - 1, 0, 1]), ints([rows - 1100, 37, 900, 1, 162])).contiguous(),
                torch.full((rows,), -1, dtype=torch.int32, device="cuda")):
        want = check(y, x, adapters, ids)
        same = y.clone()
        assert nv.apply_adapters(same, x, adapters, ids, out=same) is same and torch.equal(same, want)
        assert torch.equal(want[ids < 0], y[ids < 0])


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_of_thirty_two_rows_in_views(dtype):
    """Rows of x, y and the result between others; x and weights that are not finite keep to their rows."""
    y, x, adapters = make(2100, 100, 4500, 20, 4, dtype)
    ids = (torch.arange(2100, device="cuda") // 3 % 5 - 1).to(torch.int32)
    want = check(y, x, adapters, ids)
    wide = torch.full((2100, 5000), 7.0, device="cuda", dtype=dtype)
    wide[:, 3:103], wide[:, 301:4801] = x, y
    nv.apply_adapters(wide[:, 301:4801], wide[:, 3:103], adapters, ids, out=wide[:, 301:4801])
    assert torch.equal(wide[:, 301:4801], want) and torch.equal(wide[:, 3:103], x) and (wide[:, 103:301] == 7).all() and (wide[:, 4801:] == 7).all()
    x[100], adapters.up[1, 17] = float("nan"), float("inf")
    got = nv.apply_adapters(y, x, adapters, ids)
    clean = torch.ones(2100, dtype=torch.bool, device="cuda")
    clean[100] = False
    assert torch.equal(got[clean & (ids != 1)], want[clean & (ids != 1)]) and not got[100].isfinite().any()
    other = [i for i in range(4500) if i != 17]
    assert torch.equal(got[clean & (ids == 1)][:, other], want[clean & (ids == 1)][:, other])


def test_captured_calls_of_many_rows_follow_their_ids():
    y, x, adapters = make(2060, 256, 4352, 16, 6, torch.bfloat16)
    ids = torch.zeros(2060, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(y)
    nv.apply_adapters(y, x, adapters, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nv.apply_adapters(y, x, adapters, ids, out=out)
    for step in range(4):
        new = torch.randint(-1, 6, (2060,)).to(torch.int32)
        ids.copy_(new.sort().values if step % 2 else new)
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check(y, x, adapters, ids))
