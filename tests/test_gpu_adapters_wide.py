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
