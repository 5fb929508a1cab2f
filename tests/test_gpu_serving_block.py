"""A decoder block of a server: adapters beside the projections, positions of several axes, prompts, steps, and the choice of experts, as one run."""
import pytest
import torch

import nuvec_amd as nv
from nuvec_amd.layers import AdaptedLinear, Mlp, MoeMlp, PagedAttention, QuantizedLinear, SwitchGlu, SwitchProjection
from tests.paged_reference import attention
from tests.test_gpu_prompt_attention import expected as expected_prompt

pytestmark = pytest.mark.gpu
DIMS, HEADS, KEY_HEADS, DIM = 256, 4, 2, 64


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def linear(n, k, dtype):
    return QuantizedLinear.from_linear((torch.randn(n, k, device="cuda") * k ** -0.5).to(dtype))


def adapted(n, k, dtype, count=3, rank=8):
    put = lambda *s: torch.randn(s, device="cuda")
    return AdaptedLinear(linear(n, k, dtype), nv.Adapters((put(count, rank, k) * k ** -0.5).to(dtype), put(count, n, rank).to(dtype), put(count).abs()))


def block(dtype):
    weight = lambda: (1 + 0.1 * torch.randn(DIM, device="cuda")).to(dtype)
    axes = nv.rotary_axes((12, 10, 10), True)
    a = PagedAttention(adapted(HEADS * DIM, DIMS, dtype), linear(KEY_HEADS * DIM, DIMS, dtype), adapted(KEY_HEADS * DIM, DIMS, dtype), adapted(DIMS, HEADS * DIM, dtype),
                       HEADS, KEY_HEADS, nv.Rotation.new(DIM, 128, axes=axes), weight(), weight(), torch.randn(HEADS, device="cuda").to(dtype))
    experts = lambda n, k: (lambda q: SwitchProjection(q.weight, q.scales, q.biases, None, q.quant))(nv.quantize((torch.randn(16, n, k, device="cuda") * k ** -0.5).to(dtype)))
    m = MoeMlp(torch.randn(16, DIMS, device="cuda") * DIMS ** -0.5, SwitchGlu(experts(128, DIMS), experts(128, DIMS), experts(DIMS, 128)), 4, scores="sigmoid",
               bias=0.1 * torch.randn(16, device="cuda"), groups=4, top_groups=2, scale=1.5)
    return a, m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_prompts_then_steps(dtype):
    """The layers are their operators' composition, bit for bit; the attention of both kinds against 64 bits."""
    torch.manual_seed(1)
    a, m = block(dtype)
    caches = [nv.PagedCache.new(16, KEY_HEADS, 16, DIM, nv.Quant.affine(32, 8), dtype) for _ in range(2)]
    page_table = torch.randperm(16, device="cuda").to(torch.int32).reshape(2, 8)
    lengths = [0, 0]
    for rows in ([40, 23], [1, 1], [1, 30], [1, 1]):
        n, fresh, step = sum(rows), lengths == [0, 0], sum(rows) == 2
        x = torch.randn(n, DIMS, device="cuda").to(dtype)
        positions = ints([*range(lengths[0], lengths[0] + rows[0]), *range(lengths[1], lengths[1] + rows[1])])
        rotary = torch.randint(0, 128, (3, n), device="cuda").to(torch.int32)
        ids = (torch.arange(n, device="cuda") % 4 - 1).to(torch.int32)
        lengths = [i + j for i, j in zip(lengths, rows)]
        sequences, starts = (None, None) if step else (ints([0] * rows[0] + [1] * rows[1]), ints([0, rows[0], n]))
        got = a(x, caches[0], page_table, positions, ints(lengths), sequences, starts, None if step else max(rows), rotary, ids, fresh)
        heads = lambda y, h: y.view(n, h, DIM)
        base = [p(x) for p in (a.q_proj.linear, a.k_proj, a.v_proj.linear)]
        q = heads(nv.apply_adapters(base[0], x, a.q_proj.adapters, ids), HEADS)
        k, v = heads(base[1], KEY_HEADS), heads(nv.apply_adapters(base[2], x, a.v_proj.adapters, ids), KEY_HEADS)
        if fresh:
            q, k = (t[0].transpose(0, 1) for t in nv.head_norm_rope(q.transpose(0, 1)[None], k.transpose(0, 1)[None], a.q_norm, a.k_norm, a.rotation, rotary[:, None]))
            nv.append_paged(caches[1], k, v, page_table, positions, sequences)
            y = nv.prompt_attention(q, k, v, DIM ** -0.5, starts, sinks=a.sinks)
            want, bound = expected_prompt(q, k, v, DIM ** -0.5, rows, rows, a.sinks)
        else:
            q = nv.append_paged(caches[1], k, v, page_table, positions, sequences, a.rotation, a.k_norm, q, a.q_norm, rotary_positions=rotary)
            y = nv.paged_attention(q, caches[1], page_table, ints(lengths), DIM ** -0.5, starts, None if step else max(rows), a.sinks)
            want, bound = attention(q, caches[1], page_table, lengths, DIM ** -0.5, None if step else [0, rows[0], n], a.sinks)
        assert ((y.double() - want).abs() <= bound).all()
        y = y.flatten(1)
        assert torch.equal(got, nv.apply_adapters(a.o_proj.linear(y), y, a.o_proj.adapters, ids))
        for one, other in zip((caches[0].keys, caches[0].values), (caches[1].keys, caches[1].values)):
            assert torch.equal(one.weight.view(torch.int32), other.weight.view(torch.int32)) and torch.equal(one.scales, other.scales)
        out = m(got[None])
        top, scores = nv.moe_select(torch.nn.functional.linear(got.float(), m.gate), 4, "sigmoid", m.bias, 4, 2, scale=1.5)
        assert torch.equal(out, nv.weighted_sum(m.switch_mlp(got[None], top[None]), scores[None].to(dtype)))
    plain = a(x, caches[0], page_table, positions, ints(lengths), rotary_positions=rotary)
    y = nv.paged_attention(nv.append_paged(caches[1], heads(base[1], KEY_HEADS), heads(base[2], KEY_HEADS), page_table, positions, None, a.rotation, a.k_norm,
                                           heads(base[0], HEADS), a.q_norm, rotary_positions=rotary), caches[1], page_table, ints(lengths), DIM ** -0.5, sinks=a.sinks)
    assert torch.equal(plain, a.o_proj.linear(y.flatten(1)))  # (no ids: no adapters)


def test_fresh_sequences_and_those_read_back_agree():
    """The same prompts through their codes: as near as 8-bit codes are."""
    torch.manual_seed(2)
    a, _ = block(torch.float16)
    caches = [nv.PagedCache.new(16, KEY_HEADS, 16, DIM, nv.Quant.affine(32, 8), torch.float16) for _ in range(2)]
    page_table = torch.randperm(16, device="cuda").to(torch.int32).reshape(2, 8)
    x = torch.randn(60, DIMS, device="cuda").half()
    args = (ints([*range(40), *range(20)]), ints([40, 20]), ints([0] * 40 + [1] * 20), ints([0, 40, 60]), 40)
    one = a(x, caches[0], page_table, *args, fresh=True)
    other = a(x, caches[1], page_table, *args)
    assert (one.float() - other.float()).norm() < 0.02 * other.float().norm()
    with pytest.raises(nv.InvalidArgument, match="fresh sequences"):
        a(x[:2], caches[0], page_table, ints([0, 0]), ints([1, 1]), fresh=True)


@pytest.mark.parametrize("geglu", [False, True])
def test_mlp_with_adapters(geglu):
    torch.manual_seed(3)
    m = Mlp(adapted(512, DIMS, torch.bfloat16), linear(512, DIMS, torch.bfloat16), adapted(DIMS, 512, torch.bfloat16), geglu)
    plain = Mlp(m.gate_proj.linear, m.up_proj, m.down_proj.linear, geglu)
    for rows in (1, 5, 70):
        x = torch.randn(rows, DIMS, device="cuda").bfloat16()
        ids = (torch.arange(rows, device="cuda") % 4 - 1).to(torch.int32)
        gate = nv.apply_adapters(m.gate_proj.linear(x), x, m.gate_proj.adapters, ids)
        h = nv.glu(gate, m.up_proj(x), "geglu" if geglu else "swiglu")
        assert torch.equal(m(x, ids), nv.apply_adapters(m.down_proj.linear(h), h, m.down_proj.adapters, ids))
        assert torch.equal(m.fuse_gate_up()(x), plain(x)) and m.gate_up_proj is None


def test_captured_steps_follow_their_inputs():
    """One graph of a decode step, replayed over growing sequences, other positions and adapters, against the eager block on a second pool."""
    torch.manual_seed(4)
    a, m = block(torch.bfloat16)
    caches = [nv.PagedCache.new(8, KEY_HEADS, 16, DIM) for _ in range(2)]
    table = ints([[3, 1, 0, 2], [4, 7, 6, 5]])
    x, positions, lengths = torch.randn(2, DIMS, device="cuda", dtype=torch.bfloat16), ints([-1, -1]), ints([0, 0])
    rotary, ids = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), ints([-1, -1])
    run = lambda cache: m(a(x, cache, table, positions, lengths, rotary_positions=rotary, adapter_ids=ids)[None])
    run(caches[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(caches[0])
    for step in range(12):
        x.normal_()
        positions.copy_(ints([step, 2 * step]))
        lengths.copy_(ints([step + 1, 2 * step + 1]))
        rotary.copy_(torch.randint(0, 128, (3, 2)).to(torch.int32))
        ids.copy_(ints([step % 4 - 1, (step + 2) % 4 - 1]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, run(caches[1])), step
