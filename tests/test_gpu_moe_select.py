"""The choice of experts (csrc/select.hip) against 64 bits: the same experts, and their weights."""
import pytest
import torch

import nuvec_amd as nv

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half a step of the smallest values


def expected(logits, k, scores="softmax", bias=None, groups=1, top_groups=None, group_best=None, normalize=True, scale=1.0):
    """Row by row in 64 bits, from the definition."""
    x = logits.double().cpu().reshape(-1, logits.shape[-1])
    e = x.shape[1]
    top_groups = groups if top_groups is None else top_groups
    group_best = (1 if bias is None else 2) if group_best is None else group_best
    p = torch.sigmoid(x) if scores == "sigmoid" else torch.softmax(x, -1)
    p = torch.where((x == -float("inf")).all(-1, keepdim=True), 0.0, p) if scores == "softmax" else p
    c = p if bias is None else p + bias.double().cpu()
    exact = bias is None and (groups == 1 or group_best == 1)  # (then the logits' order)
    key = (x if exact else c).nan_to_num(nan=-float("inf"), posinf=float("inf"), neginf=-1e308)
    chosen = []
    for r in range(len(x)):
        order = lambda values, of: sorted(of, key=lambda i: (-values[i], i))
        row = key[r].tolist()
        each = e // groups
        best = [sum(sorted(row[g * each:(g + 1) * each], reverse=True)[:group_best]) for g in range(groups)]
        stay = order(best, range(groups))[:top_groups]
        chosen.append(order(row, [i for i in range(e) if i // each in stay])[:k])
    chosen = torch.tensor(chosen).reshape(-1, k)
    w = p.gather(-1, chosen)
    if normalize:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return chosen.reshape(logits.shape[:-1] + (k,)), (w * scale).reshape(logits.shape[:-1] + (k,))


def check(logits, k, *args, **more):
    experts, weights = nv.moe_select(logits, k, *args, **more)
    want, w = expected(logits, k, *args, **more)
    assert experts.dtype == torch.int32 and weights.dtype == logits.dtype and experts.shape == want.shape == weights.shape
    assert torch.equal(experts.cpu().long(), want)
    # Float32: exp, the quotients and the sums are 64 bits wide; then float32's rounding and the scale's.  16 bits: an exponential (2^-23, and the product with
    # log2 e put back), a reciprocal twice (2^-23 each), a tree of six sums, three products and the rounding of the scale (2^-24 each): 8 steps of 2^-23 at
    # most, 2^-20; then the type's rounding.
    got, t = weights.double().cpu(), logits.dtype
    both = got.isnan() & w.isnan()
    assert (both | ((got - w).abs() <= (HALF[t] + (2.0 ** -23 if t == torch.float32 else 2.0 ** -20)) * w.abs() + TINY[t])).all()
    return experts, weights


def normal(*shape, dtype=torch.float32, seed=0, size=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(shape, generator=g, device="cuda")).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,k", [(1, 1), (2, 2), (8, 2), (60, 4), (64, 64), (65, 8), (128, 1), (130, 9), (256, 8), (384, 8), (511, 10), (1000, 33), (1024, 64)])
def test_sizes(dtype, scores, e, k):
    """(16-bit logits have many ties.)"""
    x = normal(37, e, dtype=dtype, seed=e)
    check(x, k, scores)
    check(x, k, scores, normal(e, seed=1, size=0.1), normalize=False, scale=2.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,k,groups,top", [(256, 8, 8, 4), (64, 6, 8, 3), (160, 6, 8, 3), (8, 2, 4, 2), (64, 4, 64, 9), (16, 5, 1, 1), (100, 20, 5, 1), (512, 8, 16, 4), (18, 6, 3, 3)])
def test_groups(dtype, scores, e, k, groups, top):
    x, bias = normal(33, e, dtype=dtype, seed=e), normal(e, seed=2, size=0.2)
    check(x, k, scores, bias, groups, top, scale=1.5)
    check(x, k, scores, None, groups, top, normalize=False)
    check(x, k, scores, bias, groups, top, 1)
    check(x, k, scores, None, groups, top, 2)
    check(x, k, scores, bias, groups)


def test_ties_go_to_the_lowest_index():
    for e, groups, top in ((8, 1, 1), (64, 8, 2), (256, 8, 4), (300, 5, 2)):
        x = torch.zeros(3, e, device="cuda")
        x[1, e // 2:] = 1.0
        x[2, 1::2] = 1.0
        for bias in (None, torch.zeros(e, device="cuda")):
            experts, _ = check(x, 4, "sigmoid", bias, groups, top)
        assert experts[0].tolist() == [0, 1, 2, 3]
    x = torch.tensor([[0.0, -0.0, 0.0, -0.0]], device="cuda")
    assert check(x, 3, "softmax", torch.zeros(4, device="cuda"))[0].tolist() == [[0, 1, 2]]
    assert check(x, 3)[0].tolist() == [[0, 1, 2]]


def test_neighbours_that_float32_does_not_tell_apart():
    """Scores with a bias whose sums differ by less than a float32 step: the larger one first."""
    x = torch.zeros(1, 8, device="cuda")
    bias = torch.zeros(8, device="cuda")
    x[0, 5] = 1e-7  # sigmoid: 0.5 + 2.5e-8, half a step of float32
    assert check(x, 2, "sigmoid", bias)[0].tolist() == [[5, 0]]
    x = torch.full((1, 8), 30.0, device="cuda")  # sigmoid: 1 - 9e-14
    x[0, 3] = 31.0
    assert check(x, 1, "sigmoid", bias)[0].tolist() == [[3]]
    x = torch.full((1, 8), 60.0, device="cuda")  # (beyond 64 bits' reach the logits themselves tell)
    x[0, 3] = 61.0
    assert nv.moe_select(x, 1, "sigmoid")[0].tolist() == [[3]]


@pytest.mark.parametrize("e", [60, 128, 256, 512])
def test_logits_a_few_steps_apart(e):
    """Float32 logits that differ in their last bits alone, in any order, and pairs of equal ones among them."""
    order = torch.randperm(e, generator=torch.Generator().manual_seed(e)).to("cuda").float()
    for step in (2.0 ** -23, 2.0 ** -20, 2.0 ** -16):
        x = torch.stack([1 + order * step, -1 - order * step, 1 + (order // 2) * step])
        for k in (8, 33, min(e, 64)):
            check(x, k)
            check(x, k, "sigmoid")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_biases_that_all_but_meet(dtype, scores):
    """Sums with the bias a part of a float32 step to many steps apart: among those chosen, behind the last of them, between groups."""
    order = torch.randperm(256, generator=torch.Generator().manual_seed(7)).to("cuda").float()
    x = normal(9, 256, dtype=dtype) * 0
    for step in (2.0 ** -24, 2.0 ** -21, 2.0 ** -18, 2.0 ** -15):
        bias = 0.25 + order * step
        for k, groups, top in ((8, 1, 1), (64, 1, 1), (8, 8, 4), (8, 64, 9), (64, 4, 1)):
            check(x, k, scores, bias, groups, top)
            check(x, k, scores, bias, groups, top, 1)
            check(normal(9, 256, dtype=dtype, seed=3, size=1e-6), k, scores, bias, groups, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_biases_without_end(dtype):
    """A bias of -inf masks an expert, one of inf brings it to the front."""
    x, bias = normal(5, 64, dtype=dtype), normal(64, size=0.1)
    bias[::3] = float("-inf")
    check(x, 8, "sigmoid", bias)
    check(x, 8, "softmax", bias, 4, 2)
    bias[50] = float("inf")
    experts, _ = nv.moe_select(x, 8, "sigmoid", bias)
    assert (experts[:, 0] == 50).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_scores_far_from_one(dtype, scores):
    """Weights of scores near and below the smallest normal number."""
    x = normal(6, 32, dtype=dtype, size=2.0) - 88
    x[3:, 7] = 40.0
    for normalize in (True, False):
        check(x, 6, scores, normalize=normalize)
        check(x, 6, scores, torch.zeros(32, device="cuda"), normalize=normalize)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_and_missing_logits(dtype):
    """-inf: experts that are masked; rows of nothing else; NaN below everything; the lowest finite value."""
    inf, low = float("inf"), torch.finfo(dtype).min
    x = normal(8, 16, dtype=dtype)
    x[0, 3:] = -inf
    x[1] = -inf
    x[2, ::2] = low
    x[3] = low
    x[4, 5] = inf
    for scores in ("softmax", "sigmoid"):
        check(x[:4], 5, scores)
        check(x[:4], 5, scores, normal(16, size=0.1), 4, 3)
    assert nv.moe_select(x[4:5], 1, "sigmoid")[0].item() == 5
    assert (nv.moe_select(x[1:2], 4)[1] == 0).all() and (nv.moe_select(x[1:2], 4, normalize=False)[1] == 0).all()
    x[5, ::2] = float("nan")
    for scores in ("softmax", "sigmoid"):
        for more in ({}, {"groups": 4, "top_groups": 2}):
            experts, weights = nv.moe_select(x[5:6], 3, scores, **more)
            assert all(i % 2 == 1 for i in experts[0].tolist())
    x[6] = float("nan")
    for bias in (None, torch.zeros(16, device="cuda")):
        experts, weights = nv.moe_select(x[6:7], 5, "sigmoid", bias, 4, 2)
        assert experts[0].tolist() == [0, 1, 2, 3, 4] and weights.isnan().all()


def test_shapes_strides_and_nothing():
    x = normal(2, 3, 40, dtype=torch.bfloat16)
    want = check(x, 4)
    assert want[0].shape == (2, 3, 4)
    wide = torch.zeros(2, 3, 90, device="cuda", dtype=torch.bfloat16)
    wide[..., 11:51] = x
    assert torch.equal(nv.moe_select(wide[..., 11:51], 4)[0], want[0])
    assert torch.equal(nv.moe_select(x.transpose(0, 1), 4)[1], want[1].transpose(0, 1))
    one = nv.moe_select(x[0, 0], 4)
    assert one[0].shape == (4,) and torch.equal(one[0], want[0][0, 0])
    experts, weights = nv.moe_select(x[:0], 4)
    assert experts.shape == (0, 3, 4) == weights.shape
    odd = torch.zeros(2 * 3 * 40 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 3, 40)  # (rows at odd addresses)
    odd.copy_(x)
    assert torch.equal(nv.moe_select(odd, 4)[0], want[0])


def test_captured_calls_follow_their_logits():
    x, bias = normal(70, 256, dtype=torch.bfloat16), normal(256, size=0.1)
    run = lambda: nv.moe_select(x, 8, "sigmoid", bias, 8, 4)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        experts, weights = run()
    for _ in range(4):
        x.normal_()
        bias.normal_(0, 0.1)
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert torch.equal(experts, want[0]) and torch.equal(weights, want[1])
        check(x, 8, "sigmoid", bias, 8, 4)
