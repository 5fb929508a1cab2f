"""The choice of experts (csrc/select.hip): numbers of groups that are no powers of two, groups whose two best all but cancel, NaN and the last bits of weights."""
import pytest
import torch

import nuvec_amd as nv
from tests.test_gpu_moe_select import HALF, TYPES, check, expected, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,top", [(1000, 5, 2), (960, 3, 2), (720, 10, 3), (561, 17, 4), (1023, 33, 9), (1020, 60, 60), (1024, 32, 5), (1023, 3, 1)])
def test_more_than_sixteen_experts_of_a_lane(dtype, scores, e, groups, top):
    """Groups whose power of two of lanes is little more than half of the wavefront: up to 31 experts a lane."""
    x, bias = normal(19, e, dtype=dtype, seed=e), normal(e, seed=2, size=0.2)
    for k in (1, 16):
        check(x, k, scores, bias, groups, top, scale=1.5)
        check(x, k, scores, None, groups, top, normalize=False)
        check(x, k, scores, None, groups, top, 2)
    check(x, e // groups * top if e // groups * top < 64 else 64, scores, bias, groups, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1.0, 64.0, 300.0, 1e5])
def test_groups_whose_two_best_cancel(dtype, size):
    """Biases of either sign: a group's score is small beside its two values, which are what float32 rounds."""
    for e, groups, top in ((64, 32, 16), (128, 64, 9), (256, 8, 3)):
        each = e // groups
        x = normal(200, e, dtype=dtype, seed=e, size=1e-4 if dtype == torch.float32 else 1e-2)
        bias = torch.full((e,), -2 * size, device="cuda")
        bias[::each] = size * (1 + normal(groups, seed=3, size=0.1))
        bias[1::each] = -bias[::each]
        for scores in ("sigmoid", "softmax"):
            check(x, 4, scores, bias, groups, top)
            check(x, 4, scores, bias, groups, top, 1)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_nan_among_the_logits_reaches_every_weight_of_its_softmax(dtype):
    """Chosen or not; the experts are those of the others, and a sigmoid's weights too."""
    x, zeros = normal(6, 64, dtype=dtype), torch.zeros(64, device="cuda")
    x[1, 5], x[2, 60], x[3, ::2] = float("nan"), float("nan"), float("nan")
    x[4] = -float("inf")
    x[4, 7] = float("nan")
    for normalize in (True, False):
        for more in ({}, {"groups": 8, "top_groups": 2}, {"groups": 8, "top_groups": 8, "group_best": 2}):
            for bias in (None, zeros):
                experts, weights = nv.moe_select(x, 3, "softmax", bias, normalize=normalize, **more)
                assert weights[1:5].isnan().all() and weights[[0, 5]].isfinite().all()
                clean = expected(x[[0, 5]], 3, "softmax", bias, normalize=normalize, **more)[0]
                assert torch.equal(experts[[0, 5]].cpu().long(), clean)
            experts, weights = nv.moe_select(x[1:4], 3, "softmax", None, normalize=normalize)
            assert (experts[0] != 5).all() and (experts[1] != 60).all() and (experts[2] % 2 == 1).all()
            experts, weights = nv.moe_select(x[1:4], 3, "sigmoid", None, normalize=normalize, **more)
            assert weights.isfinite().all()


@pytest.mark.parametrize("e,k,groups,top", [(1024, 40, 1, 1), (256, 8, 8, 3), (60, 12, 1, 1), (17, 17, 1, 1)])
def test_float32_weights_of_a_softmax_are_rounded_once(e, k, groups, top):
    """Against 64 bits: half a step of float32, and what 64 bits lose of it (2^-50 for the sum of up to 1024 terms and the quotients)."""
    x = normal(300, e, seed=e, size=3.0)
    bias = normal(e, seed=1, size=0.1)
    for more in ({"normalize": False}, {"normalize": False, "scale": 2.5}, {"normalize": True}):
        for b in (None, bias):
            experts, weights = nv.moe_select(x, k, "softmax", b, groups, top, **more)
            want, w = expected(x, k, "softmax", b, groups, top, **more)
            assert torch.equal(experts.cpu().long(), want)
            assert ((weights.double().cpu() - w).abs() <= (HALF[torch.float32] + 2.0 ** -50) * w).all()


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_groups_by_two_without_a_bias_keep_the_order_of_the_logits(scores):
    """Scores that 64 bits do not tell apart, near 1 or 0: the larger logit first all the same."""
    g = torch.Generator().manual_seed(5)
    for base in (40.0, -900.0):
        x = base + torch.rand(20, 64, generator=g) * 8
        x[:, ::8] = 0.0 if scores == "sigmoid" else 50.0  # (one of each group: groups are as good as each other, or alike)
        x[:, 1::8] = 0.0 if scores == "sigmoid" else 50.0
        x = x.cuda()
        experts, _ = nv.moe_select(x, 40, scores, None, 8, 8, 2)
        want = sorted_experts(x, 40)
        assert torch.equal(experts.cpu().long(), want)


def sorted_experts(x, k):
    return torch.tensor([sorted(range(x.shape[1]), key=lambda i: (-row[i], i))[:k] for row in x.tolist()])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups", [2, 3, 4, 5, 6, 7, 8, 9, 13, 16, 17, 31, 32, 33, 47, 61, 64])
def test_every_number_of_groups_that_stay(dtype, groups):
    for each in (1, 2, 5):
        for top in sorted({1, 2, groups // 2, groups - 1, groups}):
            x, bias = normal(20, groups * each, dtype=dtype, seed=top, size=10.0), normal(groups * each, seed=each, size=0.3)
            k = min(64, top * each)
            for scores in ("softmax", "sigmoid"):
                check(x, k, scores, None, groups, top, normalize=False)
                check(x, k, scores, bias, groups, top)
                check(x, 1, scores, bias, groups, top, 1)
