"""Chosen experts whose scores lie below what float32 holds: the weights are those of 64-bit scores.  Tolerance and plain form are those
of test_gpu_moe_route.py (an argument's rounding is relative to the spread of the logits, which the tolerance counts)."""

import pytest
import torch

from test_gpu_moe_route import check

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module")
def moe():
    from liquidgemm_b200 import moe as _moe
    return _moe


def test_two_rows_by_hand(moe):
    want = torch.tensor([[0.7310586, 0.2689414]])
    w, ids = moe.route(torch.tensor([[-200.0, -201.0]], device="cuda"), 2, scoring="sigmoid")
    assert ids.tolist() == [[0, 1]] and torch.allclose(w.cpu(), want, rtol=1e-5, atol=0)
    w, ids = moe.route(torch.tensor([[0.0, -120.0, -121.0, -300.0]], device="cuda"), 2, bias=torch.tensor([-INF, 0, 0, 0], device="cuda"))
    assert set(ids[0].tolist()) <= {1, 2, 3}
    w, ids = moe.route(torch.tensor([[0.0, -120.0, -121.0, -300.0]], device="cuda"), 2,
                       bias=torch.tensor([-INF, 2, 1, 0], device="cuda"))
    assert ids.tolist() == [[1, 2]] and torch.allclose(w.cpu(), want, rtol=1e-5, atol=0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("low", [-60, -79, -81, -90, -100, -104, -120, -160, -173, -200, -400, -640])
def test_sigmoid(moe, dtype, low):
    """All of a row far below, by steps that 16-bit types hold; some beside ordinary scores."""
    l = torch.full((4, 70), 1.5 * low, device="cuda")
    l[0, [3, 40, 66]] = torch.tensor([low, low - 1.0, low - 2.0], device="cuda")
    l[1, [3, 40, 66]] = torch.tensor([low, low, 2.0], device="cuda")
    l[2, ::2] = low
    l[3, 5] = low
    l = l.to(dtype)
    bias = torch.zeros(70, device="cuda")
    bias[::7] = -1.0
    for how in (dict(), dict(renormalize=False, scale=2.0 ** 90), dict(bias=bias), dict(scale=2.5, n_group=7, topk_group=5)):
        check(moe, l, 3, scoring="sigmoid", **how)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("gap", [40, 79, 81, 86, 90, 95, 100, 103, 104, 120, 200, 500, 700])
def test_softmax_by_bias(moe, dtype, gap):
    """A bias that chooses experts far below the row's largest logit, beside it or without it."""
    l = torch.full((3, 100), -1.2 * gap, device="cuda")
    l[:, 0] = 0.0
    l[:, [7, 50, 90]] = torch.tensor([-gap, -gap - 1.0, -gap - 2.0], device="cuda")
    l[1, 50] = 1.0
    l[2, 7] = l[2, 90] = -gap - 3.0
    l = l.to(dtype)
    bias = torch.zeros(100, device="cuda")
    bias[[7, 50, 90]] = torch.tensor([6.0, 5.0, 4.0], device="cuda")
    for how in (dict(), dict(renormalize=False, scale=2.0 ** 90), dict(scale=2.5), dict(n_group=4, topk_group=4),
                dict(n_group=2, topk_group=2, group_score="top2")):
        check(moe, l, 3, bias=bias, **how)
    bias[0] = 8.0                     # the largest is chosen too
    check(moe, l, 4, bias=bias)
    check(moe, l, 4, bias=bias, renormalize=False, scale=2.0 ** 90)


@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_softmax_by_groups(moe, group_score):
    """Groups ranked by the bias leave the row's largest logit out; far logits chosen without a bias."""
    l = torch.full((2, 64), -300.0, device="cuda")
    l[:, 1] = 3.0
    l[0, 40:48] = torch.linspace(-100, -107, 8, device="cuda")
    l[1, 40:48] = torch.linspace(-600, -607, 8, device="cuda")
    bias = torch.zeros(64, device="cuda")
    bias[40:48] = torch.linspace(9, 8, 8, device="cuda")
    check(moe, l, 6, bias=bias, n_group=8, topk_group=1, group_score=group_score)
    for renormalize in (True, False):
        check(moe, l, 9, n_group=8, topk_group=3, group_score="max", renormalize=renormalize, scale=2.0 ** 90)


def test_scores_that_vanish_in_64_bits(moe):
    """Nothing chosen has a score: weights of zero, not a division by it."""
    l = torch.zeros(1, 8, device="cuda")
    l[0, 1:] = torch.finfo(torch.float32).min
    bias = torch.zeros(8, device="cuda")
    bias[0] = -INF
    w, ids = moe.route(l, 3, bias=bias)
    assert ids.tolist() == [[1, 2, 3]] and not w.any()
    w, ids = moe.route(torch.full((1, 8), -2000.0, device="cuda"), 3, scoring="sigmoid")
    assert ids.tolist() == [[0, 1, 2]] and not w.any()
    w, ids = moe.route(torch.tensor([[INF, -5.0, -6.0]], device="cuda"), 2, bias=torch.tensor([-INF, 1.0, 0.0], device="cuda"))
    assert ids.tolist() == [[1, 2]] and not w.any()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_sums_of_two_keys_beyond_float32(moe, scoring, sign):
    """Groups ranked by sums that only 64 bits hold: biases near float32's largest number."""
    l = torch.linspace(-2, 2, 4 * 12, device="cuda").view(4, 12).contiguous()
    apart = torch.linspace(1.0, 0.97, 4, device="cuda")      # no two keys of a group are close
    bias = torch.cat([sign * v * apart for v in (1.8e38, 3.0e38, 2.5e38)])
    for kept in (1, 2):
        check(moe, l, 3 * kept, scoring=scoring, bias=bias, n_group=3, topk_group=kept, group_score="top2")
    bias[4:8] = sign * INF            # groups that are infinite in 64 bits too
    check(moe, l, 3, scoring=scoring, bias=bias, n_group=3, topk_group=1 if sign > 0 else 2, group_score="top2")
