"""The router against its definition in 64 bits.  Ids are equal; weights are off by the rounding of float32 scores: an
exponential of x (an argument rounded to |x| 2^-24, 2 units in the last place of the function), a sum of at most 512 terms in
pairs and over lanes (at most 21 roundings of 2^-24), a division and two products (2^-24 each): (|x| + 2 * 2 + 21 + 3) 2^-24 relative for
the score, as much for the sum it is divided by."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def moe():
    from liquidgemm_b200 import moe as _moe
    return _moe


def plain(logits, k, scoring="softmax", bias=None, n_group=1, topk_group=1, group_score="max", renormalize=True, scale=1.0):
    """Row by row on the host, from the definition."""
    l = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    T, E = l.shape
    size = E // n_group
    weights, ids = np.zeros((T, k)), np.full((T, k), -1, dtype=np.int32)
    for t in range(T):
        live = [e for e in range(E) if l[t, e] > -np.inf]
        s = np.zeros(E)
        if live and scoring == "softmax":
            top = l[t, live].max()
            s[live] = [1.0 if l[t, e] == top else np.exp(l[t, e] - top) for e in live]
            s /= s.sum()
        elif live:
            s[live] = 1.0 / (1.0 + np.exp(-l[t, live]))
        key = l[t] if b is None else s + b
        live = [e for e in live if key[e] > -np.inf]
        if n_group > 1:
            rank = []
            for g in range(n_group):
                mine = sorted((e for e in live if e // size == g), key=lambda e: (-key[e], e))
                value = key if b is not None or group_score == "max" else s
                rank.append(-np.inf if not mine else value[mine[0]] if group_score == "max" else sum(value[e] for e in mine[:2]))
            kept = sorted(range(n_group), key=lambda g: (-rank[g], g))[:topk_group]
            live = [e for e in live if e // size in kept]
        chosen = sorted(live, key=lambda e: (-key[e], e))[:k]
        w = s[chosen]
        if renormalize and w.sum() > 0:
            w = w / w.sum()
        weights[t, :len(chosen)], ids[t, :len(chosen)] = w * scale, chosen
    return torch.from_numpy(weights), torch.from_numpy(ids)


def check(moe, logits, k, **how):
    w, ids = moe.route(logits, k, **how)
    want_w, want_ids = plain(logits, k, **how)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), want_ids)
    finite = logits.double()[torch.isfinite(logits)]
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    tol = 2 * (spread + 28) * 2.0 ** -24
    assert torch.all((w.cpu().double() - want_w).abs() <= tol * want_w + 1e-37)


def _logits(T, E, dtype, seed, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(T, E, device="cuda", generator=g) * spread).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (33, 64, 6), (7, 33, 8), (130, 128, 8), (9, 257, 10), (5, 512, 32), (2, 32, 32)])
def test_softmax(moe, dtype, T, E, k):
    for renormalize in (True, False):
        check(moe, _logits(T, E, dtype, T + E), k, renormalize=renormalize)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k", [(1, 8, 1), (33, 60, 6), (65, 256, 8), (4, 512, 9)])
def test_sigmoid_and_bias(moe, dtype, T, E, k):
    l = _logits(T, E, dtype, 2 * T + E)
    bias = torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(E)) * 0.2
    check(moe, l, k, scoring="sigmoid", renormalize=False)
    check(moe, l, k, scoring="sigmoid", bias=bias, scale=2.5)
    check(moe, l, k, scoring="softmax", bias=bias * 0.01)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("E,G,kept,k", [(64, 8, 3, 6), (192, 8, 4, 8), (48, 48, 5, 5), (72, 2, 1, 7), (36, 12, 12, 9), (512, 64, 7, 12), (128, 2, 2, 4)])
def test_groups(moe, scoring, group_score, E, G, kept, k):
    l = _logits(41, E, torch.bfloat16, E + G)
    bias = torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(G)) * 0.1
    for b in (None, bias):
        check(moe, l, k, scoring=scoring, bias=b, n_group=G, topk_group=kept, group_score=group_score)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_go_to_the_lowest_index(moe, scoring):
    l = torch.zeros(6, 96, device="cuda")
    l[1, ::3] = 1.0
    l[2] = -0.0
    l[2, 5:70] = 0.0                  # equal numbers, other bits
    l[3, 40:] = 2.0
    l[4] = 60.0                       # sigmoid scores that round to one
    l[4, 64:] = 61.0
    for how in (dict(), dict(bias=torch.zeros(96, device="cuda")), dict(n_group=8, topk_group=2), dict(n_group=8, topk_group=2, group_score="top2")):
        w, ids = moe.route(l[:4], 8, scoring=scoring, **how)
        want = plain(l[:4], 8, scoring=scoring, **how)
        assert torch.equal(ids.cpu(), want[1])
    w, ids = moe.route(l, 3, scoring=scoring)
    assert ids[4].tolist() == [64, 65, 66] and ids[0].tolist() == [0, 1, 2] and ids[1].tolist() == [0, 3, 6]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", [dict(), dict(scoring="sigmoid"), dict(bias=True), dict(n_group=4, topk_group=2),
                                 dict(n_group=4, topk_group=2, group_score="top2", bias=True, scoring="sigmoid")])
def test_masked_experts(moe, dtype, how):
    """-inf, NaN, the type's lowest value and +inf among the logits; rows with fewer experts than slots, and with none."""
    E, k = 40, 6
    l = _logits(12, E, dtype, 5)
    l[0] = -float("inf")
    l[1] = float("nan")
    l[2, :37] = -float("inf")
    l[3, ::2] = float("nan")
    l[4, 3:] = torch.finfo(dtype).min
    l[5] = torch.finfo(dtype).min
    l[6, 7] = -float("inf")
    l[7, :30] = -float("inf")         # whole groups
    l[8, 1:] = -float("inf")
    how = dict(how)
    if how.pop("bias", False):
        how["bias"] = torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 0.1
    w, ids = moe.route(l, k, **how)
    want_w, want_ids = plain(l, k, **how)
    assert torch.equal(ids.cpu(), want_ids)
    assert ids[0].tolist() == [-1] * k and w[0].tolist() == [0.0] * k and ids[1].tolist() == [-1] * k
    # (logits at the type's lowest value: exponentials of minus that magnitude are zero, whatever the argument's rounding)
    assert torch.all((w.cpu().double() - want_w).abs() <= 2 * (40 + 28) * 2.0 ** -24 * want_w + 1e-37)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_keys_closer_than_float32_errors(moe, scoring):
    """Biases that bring every key of a token within a few units of float32's last place of one another: the choice is that of 64 bits."""
    T, E = 60, 64
    l = _logits(T, E, torch.float32, 8)
    s = torch.sigmoid(l.double()) if scoring == "sigmoid" else torch.softmax(l.double(), 1)
    for t in (0, 7, 31):
        bias = (0.75 - s[t]).float()                       # all keys of token t are 0.75 but for the bias' rounding
        for how in (dict(), dict(n_group=8, topk_group=3), dict(n_group=8, topk_group=3, group_score="top2")):
            check(moe, l, 6, scoring=scoring, bias=bias, **how)
    # groups whose sums of two scores are nearly equal, without a bias
    l[:, 32:] = l[:, :32] + torch.randn(T, 32, device="cuda", generator=_gen_like(9)) * 1e-6
    check(moe, l, 6, scoring=scoring, n_group=2, topk_group=1, group_score="top2")


def _gen_like(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_scores_far_below_one_keep_their_ratio(moe):
    """Sigmoids below the smallest float32: the weights' ratio is that of the exponentials, and without renormalising they vanish."""
    l = torch.full((3, 16), -150.0, device="cuda")
    l[0, 3], l[0, 9] = -95.0, -95.5
    l[1, 3], l[1, 9] = -120.0, -121.0
    l[2, 3], l[2, 9] = -70.0, -90.0
    check(moe, l, 2, scoring="sigmoid")
    check(moe, l, 2, scoring="sigmoid", renormalize=False)
    check(moe, l, 2, scoring="sigmoid", bias=torch.linspace(0, -1, 16, device="cuda"), renormalize=False)


def test_infinite_logits_share(moe):
    l = torch.zeros(1, 8, device="cuda")
    l[0, 2] = l[0, 5] = float("inf")
    w, ids = moe.route(l, 3)
    assert ids.tolist() == [[2, 5, 0]] and w.tolist() == [[0.5, 0.5, 0.0]]


def test_bias_takes_experts_out(moe):
    l = _logits(5, 16, torch.float32, 1)
    bias = torch.zeros(16, device="cuda")
    bias[::2] = -float("inf")
    bias[1] = float("nan")
    w, ids = moe.route(l, 8, bias=bias)
    assert torch.equal(ids.cpu(), plain(l, 8, bias=bias)[1]) and (ids[:, 7] == -1).all() and (ids != 1).all()


def test_strides_empty_and_types(moe):
    l = _logits(64, 48, torch.float32, 9)
    for view in (l.t(), l[::3, 5:41], l[:, 1:]):
        got, want = moe.route(view, 4), moe.route(view.contiguous().clone(), 4)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w, ids = moe.route(l[:0], 4)
    assert w.shape == ids.shape == (0, 4)
    for bad, match in ((dict(logits=l.double()), "bf16"), (dict(k=0), "topk"), (dict(k=33), "topk"), (dict(n_group=5), "n_group"),
                       (dict(n_group=4, topk_group=5), "topk_group"), (dict(bias=torch.zeros(47, device="cuda")), "bias"),
                       (dict(bias=torch.zeros(48, device="cuda").half()), "bias"), (dict(bias=torch.zeros(48)), "bias"),
                       (dict(logits=torch.zeros(2, 513, device="cuda")), "experts"), (dict(logits=l[0]), "2-D")):
        bad = dict(bad)
        x, k = bad.pop("logits", l), bad.pop("k", 4)
        with pytest.raises(RuntimeError, match=match):
            moe.route(x, k, **bad)


def test_many_rows_twice_and_captured(moe):
    l = _logits(5000, 160, torch.bfloat16, 4)
    how = dict(scoring="sigmoid", n_group=8, topk_group=3, group_score="top2", bias=torch.randn(160, device="cuda") * 0.1)
    a = moe.route(l, 6, **how)
    b = moe.route(l, 6, **how)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    rows = torch.randint(0, 5000, (40,))
    want = plain(l[rows], 6, **how)
    assert torch.equal(a[1][rows].cpu(), want[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    x = l.clone()
    with torch.cuda.stream(stream):
        moe.route(x, 6, **how)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = moe.route(x, 6, **how)
    torch.cuda.synchronize()
    x.copy_(l.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y[1], a[1].flip(0)) and torch.equal(y[0], a[0].flip(0))
