"""The products grouped by expert and the gated MLP against plain forms in 64 bits.

``experts_linear`` is defined bit for bit (exact sums, two rounded float32 products, one rounding): tolerance none.

``experts_mlp`` quantises hidden values that carry float32 rounding, counted in steps of 2^-24: g and u are off by 3 each (the
conversion of the sum, two products); exp(-g) by 3 |g| for its argument and 4 for the function (2 units in the last place); the
sum 1 + exp(-g) by no more than that and 1; its approximate reciprocal by 2 (one unit), the two products by 1 each:
3 + 3 + 4 + 1 + 2 + 1 + 1 = 15, so a relative (16 + 3 |g|) 2^-24 with the products of errors.  A code can differ by one only where its quotient lies that near to a half-integer, counting the
scale's error too; the tolerance adds up what such codes can change, exactly where they are, and behind it the float32
roundings of the weighted sum (topk + 6 of 2^-24) and half a step of the output type."""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS24 = 2.0 ** -24


@pytest.fixture(scope="module")
def moe():
    from liquidgemm_b200 import moe as _moe
    return _moe


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _stack(moe, E, N, K, w4, seed, gated=False, dtype=torch.bfloat16):
    """(layer, q [E, N, K] as float64, s1 [E, N]): rows in the order given, also where the layer stores them in turn."""
    from liquidgemm_b200 import quant
    w = (torch.randn(E, N, K, device="cuda", generator=_gen(seed)) * 0.05).to(dtype)
    layer = moe.quantize_experts(w, w4=w4, gated=gated)
    q = torch.empty(E, N, K, dtype=torch.float64, device="cuda")
    s1 = torch.empty(E, N, device="cuda")
    for e in range(E):
        one = quant.quantize_weight(w[e].float().cpu())          # the package's torch quantiser, on the host
        q[e] = quant.dequantize_i8(one).cuda().double()
        s1[e] = one.s1.cuda()
    return layer, q, s1


def _rows(shape, dtype, seed):
    x = torch.randn(*shape, device="cuda", generator=_gen(seed))
    x[..., 5] *= 15
    if x.shape[0] > 2:
        x[1] = 0.0
    return x.to(dtype)


def _quantise(x):
    """Codes and float32 scale of each row, by float32 divisions."""
    flat = x.reshape(-1, x.shape[-1]).float()
    scale = flat.abs().amax(1).clamp_min(1e-12) / torch.full((), 127.0, device=x.device)
    return torch.round(flat / scale[:, None]).clamp(-127, 127).double(), scale


def _linear(xq, scale, ids, q, s1, per_pair, dtype):
    T, k = ids.shape
    y = torch.zeros(T * k, q.shape[1], dtype=torch.float32, device=q.device)
    flat = ids.reshape(-1).long()
    for e in range(q.shape[0]):
        mine = (flat == e).nonzero().flatten()
        rows = mine if per_pair else mine // k
        sums = xq[rows] @ q[e].t()                               # whole numbers below 2^53: exact
        y[mine] = (sums.float() * scale[rows, None]) * s1[e]
    return y.to(dtype).view(T, k, -1)


def _ids(T, E, k, seed, how="random"):
    if how == "one":
        return torch.full((T, k), E - 1, dtype=torch.int32, device="cuda")
    ids = torch.randint(0, E, (T, k), device="cuda", generator=_gen(seed), dtype=torch.int32)
    if how == "holes":      # no expert: below, above, far off; a row with none
        ids[torch.rand(T, k, device="cuda", generator=_gen(seed + 1)) < 0.3] = -1
        ids[0] = -1
        ids[-1, 0] = E
        ids[-1, -1] = 2 ** 31 - 1
    return ids


LINEAR = [
    # T, E, k, N, K, ids
    (1, 4, 1, 128, 128, "random"), (1, 8, 2, 512, 1024, "random"), (3, 8, 2, 200, 256, "random"), (5, 3, 4, 65, 384, "random"),
    (33, 4, 2, 128, 512, "holes"), (70, 6, 3, 320, 256, "random"), (130, 4, 2, 136, 640, "holes"), (257, 2, 1, 256, 256, "one"),
    (513, 3, 4, 384, 256, "random"), (64, 512, 8, 128, 128, "random"), (700, 17, 5, 129, 256, "holes"), (9, 2, 32, 256, 128, "random"),
    (16, 5, 2, 1, 128, "random"), (40, 8, 2, 2048, 2048, "random"),
]


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("T,E,k,N,K,how", LINEAR)
def test_linear_bits(moe, w4, T, E, k, N, K, how):
    layer, q, s1 = _stack(moe, E, N, K, w4, T + N)
    ids = _ids(T, E, k, T + E, how)
    for dtype, per_pair in ((torch.bfloat16, False), (torch.float16, True), (torch.float32, False)):
        x = _rows((T, k, K) if per_pair else (T, K), dtype, T + K)
        y = moe.experts_linear(x, ids, layer)
        xq, scale = _quantise(x)
        assert y.dtype == dtype and torch.equal(y, _linear(xq, scale, ids, q, s1, per_pair, dtype))
    # rows that come in INT8
    xq, scale = _quantise(_rows((T, k, K), torch.float32, 3))
    y = moe.experts_linear(xq.to(torch.int8).view(T, k, K), ids.long(), layer, ascale=scale.view(T, k), out_dtype=torch.float32)
    assert torch.equal(y, _linear(xq, scale, ids, q, s1, True, torch.float32))


def _mlp(x, weights, ids, q13, s13, q2, s2):
    """(y, tolerance without the output's rounding), both [T, H] float64."""
    T, k = ids.shape
    inner, H = q13.shape[1] // 2, q2.shape[1]
    xq, scale = _quantise(x)
    y = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(y)
    flat = ids.reshape(-1).long()
    for e in range(q13.shape[0]):
        mine = (flat == e).nonzero().flatten()
        if not len(mine):
            continue
        rows = mine // k
        gu = (xq[rows] @ q13[e].t()) * scale[rows, None].double() * s13[e].double()
        g, u = gu[:, :inner], gu[:, inner:]
        h = g * torch.sigmoid(g) * u
        amax, at = h.abs().max(1, keepdim=True)
        hs = (amax.clamp_min(1e-12) / 127.0).float().double()
        quot = h / hs
        off = ((16 + 3 * g.abs()) + (16 + 3 * g.abs().gather(1, at)) + 3) * EPS24        # relative, of the quotient
        near = ((quot.abs() % 1.0) - 0.5).abs() <= quot.abs() * off + 1e-30
        code = torch.round(quot.float()).clamp(-127, 127).double()
        w = weights.reshape(-1)[mine, None].double()
        o = (code @ q2[e].t()) * hs * s2[e].double() * w
        y.index_add_(0, rows, o)
        flips = (near.double() @ q2[e].abs().t()) * hs * s2[e].double() * w.abs()
        scale_off = (16 + 3 * g.abs().gather(1, at) + 4) * EPS24
        tol.index_add_(0, rows, flips + o.abs() * (scale_off + (k + 6) * EPS24))
    return y, tol


def _check_mlp(moe, T, E, k, H, inner, w4, how, dtype, seed):
    w13, q13, s13 = _stack(moe, E, 2 * inner, H, w4, seed, gated=True)
    w2, q2, s2 = _stack(moe, E, H, inner, w4, seed + 1)
    x = _rows((T, H), dtype, seed + 2)
    ids = _ids(T, E, k, seed + 3, how)
    weights = torch.rand(T, k, device="cuda", generator=_gen(seed + 4))
    y = moe.experts_mlp(x, weights, ids, w13, w2)
    want, tol = _mlp(x, weights, ids, q13, s13, q2, s2)
    assert y.dtype == dtype and y.shape == (T, H)
    half_step = torch.finfo(dtype).eps / 2
    tol = tol + half_step * (want.abs() + tol) + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0.0)   # (fp16's subnormal step)
    off = (y.double() - want).abs() - tol
    assert torch.all(off <= 0), f"{int((off > 0).sum())} of {off.numel()} outputs off, by {float(off.max())} more than allowed"
    assert torch.isfinite(y).all()


MLP = [
    (1, 4, 1, 128, 128, "random"), (1, 8, 2, 512, 1024, "random"), (2, 8, 3, 256, 384, "random"), (17, 4, 2, 384, 128, "holes"),
    (33, 8, 2, 1024, 512, "random"), (100, 5, 4, 256, 256, "holes"), (300, 3, 2, 256, 640, "random"), (129, 2, 1, 384, 256, "one"),
    (64, 64, 6, 256, 128, "random"), (1000, 6, 3, 128, 256, "random"), (12, 512, 8, 128, 128, "random"),
]


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("T,E,k,H,inner,how", MLP)
def test_mlp(moe, w4, T, E, k, H, inner, how):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        _check_mlp(moe, T, E, k, H, inner, w4, how, dtype, T + E)


# rows of each expert; with 144 rows on average (45 with INT8 weights) the pair kernel runs, whose tiles are 192 (256) rows at most
COUNTS = [
    [1, 400, 0, 250], [193, 192, 191, 31], [255, 256, 257, 33], [385, 513, 0, 1], [577, 0, 0, 0], [161, 129, 97, 224],
    [0, 32, 64, 600], [96, 48, 16, 450],
]


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("counts", COUNTS)
def test_every_tile_width(moe, w4, counts):
    """Linear and MLP where the experts' rows end just behind, at and ahead of tile borders; channels an odd number of 128."""
    E, K, N = len(counts), 256, 384
    ids = torch.cat([torch.full((c,), e, dtype=torch.int32) for e, c in enumerate(counts)]).cuda()
    ids = ids[torch.randperm(len(ids), device="cuda", generator=_gen(len(ids)))][:, None].contiguous()
    layer, q, s1 = _stack(moe, E, N, K, w4, 5)
    x = _rows((len(ids), K), torch.bfloat16, 6)
    xq, scale = _quantise(x)
    assert torch.equal(moe.experts_linear(x, ids, layer), _linear(xq, scale, ids, q, s1, False, torch.bfloat16))
    w13, q13, s13 = _stack(moe, E, 2 * 128, K, w4, 7, gated=True)
    w2, q2, s2 = _stack(moe, E, K, 128, w4, 8)
    weights = torch.rand(len(ids), 1, device="cuda", generator=_gen(9))
    want, tol = _mlp(x, weights, ids, q13, s13, q2, s2)
    y = moe.experts_mlp(x, weights, ids, w13, w2)
    assert torch.all((y.double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30)


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("T,E,k,N,K", [(64, 64, 1, 256, 4096), (200, 100, 2, 128, 8192), (7, 16, 3, 1024, 2048)])
def test_fewer_experts_than_expected(moe, w4, T, E, k, N, K):
    """All tokens choose one expert of many, so that k is cut more often than the sizes alone would have it; and the even choice."""
    layer, q, s1 = _stack(moe, E, N, K, w4, T)
    x = _rows((T, K), torch.float16, 2)
    xq, scale = _quantise(x)
    for how in ("one", "random"):
        ids = _ids(T, E, k, T, how)
        assert torch.equal(moe.experts_linear(x, ids, layer), _linear(xq, scale, ids, q, s1, False, torch.float16))


# pair kernel, long k: fewer tiles than pairs, and a few tiles behind full rounds
@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("T,E,N,K", [(200, 1, 256, 8192), (150, 1, 384, 14336), (700, 2, 640, 4096), (900, 3, 6400, 4096), (577, 1, 9600, 6144)])
def test_long_k_and_partial_rounds(moe, w4, T, E, N, K):
    layer, q, s1 = _stack(moe, E, N, K, w4, T)
    ids = _ids(T, E, 1, T)
    x = _rows((T, K), torch.bfloat16, 2)
    xq, scale = _quantise(x)
    want = _linear(xq, scale, ids, q, s1, False, torch.bfloat16)
    for _ in range(5):
        assert torch.equal(moe.experts_linear(x, ids, layer), want)


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("T,E,H,inner", [(300, 1, 4096, 128), (300, 1, 128, 4096), (650, 2, 4096, 4096)])
def test_mlp_of_long_and_short_k(moe, w4, T, E, H, inner):
    _check_mlp(moe, T, E, 1, H, inner, w4, "random", torch.bfloat16, T)


@pytest.mark.parametrize("dtype,K", [(torch.bfloat16, 65536 + 128), (torch.float32, 32768 + 256), (torch.float16, 130944)])
def test_rows_too_long_for_registers(moe, dtype, K):
    layer, q, s1 = _stack(moe, 2, 65, K, True, 3)
    x = _rows((5, K), dtype, 4)
    for T in (1, 5):
        ids = _ids(T, 2, 2, 5)
        xq, scale = _quantise(x[:T])
        assert torch.equal(moe.experts_linear(x[:T], ids, layer), _linear(xq, scale, ids, q, s1, False, dtype))


def test_largest_sums(moe):
    """Every product at its largest magnitude: the int32 sums of the longest rows."""
    K = 130944
    layer = {"w": torch.full((1, 128, K), -128, dtype=torch.int8, device="cuda"), "s1": torch.ones(1, 128, device="cuda"), "E": 1, "N": 128,
             "K": K, "gated": False}
    x = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    y = moe.experts_linear(x, torch.zeros(3, 1, dtype=torch.int32, device="cuda"), layer, ascale=torch.ones(3, device="cuda"), out_dtype=torch.float32)
    assert torch.all(y == float(128 * 128 * K))


def test_groups_of_128(moe):
    from liquidgemm_b200 import quant
    w = (torch.randn(2, 192, 512, device="cuda", generator=_gen(1)) * 0.05).to(torch.bfloat16)
    x, ids = _rows((40, 512), torch.bfloat16, 2), _ids(40, 2, 2, 3)
    xq, scale = _quantise(x)
    ref = [quant.quantize_weight(w[e].float().cpu(), group_size=128) for e in range(2)]
    q = torch.stack([quant.dequantize_i8(r).cuda().double() for r in ref])
    s1 = torch.stack([r.s1.cuda() for r in ref])
    for w4 in (True, False):
        assert torch.equal(moe.experts_linear(x, ids, moe.quantize_experts(w, w4=w4, group_size=128)),
                           _linear(xq, scale, ids, q, s1, False, torch.bfloat16))


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("T", [3, 40, 700])
def test_infinite_rows_of_the_mlp_stay_with_their_tokens(moe, w4, T):
    w13, w2 = _layer(moe, 3, 256, 1024, w4, 31)
    x, ids, weights = _rows((T, 256), torch.float32, 5), _ids(T, 3, 2, 6), torch.rand(T, 2, device="cuda", generator=_gen(7))
    clean = moe.experts_mlp(x, weights, ids, w13, w2)
    bad = x.clone()
    bad[0, 3], bad[2, 0] = float("inf"), float("nan")
    got = moe.experts_mlp(bad, weights, ids, w13, w2)
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[[0, 2]] = False
    assert torch.equal(got[keep], clean[keep])
    bad[2, 0] = 0.0
    assert torch.equal(moe.experts_mlp(bad, weights, ids, w13, w2)[2], got[2])      # a NaN counts as zero


def test_quantised_stacks_are_those_of_the_dense_linear(moe):
    from liquidgemm_b200 import ops
    w = (torch.randn(3, 200, 256, device="cuda", generator=_gen(1)) * 0.05).to(torch.bfloat16)
    four, eight = moe.quantize_experts(w), moe.quantize_experts(w, w4=False)
    for e in range(3):
        qw, blob = ops.quantize_weight_cuda(w[e], 64, want_codes=True, want_blob=True)
        assert torch.equal(four["w"][e], blob) and torch.equal(four["s1"][e], qw.s1) and torch.equal(eight["s1"][e], qw.s1)
        assert torch.equal(eight["w"][e], torch.ops.liquidgemm.dequant_weight(qw.qweight_u4, qw.s_u8, qw.offset_a, 200, 256, 64))
    turned = torch.empty_like(w)
    turned[:, 0::2], turned[:, 1::2] = w[:, :100], w[:, 100:]
    for source in (w, w.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(moe.quantize_experts(source, gated=True)["w"], moe.quantize_experts(turned)["w"])
    assert torch.equal(moe.quantize_experts(w, group_size=128)["s1"], four["s1"])


def test_linear_equals_the_dense_linear(moe):
    """One expert for every token: the dense operator's outputs, bit for bit."""
    from liquidgemm_b200 import ops
    w = (torch.randn(2, 256, 512, device="cuda", generator=_gen(2)) * 0.05).to(torch.bfloat16)
    layer = moe.quantize_experts(w)
    qw, blob = ops.quantize_weight_cuda(w[1], 64, want_codes=False, want_blob=True)
    dense = {"s1": qw.s1, "s_u8": qw.s_u8, "offset_a": qw.offset_a, "N": 256, "K": 512, "rs": blob.reshape(-1)}
    for T in (1, 40, 300):
        x = _rows((T, 512), torch.bfloat16, T)
        y = moe.experts_linear(x, torch.ones(T, 1, dtype=torch.int32, device="cuda"), layer)
        assert torch.equal(y[:, 0], ops.w4a8_linear(x, dense))


def test_strides_and_offsets(moe):
    layer, q, s1 = _stack(moe, 4, 128, 256, True, 7)
    wide = _rows((50, 300), torch.bfloat16, 8)
    ids = _ids(50, 4, 4, 9)
    for x, i in ((wide[:, 3:259], ids), (wide[:, 1:257].t().contiguous().t(), ids[:, ::2]), (wide[5:45, 40:296], ids[5:45]),
                 (wide.reshape(-1)[1:1 + 256 * 50].view(50, 256), ids)):
        assert torch.equal(moe.experts_linear(x, i, layer), moe.experts_linear(x.clone().contiguous(), i.clone(), layer))


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
def test_empty_batches_and_no_experts_at_all(moe, w4):
    layer, _, _ = _stack(moe, 3, 256, 256, w4, 1)
    w13, _, _ = _stack(moe, 3, 256, 256, w4, 1, gated=True)
    w2, _, _ = _stack(moe, 3, 256, 128, w4, 1)
    x = _rows((70, 256), torch.bfloat16, 1)
    assert moe.experts_linear(x[:0], torch.zeros(0, 2, dtype=torch.int32, device="cuda"), layer).shape == (0, 2, 256)
    assert moe.experts_mlp(x[:0], torch.zeros(0, 2, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), w13, w2).shape == (0, 256)
    for T in (1, 70):
        none = torch.full((T, 2), -1, dtype=torch.int64, device="cuda")
        junk = torch.full((T, 2), float("nan"), device="cuda")
        torch.empty(1 << 22, device="cuda").fill_(float("nan"))      # what the allocator hands out next is not zero
        assert not moe.experts_linear(x[:T], none, layer).any()
        assert not moe.experts_mlp(x[:T], junk, none, w13, w2).any()


def test_infinite_rows_stay_with_their_tokens(moe):
    """A row with an infinity or a NaN gives what the dense quantiser makes of it, and nothing of it reaches other rows."""
    layer, _, _ = _stack(moe, 3, 128, 256, True, 1)
    x = _rows((40, 256), torch.float32, 5)
    ids = _ids(40, 3, 2, 6)
    clean = moe.experts_linear(x, ids, layer)
    bad = x.clone()
    bad[7, 3], bad[20, 0] = float("inf"), float("nan")
    got = moe.experts_linear(bad, ids, layer)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[7, 20]] = False
    assert torch.equal(got[keep], clean[keep])


def _layer(moe, E, H, inner, w4, seed):
    return _stack(moe, E, 2 * inner, H, w4, seed, gated=True)[0], _stack(moe, E, H, inner, w4, seed + 1)[0]


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("T", [1, 30, 600])
def test_layer_as_used_captured_and_replayed(moe, w4, T):
    """Router and experts together, eager and as a graph replayed on new inputs that choose other experts."""
    E, k, H, inner = 12, 3, 384, 256
    w13, w2 = _layer(moe, E, H, inner, w4, 11)
    gate = torch.randn(E, H, device="cuda", generator=_gen(1)) * 0.1

    def layer(x):
        weights, ids = moe.route((x.float() @ gate.t()), k, scoring="sigmoid", bias=torch.zeros(E, device="cuda"))
        return moe.experts_mlp(x, weights, ids, w13, w2), ids

    batches = [_rows((T, H), torch.bfloat16, s) for s in (1, 2, 3)]
    want = [layer(x) for x in batches]
    again = [layer(x) for x in batches]
    for (y, i), (z, j) in zip(want, again):
        assert torch.equal(y, z) and torch.equal(i, j)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    x = batches[0].clone()
    with torch.cuda.stream(stream):
        layer(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y, _ = layer(x)
    torch.cuda.synchronize()
    for _ in range(2):
        for b, (z, _) in zip(batches, want):
            x.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, z)


def test_two_streams_and_two_graphs_at_once(moe):
    w13, w2 = _layer(moe, 8, 512, 512, True, 21)
    work = []
    for s in range(2):
        x = _rows((150, 512), torch.bfloat16, 30 + s)
        ids, weights = _ids(150, 8, 2, 40 + s), torch.rand(150, 2, device="cuda", generator=_gen(50 + s))
        work.append((x, weights, ids, moe.experts_mlp(x, weights, ids, w13, w2)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    outs = [[] for _ in work]
    for _ in range(20):
        for i, (st, (x, weights, ids, _)) in enumerate(zip(streams, work)):
            with torch.cuda.stream(st):
                outs[i].append(moe.experts_mlp(x, weights, ids, w13, w2))
    torch.cuda.synchronize()
    for got, (_, _, _, want) in zip(outs, work):
        assert all(torch.equal(y, want) for y in got)
    graphs, ys = [], []
    for st, (x, weights, ids, _) in zip(streams, work):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ys.append(moe.experts_mlp(x, weights, ids, w13, w2))
        graphs.append(g)
    for _ in range(20):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for y, (_, _, _, want) in zip(ys, work):
        assert torch.equal(y, want)
    from liquidgemm_b200 import ops
    ops.poll_status()


def test_inputs_written_just_before(moe):
    """Rows, ids and weights are the output of the kernel directly before the call."""
    layer, q, s1 = _stack(moe, 4, 256, 256, True, 3)
    src = [_rows((90, 256), torch.bfloat16, s) for s in range(6)]
    idx = [_ids(90, 4, 2, s) for s in range(6)]
    x, ids = torch.empty_like(src[0]), torch.empty_like(idx[0])
    got = []
    for s, i in zip(src, idx):
        x.copy_(s)
        ids.copy_(i)
        got.append(moe.experts_linear(x, ids, layer))
    for s, i, y in zip(src, idx, got):
        xq, scale = _quantise(s)
        assert torch.equal(y, _linear(xq, scale, i, q, s1, False, torch.bfloat16))


def test_refusals_on_the_device(moe):
    layer, _, _ = _stack(moe, 4, 128, 256, True, 3)
    w13, w2 = _layer(moe, 4, 256, 128, True, 4)
    x, ids, wts = _rows((5, 256), torch.bfloat16, 1), _ids(5, 4, 2, 1), torch.rand(5, 2, device="cuda")
    for call, match in (
            (lambda: moe.experts_linear(x.double(), ids, layer, out_dtype=torch.float32), "bfloat16"),
            (lambda: moe.experts_linear(x[:, :128], ids, layer), "x must"),
            (lambda: moe.experts_linear(x[:4], ids, layer), "same tokens"),
            (lambda: moe.experts_linear(x.view(5, 1, 256), ids, layer), "same tokens"),
            (lambda: moe.experts_linear(x, ids.float(), layer), "ids"),
            (lambda: moe.experts_linear(x, ids[0], layer), "ids"),
            (lambda: moe.experts_linear(x, ids.cpu(), layer), "ids"),
            (lambda: moe.experts_linear(x, ids, layer, ascale=torch.ones(5, device="cuda")), "int8"),
            (lambda: moe.experts_linear(x.to(torch.int8), ids, layer), "ascale"),
            (lambda: moe.experts_linear(x.to(torch.int8), ids, layer, ascale=torch.ones(4, device="cuda")), "ascale"),
            (lambda: moe.experts_linear(x, ids, dict(layer, N=256)), "float32"),
            (lambda: moe.experts_linear(x, ids, dict(layer, w=layer["w"][:3])), "tile blobs"),
            (lambda: moe.experts_mlp(x, wts[:, :1], ids, w13, w2), "weights"),
            (lambda: moe.experts_mlp(x, wts.half(), ids, w13, w2), "weights"),
            (lambda: moe.experts_mlp(x, wts, ids, w13, dict(w2, s1=w2["s1"][:2], w=w2["w"][:2])), "same experts"),
            (lambda: moe.quantize_experts(torch.zeros(2, 128, 100, device="cuda")), "K % 128"),
            (lambda: moe.quantize_experts(torch.zeros(2, 127, 128, device="cuda"), gated=True), "up rows"),
            (lambda: moe.quantize_experts(torch.zeros(2, 128, 128, device="cuda"), group_size=32), "group_size")):
        with pytest.raises(RuntimeError, match=match):
            call()
