"""Norms around a block on the device, against the formula in 64 bits.

Bounds: the inverse root is a float32 sum of squares (at most 64 additions one after the other in a thread, 10 across the CTA),
a division and a root: its relative error is below (74 / 2 + 4) 2^-24; with the products behind it everything is within
C = 48 x 2^-24 of the terms' magnitudes before it is rounded to its type (half a step)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

C = 48 * 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _stream(x, residual, post, gate, eps, scale, residual_scale, offset):
    """(h in 64 bits, the magnitudes that its error is measured by)."""
    p = x.double()
    if post is not None:
        p = p * (p.square().mean(-1, keepdim=True) + eps) ** -0.5 * (post.double() + offset)
    if gate is not None:
        p = p * gate.double()
    p = p * scale
    if residual is None:
        return p, p.abs()
    r = residual.double() * residual_scale
    return p + r, p.abs() + r.abs()


def _check(out, x, weight, residual=None, post_weight=None, gate=None, eps=1e-6, scale=1.0, residual_scale=1.0, weight_offset=0.0):
    rows, scales, h = out if len(out) == 3 else (out[0], None, out[1])
    stream = x.dtype if residual is None else residual.dtype
    assert h.dtype == stream and h.shape == x.shape and rows.shape == x.shape
    want, size = _stream(x, residual, post_weight, gate, eps, scale, residual_scale, weight_offset)
    tiny = torch.finfo(stream).tiny
    assert bool(((h.double() - want).abs() <= _half(stream) * want.abs() + 2 * C * size + tiny).all())
    # what follows is the norm of the stream as stored
    hd = h.double()
    w = torch.ones(x.shape[-1], device=x.device) if weight is None else weight.float() + weight_offset
    root = (hd.square().mean(-1, keepdim=True) + eps) ** -0.5
    if scales is None:
        z = hd * root * w.double()
        assert rows.dtype == x.dtype
        assert bool(((rows.double() - z).abs() <= (_half(x.dtype) + C) * z.abs() + torch.finfo(x.dtype).tiny).all())
        return
    t = (h.float() * w).double()
    top = t.abs().amax(-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(127.0 * t / top), 0.0)
    assert rows.dtype == torch.int8 and scales.dtype == torch.float32 and scales.shape == x.shape[:-1]
    assert torch.equal(rows, codes.to(torch.int8))
    want = (top * root / 127.0).squeeze(-1)
    assert bool(((scales.double() - want).abs() <= C * want + torch.finfo(torch.float32).tiny).all())


def _both(x, weight, **more):
    from liquidgemm_b200 import norms
    _check(norms.block_norm(x, weight, **more), x, weight, **more)
    _check(norms.block_norm_quant(x, weight, **more), x, weight, **more)


def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 4096), (3, 7), (5, 8), (2, 24), (33, 129), (300, 1000), (7, 5001), (64, 8192), (2, 14336),
                                 (3, 16384), (2, 32768), (1, 32767), (2000, 512)])
def test_sizes(T, H, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T + H)
    dtype = DTYPES[dtype]
    x = _randn(gen, T, H).to(dtype)
    weight = (1 + 0.3 * _randn(gen, H)).to(dtype)
    _both(x, weight)
    _both(x, weight, residual=(3 * _randn(gen, T, H)).to(dtype), eps=1e-5)


@pytest.mark.parametrize("H", [256, 1023])
@pytest.mark.parametrize("stream", ["same", "fp32", "none"])
@pytest.mark.parametrize("post", [None, "same", "fp32"])
@pytest.mark.parametrize("gate", [None, "channel", "row", "all", "number"])
def test_forms(H, stream, post, gate):
    gen = torch.Generator(device="cuda").manual_seed(H)
    for dtype in DTYPES.values():
        T = 37
        x = (2 * _randn(gen, T, H)).to(dtype)
        residual = None if stream == "none" else _randn(gen, T, H).to(dtype if stream == "same" else torch.float32)
        shape = {None: None, "channel": (H,), "row": (T, 1), "all": (T, H), "number": ()}[gate]
        _both(x, (0.2 * _randn(gen, H)).to(dtype), residual=residual, eps=1e-5,
              post_weight=None if post is None else (0.3 * _randn(gen, H)).to(dtype if post == "same" else torch.float32),
              gate=None if shape is None else _randn(gen, *shape).to(dtype), scale=0.4, residual_scale=1.5, weight_offset=1.0)
        _both(x, None, residual=residual, gate=None if shape is None else _randn(gen, *shape))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H", [(9000, 40), (6000, 512), (5000, 1000), (3001, 4096), (1500, 8192), (700, 10240), (400, 16384), (3001, 1001)])
def test_more_rows_than_the_gpu_holds(T, H, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T)
    dtype = DTYPES[dtype]
    x, weight = _randn(gen, T, H).to(dtype), (1 + 0.3 * _randn(gen, H)).to(dtype)
    x[::7] *= 30.0
    _both(x, weight)
    _both(x, weight, residual=_randn(gen, T, H).to(dtype), gate=_randn(gen, T, 1).to(dtype))
    _both(x, weight, residual=_randn(gen, T, H), post_weight=_randn(gen, H), gate=_randn(gen, T, H).to(dtype), scale=0.3, weight_offset=1.0)
    if dtype != torch.float16:
        x[T - 2] *= 1e30
        _both(x, weight, gate=_randn(gen, H))
    wide = torch.empty(T // 4, 4, H + 8, dtype=dtype, device="cuda").normal_(generator=gen)
    _both(wide[:, 1:3, 8:], weight, residual=wide[:, :2, :H], gate=_randn(gen, T // 4, 1, H))


def test_plain_norm_returns_its_rows():
    from liquidgemm_b200 import norms
    x = torch.randn(4, 64, device="cuda").to(torch.bfloat16)
    weight = torch.ones(64, device="cuda")
    assert norms.block_norm(x, weight)[1] is x and norms.block_norm_quant(x, weight)[2] is x


@pytest.mark.parametrize("gate_shape", [(5, 1, 96), (1, 96), (5, 1, 1), (1, 7, 1), (5, 7, 96), (1, 1, 1), (7, 96)])
def test_sequences_and_their_gates(gate_shape):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, residual = _randn(gen, 5, 7, 96).to(torch.bfloat16), _randn(gen, 5, 7, 96)
    _both(x, _randn(gen, 96), residual=residual, gate=_randn(gen, *gate_shape).to(torch.bfloat16))


def test_strides():
    gen = torch.Generator(device="cuda").manual_seed(2)
    wide = _randn(gen, 20, 400).to(torch.float16)
    stream = _randn(gen, 20, 2, 136).to(torch.float16)
    weight = _randn(gen, 300).to(torch.float16)
    for first in (0, 8, 3):   # rows on 16-byte boundaries, and not
        x = wide[:, first:first + 128]
        _both(x, weight[first:first + 128], residual=stream[:, 1, :128], gate=wide[:, 200:328])
        _both(x, weight[::2][:128], residual=stream[:, 0, 5:133], gate=wide[:, 7:8])
    x = wide.view(4, 5, 400)[:, 1:4, 16:144]          # two strides
    _both(x, weight[:128], residual=stream.view(4, 5, 2, 136)[:, 1:4, 1, 8:136], gate=wide.view(4, 5, 400)[:, :1, :128])
    _both(wide.t(), None, residual=stream[0, :, :20].reshape(-1)[:1].expand(400, 20))
    _both(x.transpose(0, 1), weight[:128])


def test_no_rows():
    from liquidgemm_b200 import norms
    x = torch.empty(0, 64, device="cuda")
    rows, scales, h = norms.block_norm_quant(x, None, residual=x)
    assert rows.shape == (0, 64) and scales.shape == (0,) and h.shape == (0, 64)
    assert norms.block_norm(torch.empty(3, 0, 64, device="cuda"), None)[0].shape == (3, 0, 64)


@pytest.mark.parametrize("H", [512, 1001])
def test_special_rows(H):
    """Rows of zeros, an infinity, NaN, and magnitudes whose squares float32 does not hold."""
    from liquidgemm_b200 import norms
    gen = torch.Generator(device="cuda").manual_seed(3)
    for dtype in (torch.bfloat16, torch.float32):
        x = _randn(gen, 9, H)
        x[1], x[2, 5], x[3, 7] = 0.0, float("inf"), float("nan")
        x[4] *= 1e30
        x[5] *= 1e-15
        x[6, 1:] = 0.0
        x[7, ::2] = -x[7, ::2].abs().max()
        x = x.to(dtype)
        weight = (1 + 0.1 * _randn(gen, H)).to(dtype)
        fine = [0, 1, 4, 5, 6, 7, 8]
        z, h = norms.block_norm(x, weight)
        rows, scales, _ = norms.block_norm_quant(x, weight)
        _check((z[fine], h[fine]), x[fine], weight)
        _check((rows[fine], scales[fine], h[fine]), x[fine], weight)
        assert scales[1] == 0 and not rows[1].any() and not z[1].any()
        assert torch.isnan(z[2, 5]) and torch.isnan(z[3]).all()
        assert torch.isnan(scales[2]) and torch.isnan(scales[3])


def test_ties_go_to_even():
    from liquidgemm_b200 import norms
    x = torch.tensor([[254.0] + [float(2 * i + 1) for i in range(127)]], device="cuda")   # 127 t / 254 = i + 1/2
    rows = norms.block_norm_quant(x, None)[0]
    assert rows[0].tolist() == [127] + [i + i % 2 for i in range(127)]


def test_weights_of_zero_and_subnormal_rows():
    from liquidgemm_b200 import norms
    x = torch.full((2, 128), 1e-41, device="cuda")
    x[1, 3] = -2e-41
    rows, scales, _ = norms.block_norm_quant(x, None, eps=1e-6)
    assert rows[0].tolist() == [127] * 128 and rows[1, 3] == -127 and torch.isfinite(scales).all()
    rows, scales, _ = norms.block_norm_quant(x + 1, torch.zeros(128, device="cuda"))
    assert not rows.any() and not scales.any()


def test_graph_and_streams():
    from liquidgemm_b200 import norms
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, residual, weight = _randn(gen, 300, 1024).to(torch.bfloat16), _randn(gen, 300, 1024), _randn(gen, 1024).to(torch.bfloat16)
    norms.block_norm_quant(x, weight, residual=residual)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = norms.block_norm_quant(x, weight, residual=residual)
        then = norms.block_norm(out[2].to(torch.bfloat16), weight, residual=out[2])
    for seed in range(3):
        gen.manual_seed(seed)
        x.copy_(_randn(gen, 300, 1024))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x, weight, residual=residual)
        _check(then, out[2].to(torch.bfloat16), weight, residual=out[2])
    want = norms.block_norm_quant(x, weight, residual=residual)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(10):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(norms.block_norm_quant(x, weight, residual=residual))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_through_the_dispatcher():
    from liquidgemm_b200 import norms
    x = torch.randn(6, 64, device="cuda")
    weight = torch.randn(64, device="cuda")
    z, scales, h = torch.ops.liquidgemm.block_norm(x, weight, x, None, None, 1e-6, 1.0, 1.0, 0.0, False)
    want = norms.block_norm(x, weight, residual=x)
    assert torch.equal(z, want[0]) and torch.equal(h, want[1]) and scales.numel() == 0
    with torch.no_grad():
        got = norms.block_norm(x.clone().requires_grad_(True), weight, residual=x)
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("T", [1, 3, 16, 200])
def test_a_layer_s_projection(T):
    """Norm and residual, INT8 rows, 4-bit and INT8 linears on them, adapters beside: one chain, against 64 bits."""
    from liquidgemm_b200 import adapters, norms, ops
    H, N = 512, 384
    gen = torch.Generator(device="cuda").manual_seed(T)
    w = (_randn(gen, N, H) * 0.05).to(torch.bfloat16)
    q, blob = ops.quantize_weight_cuda(w, want_codes=True, want_blob=True)
    w_i8 = ops.dequant_weight_i8(q)
    stack = adapters.make_stack(3, 8, H, (256, 128))
    for slot in range(3):
        adapters.load(stack, slot, [_randn(gen, 8, H) * 0.05 for _ in range(2)], [_randn(gen, n, 8) for n in (256, 128)], 0.5)
    x, residual = _randn(gen, T, H).to(torch.bfloat16), (2 * _randn(gen, T, H)).to(torch.bfloat16)
    weight = (1 + 0.2 * _randn(gen, H)).to(torch.bfloat16)
    ids = torch.randint(-1, 3, (T,), device="cuda", generator=gen)
    rows, scales, h = norms.block_norm_quant(x, weight, residual=residual)
    z, h2 = norms.block_norm(x, weight, residual=residual)
    assert torch.equal(h, h2)
    y4 = torch.ops.liquidgemm.w4a8_wgmma_rs_fused(rows, blob, q.s_u8, q.offset_a, scales, q.s1, N, H, 64, 0)
    y8 = torch.ops.liquidgemm.i8_gemm_scaled(rows, w_i8, scales, q.s1, 0)
    assert torch.equal(y4, y8)
    exact = (rows.double() @ w_i8.double().t()) * scales.double()[:, None] * q.s1.double().flatten()
    assert bool(((y4.double() - exact).abs() <= (2.0 ** -8 + 2.0 ** -22) * exact.abs() + 1e-30).all())
    out = adapters.add(y4, z, stack, ids)
    want, zd = y4.double(), z.double()
    for l in range(3):
        mine = ids == l
        for s, (a, b) in enumerate(((0, 256), (256, 384))):
            want[mine, a:b] += 0.5 * (zd[mine] @ stack["a"][l, s].double().t()) @ stack["b"][l, a:b].double().t()
    # half a step of bf16, and what the adapters' float32 sums and 16-bit parts are off (8 terms of a few units each)
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * 8 * zd.abs().amax(1, keepdim=True)).all())
