"""Low-rank adapters on the device, against the formula in 64 bits.

Bounds: a product of two 16-bit numbers is exact in float32.  A sum of n of them by MMAs of 16 is at most n / 16 + 40 additions one
after the other (8 warps and 16 parts of K are added up behind them), each off by at most 2^-22 of the sum of magnitudes (an MMA may
cut instead of rounding).  The intermediate row goes on as two 16-bit numbers: at most 2^-16 of it is lost (bf16: two halves
of 2^-9 each), and in fp16 never more than 2^-37 of the row's largest magnitude.  The result is rounded once: half a step."""

import pytest
import torch

gpu = pytest.mark.gpu
pytestmark = gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _stack(L, rank, K, widths, dtype, seed, ranks=None):
    from liquidgemm_b200 import adapters
    gen = torch.Generator(device="cuda").manual_seed(seed)
    stack = adapters.make_stack(L, rank, K, widths, dtype=dtype)
    for l in range(L):
        r = rank if ranks is None else ranks[l % len(ranks)]
        if r == 0:
            continue
        a = [(torch.randn(r, K, device="cuda", generator=gen) / K ** 0.5).to(dtype) for _ in stack["widths"]]
        b = [(torch.randn(w, r, device="cuda", generator=gen) * 0.5).to(dtype) for w in stack["widths"]]
        adapters.load(stack, l, a, b, 0.25 + 0.5 * l)
    return stack


def _reference(y, x, stack, ids):
    """(result in 64 bits, bound of its error before the last rounding)."""
    y, x = y.double(), x.double()
    out, bound = y.clone(), torch.zeros_like(y)
    K, least = stack["K"], 2.0 ** -37
    for l in range(stack["rank"].shape[0]):
        mine = (ids == l).nonzero().flatten()
        at = 0
        for s, w in enumerate(stack["widths"]):
            r = int(stack["rank"][l, s])
            if r and len(mine):
                a, b = stack["a"][l, s, :r].double(), stack["b"][l, at:at + w, :r].double()
                scale = stack["scale"][l].double()
                v, va = x[mine] @ a.t(), x[mine].abs() @ a.abs().t()
                ev = (K / 16 + 40) * 2.0 ** -22 * va + 2.0 ** -16 * v.abs() + least * v.abs().amax(1, keepdim=True)
                out[mine, at:at + w] += scale * (v @ b.t())
                bound[mine, at:at + w] = scale * (ev @ b.abs().t() + (r / 8 + 40) * 2.0 ** -22 * (v.abs() @ b.abs().t()))
            at += w
    return out, bound


def _check(got, y, x, stack, ids):
    want, bound = _reference(y, x, stack, ids)
    half = torch.finfo(got.dtype).eps / 2
    limit = bound + half * (want.abs() + bound) + 2.0 ** -23 * (y.double().abs() + want.abs()) + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), f"off by {(off / limit).max().item():.2f} of the bound"


def _inputs(T, K, N, dtype, seed, y_dtype=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, K, device="cuda", generator=gen).to(dtype)
    y = (2 * torch.randn(T, N, device="cuda", generator=gen)).to(y_dtype or dtype)
    return x, y, gen


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,widths,L,rank", [
    (1, 128, 64, 1, 8), (1, 4096, (512, 128, 128), 5, 16), (2, 8, 8, 3, 1), (7, 264, (72, 24), 4, 5), (32, 1024, 520, 40, 16),
    (63, 520, 136, 3, 12), (64, 512, 256, 2, 32), (65, 512, 256, 1, 24), (200, 2048, (64, 1000, 8), 9, 64),
    (333, 1000, 328, 16, 40), (1000, 640, 1032, 300, 16), (700, 768, (128, 256), 4, 128), (130, 384, 512, 2, 256),
    (129, 256, (512,) * 8, 3, 72), (4096, 256, 512, 8, 16), (20, 128, (64,) * 8, 4, 72), (100, 64, 8200, 7, 16), (10, 384, 512, 3, 256),
    (128, 4096, 8192, 128, 16), (65, 256, 8192, 1, 48), (3, 14336, (128, 64, 8), 2, 33), (9000, 64, 72, 500, 8),
])
def test_add(T, K, widths, L, rank, dtype):
    from liquidgemm_b200 import adapters
    dtype = DTYPES[dtype]
    stack = _stack(L, rank, K, widths, dtype, T + K)
    x, y, gen = _inputs(T, K, stack["N"], dtype, T)
    ids = torch.randint(-1, L + 1, (T,), device="cuda", generator=gen)
    before = y.clone()
    got = adapters.add(y, x, stack, ids)
    assert torch.equal(y, before) and got.dtype == y.dtype
    _check(got, y, x, stack, ids)
    none = (ids < 0) | (ids >= L)
    assert torch.equal(got[none], y[none])
    again = adapters.add(y, x, stack, ids.int())
    assert torch.equal(got, again)
    assert adapters.add(y, x, stack, ids, inplace=True) is y and torch.equal(y, got)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,rank", [(3, 16), (90, 32), (300, 64), (65, 200), (131, 8), (200, 32), (140, 120), (150, 250)])
def test_float32_outputs(T, rank, dtype):
    from liquidgemm_b200 import adapters
    stack = _stack(4, rank, 512, (136, 72), DTYPES[dtype], 3)
    x, y, gen = _inputs(T, 512, 208, DTYPES[dtype], T, torch.float32)
    ids = torch.randint(0, 4, (T,), device="cuda", generator=gen)
    got = adapters.add(y, x, stack, ids)
    assert got.dtype == torch.float32
    _check(got, y, x, stack, ids)


def test_ranks_of_their_own_and_empty_slots():
    from liquidgemm_b200 import adapters
    stack = _stack(6, 64, 256, (64, 128), torch.bfloat16, 5, ranks=[1, 8, 17, 0, 40, 64])
    a, b = stack["a"], stack["b"]
    adapters.load(stack, 3, [torch.randn(9, 256), None], [torch.randn(64, 9), None], 2.0)
    x, y, gen = _inputs(150, 256, 192, torch.bfloat16, 6)
    ids = torch.randint(0, 6, (150,), device="cuda", generator=gen)
    got = adapters.add(y, x, stack, ids)
    _check(got, y, x, stack, ids)
    mine = ids == 3
    assert torch.equal(got[mine, 64:], y[mine, 64:])   # the slice without matrices
    adapters.unload(stack, 5)
    assert stack["a"] is a and stack["b"] is b
    got = adapters.add(y, x, stack, ids)
    assert torch.equal(got[ids == 5], y[ids == 5])
    _check(got, y, x, stack, ids)


@pytest.mark.parametrize("order", ["one", "sorted", "mixed", "none"])
def test_batches(order):
    """One adapter for all, requests one behind the other, mixed rows, no adapter at all; a -0 without an adapter stays one."""
    from liquidgemm_b200 import adapters
    stack = _stack(12, 16, 384, 136, torch.float16, 8)
    T = 500
    x, y, gen = _inputs(T, 384, 136, torch.float16, 9)
    y[:, 0] = -0.0
    ids = torch.randint(0, 12, (T,), device="cuda", generator=gen)
    ids = {"one": torch.full_like(ids, 7), "sorted": ids.sort().values, "mixed": ids, "none": torch.full_like(ids, -5)}[order]
    got = adapters.add(y, x, stack, ids)
    _check(got, y, x, stack, ids)
    if order == "none":
        assert torch.equal(got.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("T", [40, 160])
def test_strides(T):
    from liquidgemm_b200 import adapters
    stack = _stack(3, 16, 256, 64, torch.bfloat16, 1)
    ids = torch.arange(T, device="cuda") % 3
    wide_x, wide_y, _ = _inputs(T, 512, 200, torch.bfloat16, 2)
    x, y = wide_x[:, 128:384], wide_y[:, 8:72]
    want = adapters.add(y.contiguous(), x.contiguous(), stack, ids)
    rest = wide_y.clone()
    assert torch.equal(adapters.add(y, x, stack, ids), want)
    assert torch.equal(adapters.add(wide_y[:, 8:72].t().contiguous().t(), wide_x[:, 128:384].t().contiguous().t(), stack, ids), want)
    odd = torch.zeros(T * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, 64)
    odd.copy_(y)
    assert torch.equal(adapters.add(odd, x, stack, torch.stack([ids, ids], 1)[:, 0]), want)
    adapters.add(y, x, stack, ids, inplace=True)   # a part of a larger tensor: what stands beside it stays
    assert torch.equal(y, want)
    rest[:, 8:72] = want
    assert torch.equal(wide_y, rest)
    with pytest.raises(RuntimeError, match="in place"):
        adapters.add(odd, x, stack, ids, inplace=True)
    one = wide_y[:1, 8:72]
    assert torch.equal(adapters.add(one, x[:1], stack, ids[:1]), adapters.add(one.clone(), x[:1], stack, ids[:1]))


def test_no_rows():
    from liquidgemm_b200 import adapters
    stack = _stack(2, 8, 64, 64, torch.bfloat16, 1)
    y = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    assert adapters.add(y, torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), stack,
                        torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, 64)


@pytest.mark.parametrize("T", [70, 200])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_special_values_stay_in_their_rows(dtype, T):
    """Infinities and NaN in x or y reach their own row alone; large and small rows keep their precision."""
    from liquidgemm_b200 import adapters
    dtype = DTYPES[dtype]
    stack = _stack(2, 12, 128, (64, 64), dtype, 4)
    stack["rank"][1, 1] = 0                     # a slice without matrices: not touched by what x holds
    x, y, _ = _inputs(T, 128, 128, dtype, 5)
    x[3, 5], x[9, 0], y[11, 2] = float("inf"), float("nan"), float("-inf")
    x[20] *= 100.0
    x[21] *= 1e-4
    x[22] = 0.0
    ids = torch.arange(T, device="cuda") % 2
    got = adapters.add(y, x, stack, ids)
    plain = torch.ones(T, dtype=torch.bool, device="cuda")
    plain[[3, 9, 11]] = False
    _check(got[plain], y[plain], x[plain], stack, ids[plain])
    assert torch.equal(got[22], y[22])
    assert not torch.isfinite(got[3, :64]).any() and torch.isnan(got[9, :64]).all()
    assert torch.equal(got[[3, 9], 64:], y[[3, 9], 64:])
    assert got[11, 2] == float("-inf") and torch.isfinite(got[11, 3:]).all()


@pytest.mark.parametrize("T", [5, 150])
def test_fp16_intermediate_beyond_its_range(T):
    from liquidgemm_b200 import adapters
    stack = adapters.make_stack(1, 8, 1024, 64, dtype=torch.float16)
    adapters.load(stack, 0, torch.full((8, 1024), 30.0), torch.full((64, 8), 2.0 ** -14), 1.0)
    x = torch.full((T, 1024), 60.0, dtype=torch.float16, device="cuda")   # A x = 1 843 200
    y = torch.zeros(T, 64, dtype=torch.float16, device="cuda")
    got = adapters.add(y, x, stack, torch.zeros(T, dtype=torch.int32, device="cuda"))
    assert torch.equal(got, torch.full_like(got, 900.0))


@pytest.mark.parametrize("w4", [True, False])
@pytest.mark.parametrize("T", [1, 2, 16, 300])
def test_linear_is_the_linear_and_add(T, w4):
    from liquidgemm_b200 import adapters, ops
    N, K = 256, 512
    gen = torch.Generator(device="cuda").manual_seed(7)
    w = (torch.randn(N, K, device="cuda", generator=gen) * 0.05).to(torch.bfloat16)
    q, blob = ops.quantize_weight_cuda(w, want_codes=True, want_blob=True)
    layer = {"s1": q.s1, "N": N, "K": K}
    layer.update({"rs": blob, "s_u8": q.s_u8, "offset_a": q.offset_a} if w4 else {"w_i8": ops.dequant_weight_i8(q)})
    stack = _stack(3, 16, K, (128, 64, 64), torch.bfloat16, 2)
    x, _, gen = _inputs(T, K, N, torch.bfloat16, 3)
    bias = torch.randn(N, device="cuda", generator=gen).to(torch.bfloat16)
    ids = torch.randint(-1, 3, (T,), device="cuda", generator=gen)
    rows, scales = torch.ops.liquidgemm.quant_per_token(x)
    base = torch.ops.liquidgemm.w4a8_linear_bias(rows, blob, scales, q.s1, None, N, K, 0)
    for b in (None, bias):
        y = base if b is None else base + b
        got = adapters.linear(x, layer, stack, ids, bias=b)
        assert torch.equal(got, adapters.add(y, x, stack, ids))
        _check(got, y, x, stack, ids)
    wide = adapters.linear(x, layer, stack, ids, out_dtype=torch.float32)
    assert wide.dtype == torch.float32
    _check(wide, torch.ops.liquidgemm.w4a8_linear_bias(rows, blob, scales, q.s1, None, N, K, 2), x, stack, ids)


@pytest.mark.parametrize("T", [1, 100, 300])
def test_graph_replayed_with_other_ids_and_slots(T):
    from liquidgemm_b200 import adapters
    stack = _stack(4, 16, 256, 128, torch.bfloat16, 1)
    x, y, gen = _inputs(T, 256, 128, torch.bfloat16, 2)
    ids = torch.randint(-1, 4, (T,), device="cuda", generator=gen)
    adapters.add(y, x, stack, ids)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        a = adapters.add(y, x, stack, ids)
    with torch.cuda.graph(second):   # graphs of their own: neither uses what the other holds
        b = adapters.add(y, x, stack, ids)
    for seed in (3, 4):
        gen.manual_seed(seed)
        ids.copy_(torch.randint(-1, 4, (T,), device="cuda", generator=gen))
        x.copy_(torch.randn(T, 256, device="cuda", generator=gen))
        adapters.load(stack, 1, torch.randn(5, 256, device="cuda", generator=gen) * 0.1, torch.randn(128, 5, device="cuda", generator=gen))
        a.zero_(), b.zero_()
        first.replay()
        second.replay()
        first.replay()
        torch.cuda.synchronize()
        want = adapters.add(y, x, stack, ids)
        assert torch.equal(a, want) and torch.equal(b, want)
        _check(want, y, x, stack, ids)


def test_streams_side_by_side():
    from liquidgemm_b200 import adapters
    stack = _stack(4, 32, 512, 256, torch.bfloat16, 1)
    work = []
    for i in range(4):
        x, y, gen = _inputs(50 + 40 * i, 512, 256, torch.bfloat16, i)
        work.append((y, x, torch.randint(0, 4, (x.shape[0],), device="cuda", generator=gen)))
    want = [adapters.add(y, x, stack, ids) for y, x, ids in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(10):
        got = []
        for s, (y, x, ids) in zip(streams, work):
            with torch.cuda.stream(s):
                got.append(adapters.add(y, x, stack, ids))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_through_the_dispatcher():
    from liquidgemm_b200 import adapters
    stack = _stack(2, 16, 128, 64, torch.bfloat16, 1)
    x, y, _ = _inputs(9, 128, 64, torch.bfloat16, 2)
    ids = torch.arange(9, device="cuda") % 3
    want = adapters.add(y, x, stack, ids)
    args = (x, stack["a"], stack["b"], stack["rank"], stack["scale"], ids, [64])
    assert torch.equal(torch.ops.liquidgemm.adapters_add(y, *args), want)
    changed = y.clone()
    assert torch.ops.liquidgemm.adapters_add_(changed, *args) is None
    assert torch.equal(changed, want)
    with torch.no_grad():
        assert torch.equal(adapters.add(y, x.clone().requires_grad_(True), stack, ids), want)
