"""The down product of an MLP with its k-steps dealt out in equal shares: alone and together with the gate/up product, behind plans made by
the placing kernel (up to 2048 pairs, with rows so short that it runs as a single warp) and by the plan kernel.  Scratch may hold
anything before a call.  The tolerance is the one derived in test_gpu_experts.py; repeated calls give the same bits."""

import pytest
import torch

from test_gpu_experts import _gen, _mlp, _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe():
    from liquidgemm_b200 import moe as _moe
    return _moe


def _stack(moe, E, N, K, seed, gated):
    """(4-bit layer, its values [E, N, K] in the order given, scales)."""
    w = (torch.randn(E, N, K, device="cuda", generator=_gen(seed)) * 0.05).to(torch.bfloat16)
    values = moe.quantize_experts(w, w4=False)
    return moe.quantize_experts(w, gated=gated), values["w"], values["s1"]


def _call(moe, x, weights, ids, w13, w2, fill):
    """The C entry on scratch filled with one byte."""
    from liquidgemm_b200._lib import check, lib
    T, H = x.shape
    k, E, inner = ids.shape[1], w2["E"], w2["K"]
    scratch = torch.full((lib.lq_experts_mlp_scratch_bytes(T, k, E, H, inner, 0),), fill, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x)
    check(lib.lq_experts_mlp(x.data_ptr(), moe._DTYPE_CODES[x.dtype], weights.data_ptr(), ids.data_ptr(), w13["w"].data_ptr(),
                             w13["s1"].data_ptr(), w2["w"].data_ptr(), w2["s1"].data_ptr(), 0, y.data_ptr(),
                             moe._DTYPE_CODES[x.dtype], T, k, E, H, inner, scratch.data_ptr(), scratch.numel(),
                             torch.cuda.current_stream().cuda_stream), "experts_mlp")
    return y


# With 2 x 148 CTAs.  T, k, E, H, I, dtype: one warp places rows of 256 bytes (512) in the first four; 300 to 320 tiles of 32 k-steps
CASES = [
    (200, 8, 300, 128, 4096, torch.bfloat16), (200, 8, 150, 256, 4096, torch.float16), (150, 2, 300, 128, 4096, torch.float32),
    (38, 8, 300, 128, 4096, torch.bfloat16),
    (200, 8, 150, 256, 4096, torch.float32),                                                   # two warps
    (400, 8, 320, 128, 4096, torch.bfloat16), (300, 8, 300, 256, 4096, torch.float32),         # more than 2048 pairs
    (50, 2, 10, 4096, 2304, torch.bfloat16), (16, 1, 10, 4096, 2304, torch.float16),           # both products
]


@pytest.mark.parametrize("T,k,E,H,inner,dtype", CASES)
def test_second_product_in_shares(moe, T, k, E, H, inner, dtype):
    w13, q13, s13 = _stack(moe, E, 2 * inner, H, 1, True)
    w2, q2, s2 = _stack(moe, E, H, inner, 2, False)
    x = _rows((T, H), dtype, 3)
    weights = torch.rand(T, k, device="cuda", generator=_gen(4))
    # every expert is reached, in an order of its own
    ids = ((torch.arange(T * k, device="cuda") * 7) % E).view(T, k).to(torch.int32)
    assert len(ids.unique()) == min(E, T * k)
    want, tol = torch.zeros(T, H, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e0 in range(0, E, 50):          # (the values of all experts in 64 bits would fill gigabytes)
        mine = (ids >= e0) & (ids < e0 + 50)
        part, off = _mlp(x, weights, torch.where(mine, ids - e0, -1), q13[e0:e0 + 50].double(), s13[e0:e0 + 50],
                         q2[e0:e0 + 50].double(), s2[e0:e0 + 50])
        want += part
        tol += off
    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    first = None
    for fill in (1, 0, 255, 1, 127):
        y = _call(moe, x, weights, ids, w13, w2, fill)
        assert torch.all((y.double() - want).abs() <= tol)
        assert first is None or torch.equal(y, first)
        first = y
    for _ in range(3):                  # scratch as the call before left it
        assert torch.equal(moe.experts_mlp(x, weights, ids, w13, w2), first)
