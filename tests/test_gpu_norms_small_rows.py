"""Norms of rows whose squares float32 cannot tell from 0, where eps does not stand above them: against the formula in 64 bits (bounds as
in test_gpu_norms).  Rows of zeros stay zeros whatever eps."""

import pytest
import torch

from test_gpu_norms import _both, _check, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-300, 1e-50, 1e-40, 1e-37])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(14, 512), (14, 1001), (700, 4096), (14, 5000), (14, 16384), (14, 32767)])
def test_small_rows(T, H, dtype, eps):
    gen = torch.Generator(device="cuda").manual_seed(H)
    x = _randn(gen, T, H)
    for i, size in enumerate((1e-15, 2.0 ** -59, 2.0 ** -60, 2.0 ** -61, 1e-25, 1e-38, 1e-40)):   # (between them the border, and subnormal numbers)
        x[i::7] *= size
    x = x.to(dtype)
    weight, post = (1 + 0.2 * _randn(gen, H)).to(dtype), (1 + 0.2 * _randn(gen, H)).to(dtype)
    _both(x, weight, eps=eps)
    _both(x, None, post_weight=post, gate=_randn(gen, H), scale=0.5, eps=eps)
    _both(x, weight, residual=x.flip(1).contiguous(), residual_scale=0.5, eps=eps)
    _both(x, weight, residual=_randn(gen, T, H), post_weight=post, eps=eps)


@pytest.mark.parametrize("eps", [0.0, 1e-50, 1e-6])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H", [64, 1001, 4096])
def test_rows_of_zeros(H, dtype, eps):
    from liquidgemm_b200 import norms
    gen = torch.Generator(device="cuda").manual_seed(H)
    x = _randn(gen, 9, H).to(dtype)
    x[::2] = 0.0
    x[0, ::3] = -0.0
    weight, post = _randn(gen, H).to(dtype), _randn(gen, H)
    for more in ({}, {"post_weight": post}, {"residual": torch.zeros(9, H, device="cuda"), "post_weight": post, "gate": _randn(gen, 9, 1).to(dtype)}):
        z, h = norms.block_norm(x, weight, eps=eps, **more)
        rows, scales, h2 = norms.block_norm_quant(x, weight, eps=eps, **more)
        assert not z[::2].any() and not h[::2].any() and not rows[::2].any() and not scales[::2].any() and torch.equal(h, h2)
        more = {k: v[1::2] if v.shape[0] == 9 else v for k, v in more.items()}
        _check((z[1::2], h[1::2]), x[1::2], weight, eps=eps, **more)
        _check((rows[1::2], scales[1::2], h[1::2]), x[1::2], weight, eps=eps, **more)
