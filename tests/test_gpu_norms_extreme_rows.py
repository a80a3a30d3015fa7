"""Norms of rows whose squares float32 does not hold, against the formula in 64 bits (bounds as in test_gpu_norms)."""

import pytest
import torch

from test_gpu_norms import _both, _randn

pytestmark = pytest.mark.gpu


def _large(gen, T, H, dtype):
    """Elements between 1e38 and 3e38, one such element among ordinary ones, squares that float32 just does not hold, and ordinary rows between."""
    x = _randn(gen, T, H)
    huge = (1.0 + 2.0 * torch.rand(T, H, device="cuda", generator=gen)) * torch.where(x > 0, 1e38, -1e38)
    x[0::5] = huge[0::5]
    x[1::5, H // 3] = huge[1::5, H // 3]
    x[2::5] *= 2e19
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(10, 512), (10, 1001), (1000, 4096), (10, 5000), (10, 16384), (10, 32768), (10, 32767)])
def test_large_rows_through_the_norm_of_the_output(T, H, dtype):
    """By the root first, then by weight and gate: ``h`` is an ordinary number however large ``x`` is."""
    gen = torch.Generator(device="cuda").manual_seed(H)
    x, weight, post = _large(gen, T, H, dtype), (1 + 0.2 * _randn(gen, H)).to(dtype), 3.0 * _randn(gen, H)
    _both(x, weight, post_weight=post)
    _both(x, weight, residual=_randn(gen, T, H), post_weight=post.to(dtype), gate=4.0 * _randn(gen, H), scale=0.7, residual_scale=1.5)
    _both(x, None, residual=_randn(gen, T, H).to(dtype), post_weight=post, gate=4.0 * _randn(gen, T, H).to(dtype), weight_offset=1.0)
    _both(x, weight, post_weight=post, gate=_randn(gen, T, 1).to(dtype), scale=-3.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", [8, 256, 1001])
def test_rows_that_lie_apart(H, dtype):
    """Two strides, gates of a sequence and of a row, more rows than CTAs: ordinary, large and small rows side by side."""
    gen = torch.Generator(device="cuda").manual_seed(H)
    B, S = 40, 60
    wide = _randn(gen, B, S + 2, H + 24)
    wide[:, 0::7] *= 1e30
    wide[:, 3::7] *= 1e-30
    wide = wide.to(dtype)
    x, residual = wide[:, 1:S + 1, 8:H + 8], wide[:, 2:S + 2, 16:H + 16]
    post = (1 + 0.2 * _randn(gen, H)).to(dtype)
    _both(x, post, eps=0.0)
    _both(x, None, post_weight=post, residual=residual, gate=_randn(gen, B, 1, H), eps=0.0)
    _both(x, post, post_weight=post, residual=_randn(gen, B, S, H), gate=_randn(gen, B, S, 1).to(dtype), eps=1e-5)
    _both(x, post, residual=residual, gate=_randn(gen, S, 1), scale=0.5, eps=1e-5)
