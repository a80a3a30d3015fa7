"""Products of an element with its gate that float32 does not hold, where the formula's stream is an ordinary number: against
64 bits (bounds as in test_gpu_norms)."""

import pytest
import torch

from test_gpu_norms import _both, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(6, 256), (6, 1001), (900, 4096), (6, 16384), (6, 32767)])
def test_scales_that_bring_the_product_back(T, H, dtype):
    gen = torch.Generator(device="cuda").manual_seed(H)
    x, residual = _randn(gen, T, H), _randn(gen, T, H)
    x[::3] = ((1.0 + 2.0 * torch.rand(T, H, device="cuda", generator=gen)) * 1e38)[::3]
    x[1::3, H // 2] = -3e38
    x = x.to(dtype)
    for gate in (3.0 + _randn(gen, T, H).abs(), (3.0 + _randn(gen, H).abs()).to(dtype), torch.full((T, 1), 8.0, device="cuda", dtype=dtype)):
        for more in ({}, {"residual": residual}, {"residual": residual.to(dtype), "residual_scale": 0.5}):
            _both(x, None, gate=gate, scale=2.0 ** -96, **more)
            _both(x, _randn(gen, H).to(dtype), gate=gate, scale=-1e-25, **more)
    _both(residual.to(dtype), None, post_weight=torch.full((H,), 1e30, device="cuda"), gate=torch.full((H,), 1e30, device="cuda"), scale=1e-30)
