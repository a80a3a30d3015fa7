"""``scale`` and ``residual_scale`` of any size: what a factor of 0 takes out is out, however large, and an infinity stays one."""

import pytest
import torch

from test_gpu_norms import _both, _randn

pytestmark = pytest.mark.gpu


def _huge(gen, T, H, dtype):
    return ((1.0 + 2.0 * torch.rand(T, H, device="cuda", generator=gen)) * 1e38).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", [256, 1001])
def test_factors_of_zero(H, dtype):
    from liquidgemm_b200 import norms
    gen = torch.Generator(device="cuda").manual_seed(H)
    huge, some = _huge(gen, 6, H, dtype), _randn(gen, 6, H).to(dtype)
    some[:, ::3] = 0.0
    weight = torch.ones(H, device="cuda")
    for zero in (0.0, -0.0, 1e-300):
        for more in ({}, {"gate": torch.ones(H, device="cuda")}, {"post_weight": weight}):
            for f in (norms.block_norm, norms.block_norm_quant):
                assert torch.equal(f(huge, weight, residual=some, scale=zero, **more)[-1], some)
        assert torch.equal(norms.block_norm(some, weight, residual=huge, residual_scale=zero, scale=2.0)[1], some * 2.0)
        assert not norms.block_norm(huge, weight, scale=zero)[1].any()


@pytest.mark.parametrize("H", [256, 1001])
def test_small_factors(H):
    gen = torch.Generator(device="cuda").manual_seed(H)
    huge, some = _huge(gen, 6, H, torch.float32), _randn(gen, 6, H)
    for f in (1e-30, 2.0 ** -100, 2.0 ** -101, 1e-37, 2.0 ** -127, 3e-39):
        _both(huge, None, scale=f)
        _both(huge, None, residual=some, scale=f, gate=some)
        _both(some * 1e-3, None, residual=huge, residual_scale=f)


@pytest.mark.parametrize("scale", [1.0, 0.5, -0.3, 1e-20, 3.0])
def test_infinities_keep_their_sign(scale):
    from liquidgemm_b200 import norms
    x = torch.ones(3, 64, device="cuda")
    x[1, 5], x[2, 7] = float("inf"), float("-inf")
    h = norms.block_norm(x, None, residual=torch.ones(3, 64, device="cuda"), scale=scale, residual_scale=2.0)[1]
    assert torch.equal(h.isinf(), x.isinf()) and torch.equal(h.sign()[x.isinf()], (x * scale).sign()[x.isinf()]) and not h.isnan().any()
    h = norms.block_norm(torch.ones(3, 64, device="cuda"), None, residual=x, residual_scale=scale)[1]
    assert torch.equal(h.isinf(), x.isinf()) and torch.equal(h.sign()[x.isinf()], (x * scale).sign()[x.isinf()]) and not h.isnan().any()
