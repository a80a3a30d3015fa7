"""Every tile width of both weight kinds, on both sides of each limit of the rule that chooses it by the rows an expert gets on average:
products bit for bit, the MLP by the tolerance derived in test_gpu_experts.py."""

import pytest
import torch

from test_gpu_experts import _check_mlp, _gen, _linear, _quantise, _rows, _stack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe():
    from liquidgemm_b200 import moe as _moe
    return _moe


@pytest.mark.parametrize("w4", [True, False], ids=["w4", "int8"])
@pytest.mark.parametrize("mean", [10, 11, 40, 41, 44, 45, 48, 49, 96, 127, 128])
def test_both_sides_of_each_limit(moe, w4, mean):
    E, N, K = 5, 328, 384
    layer, q, s1 = _stack(moe, E, N, K, w4, mean)
    T = mean * E + 3
    popular = torch.tensor([4.0, 2.0, 1.0, 1.0, 0.0], device="cuda")       # one expert has half of the rows, one none
    ids = torch.multinomial(popular, T, replacement=True, generator=_gen(mean)).to(torch.int32)[:, None].contiguous()
    x = _rows((T, K), torch.bfloat16, mean)
    xq, scale = _quantise(x)
    assert torch.equal(moe.experts_linear(x, ids, layer), _linear(xq, scale, ids, q, s1, False, torch.bfloat16))
    for k in (1, 4):
        _check_mlp(moe, mean * E // k + 1, E, k, 256, 384, w4, "random", torch.bfloat16, mean)
