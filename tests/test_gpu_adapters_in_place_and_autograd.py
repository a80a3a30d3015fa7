"""``y`` changed in place beside autograd: the change is one that autograd knows of."""

import pytest
import torch

pytestmark = pytest.mark.gpu

K, N = 64, 32


def _call(T=5, dtype=torch.bfloat16):
    from liquidgemm_b200 import adapters
    gen = torch.Generator(device="cuda").manual_seed(T)
    stack = adapters.make_stack(2, 8, K, N, dtype=dtype)
    adapters.load(stack, 0, torch.randn(8, K, device="cuda", generator=gen), torch.randn(N, 8, device="cuda", generator=gen))
    x, y = (torch.randn(T, n, device="cuda", generator=gen).to(dtype) for n in (K, N))
    return y, x, stack, torch.zeros(T, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("through", ["entry", "operator"])
@pytest.mark.parametrize("T", [5, 200])
def test_what_autograd_has_kept_of_y_is_known_to_be_gone(T, through):
    from liquidgemm_b200 import adapters
    y, x, stack, ids = _call(T)
    w = torch.ones(N, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    loss = (w * y).sum()   # keeps y for w's gradient
    before = y._version
    if through == "entry":
        adapters.add(y, x, stack, ids, inplace=True)
    else:
        torch.ops.liquidgemm.adapters_add_(y, x, stack["a"], stack["b"], stack["rank"], stack["scale"], ids, [N])
    assert y._version > before
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    part = y[:2]   # a view counts for the whole
    before = y._version
    adapters.add(part, x[:2], stack, ids[:2], inplace=True)
    assert y._version > before
    before = y._version
    adapters.add(y, x, stack, ids)
    assert y._version == before


def test_inference_mode():
    from liquidgemm_b200 import adapters
    y, x, stack, ids = _call()
    want = adapters.add(y, x, stack, ids)
    with torch.inference_mode():
        z = y.clone()
        assert torch.equal(adapters.add(z, x, stack, ids, inplace=True), want)
        assert torch.equal(adapters.add(y, x, stack, ids, inplace=True), want)
    assert torch.equal(adapters.add(z, x, stack, ids, inplace=True), adapters.add(want, x, stack, ids))
