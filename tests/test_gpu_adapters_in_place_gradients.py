"""``y`` changed in place where gradients are asked for: refused, since the adapters have none to give; out of place torch says so itself
in the backward pass."""

import pytest
import torch

from test_gpu_adapters_in_place_and_autograd import _call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("through", ["entry", "operator"])
@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("asks", ["y", "y's leaf", "x", "a", "b", "scale"])
def test_refused(asks, T, through):
    from liquidgemm_b200 import adapters
    y, x, stack, ids = _call(T)
    stack = dict(stack)
    if asks == "y":
        y.requires_grad_()
    elif asks == "y's leaf":
        y = y.clone().requires_grad_() * 2
    elif asks == "x":
        x.requires_grad_()
    else:
        stack[asks] = stack[asks].clone().requires_grad_()

    def call():
        if through == "entry":
            return adapters.add(y, x, stack, ids, inplace=True)
        return torch.ops.liquidgemm.adapters_add_(y, x, stack["a"], stack["b"], stack["rank"], stack["scale"], ids, [y.shape[1]])

    before = y.detach().clone()
    with pytest.raises(RuntimeError, match="no gradients"):
        call()
    assert torch.equal(y.detach(), before)
    assert adapters.add(y, x, stack, ids).requires_grad
    want = adapters.add(y.detach(), x.detach(), {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in stack.items()}, ids)
    with torch.no_grad():
        call()
    assert torch.equal(y.detach(), want)
