"""Adapters loaded from matrices that are the stack's own: rescaled in place, copied to another slot, their slices exchanged."""

import pytest
import torch

from liquidgemm_b200 import adapters

K, WIDTHS, R = 32, (16, 16), (5, 8)


def _stack():
    gen = torch.Generator().manual_seed(1)
    stack = adapters.make_stack(3, 8, K, WIDTHS, device="cpu")
    pairs = []
    for slot in range(2):
        a, b = [torch.randn(r, K, generator=gen) for r in R], [torch.randn(w, r, generator=gen) for w, r in zip(WIDTHS, R)]
        adapters.load(stack, slot, a, b, 0.5 + slot)
        pairs.append(([t.to(torch.bfloat16) for t in a], [t.to(torch.bfloat16) for t in b]))
    return stack, pairs


def _own(stack, slot, order=(0, 1), ranks=R):
    """Views of a slot's matrices, as many rows as `ranks` says."""
    a = [stack["a"][slot, s, :ranks[s]] for s in order]
    b = [stack["b"][slot, s * 16:s * 16 + 16, :ranks[s]] for s in order]
    return a, b


def _holds(stack, slot, a, b, scale):
    assert stack["rank"][slot].tolist() == [t.shape[0] for t in a] and stack["scale"][slot] == scale
    for s in range(2):
        r = a[s].shape[0]
        assert torch.equal(stack["a"][slot, s, :r], a[s]) and not stack["a"][slot, s, r:].any()
        assert torch.equal(stack["b"][slot, s * 16:s * 16 + 16, :r], b[s]) and not stack["b"][slot, s * 16:s * 16 + 16, r:].any()


def test_another_scale_for_what_a_slot_holds():
    stack, pairs = _stack()
    adapters.load(stack, 1, *_own(stack, 1), 3.0)
    _holds(stack, 1, *pairs[1], 3.0)
    _holds(stack, 0, *pairs[0], 0.5)


def test_slices_exchanged():
    stack, pairs = _stack()
    adapters.load(stack, 1, *_own(stack, 1, order=(1, 0)), 1.0)
    a, b = pairs[1]
    _holds(stack, 1, a[::-1], b[::-1], 1.0)


@pytest.mark.parametrize("name", ["a", "b"])
def test_one_of_the_matrices(name):
    stack, pairs = _stack()
    a, b = _own(stack, 0)
    new = [t.clone() * 2 for t in (b if name == "a" else a)]
    adapters.load(stack, 0, a if name == "a" else new, new if name == "a" else b, 1.0)
    _holds(stack, 0, pairs[0][0] if name == "a" else new, new if name == "a" else pairs[0][1], 1.0)


def test_fewer_ranks_and_another_slot():
    stack, pairs = _stack()
    adapters.load(stack, 2, *_own(stack, 0), 2.0)
    _holds(stack, 2, *pairs[0], 2.0)
    _holds(stack, 0, *pairs[0], 0.5)
    adapters.load(stack, 0, *_own(stack, 0, ranks=(2, 3)), 2.0)
    a, b = pairs[0]
    _holds(stack, 0, [a[0][:2], a[1][:3]], [b[0][:, :2], b[1][:, :3]], 2.0)
