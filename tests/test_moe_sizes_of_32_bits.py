"""Sizes of the expert layers that 32 bits do not hold are refused, by the C calls and in Python, before anything reaches a device."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from liquidgemm_b200 import moe
from liquidgemm_b200._lib import lib

SHAPE, P, BIG = -2, 4096, 1 << 50


@pytest.mark.parametrize("N", [1 << 30, (1 << 31) - 128])
def test_rows_of_outputs(N):
    for kind in (0, 1):
        assert lib.lq_experts_linear_scratch_bytes(2, 1, 1, N, 128, kind) == 0
        assert lib.lq_experts_linear(P, 0, None, 0, P, P, kind, P, P, 2, 2, 1, 1, N, 128, P, BIG, None) == SHAPE
    assert lib.lq_experts_linear_scratch_bytes(2, 1, 1, (1 << 30) - 128, 128, 0) > 0


def test_the_same_in_python():
    with FakeTensorMode():
        w, s1 = torch.empty(1, dtype=torch.uint8, device="cuda"), torch.empty(1, 1 << 30, device="cuda")
        with pytest.raises(RuntimeError, match="2\\^30"):
            moe._weights(w, s1, 1 << 30, 128, "w")


@pytest.mark.parametrize("T", [1 << 31, (1 << 32) + 5])
def test_tokens_of_the_router(T):
    with FakeTensorMode():
        logits = torch.empty(T, 2, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(RuntimeError, match="2\\^31"):
            moe._moe_route(logits, None, 1, 0, 1, 1, 0, True, 1.0)
