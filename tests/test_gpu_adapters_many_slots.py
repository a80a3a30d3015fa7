"""Stacks of up to 4096 slots on the path of many rows: what the plan of a batch keeps for each slot passes 48 KB of shared memory
between 4073 and 4095 of them, static and dynamic together."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_CALLS = """
import torch
from liquidgemm_b200 import adapters

T, K, N, R = 200, 8, 8, 8
for L in {slots}:
    gen = torch.Generator(device="cuda").manual_seed(L)
    stack = adapters.make_stack(L, R, K, N, dtype=torch.float16)
    small = lambda *shape: torch.randint(-2, 3, shape, device="cuda", generator=gen).to(torch.float16)
    stack["a"].copy_(small(L, 1, R, K))
    stack["b"].copy_(small(L, N, R))
    stack["rank"].fill_(R)
    stack["scale"].fill_(1.0)
    x, y = small(T, K), small(T, N)
    ids = torch.randint(-1, L + 1, (T,), device="cuda", generator=gen)
    ids[0], ids[1] = 0, L - 1
    got = adapters.add(y, x, stack, ids)
    torch.cuda.synchronize()
    mine, want = (ids >= 0) & (ids < L), y.double()
    l = ids[mine]
    v = (stack["a"][l, 0].double() @ x[mine].double()[:, :, None])
    want[mine] += (stack["b"][l].double() @ v)[:, :, 0]
    assert torch.equal(got.double(), want), L   # whole numbers up to 2 + 8 * 2 * 8 * 4: exact on the way and in fp16
print("done")
"""


@pytest.mark.parametrize("slots", [(4073, 4074, 4094, 4095, 4096), (4096, 1, 4094), (4080,)])
def test_as_many_slots_as_a_stack_may_have(slots):
    """In processes of their own: a kernel's limit of shared memory, once raised, would hide that a smaller call needs it too."""
    got = subprocess.run([sys.executable, "-c", _CALLS.format(slots=slots)], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert got.returncode == 0 and got.stdout.strip() == "done", got.stderr[-2000:]
