"""Few rows an expert and more tiles than CTAs that run together: the k-steps of all tiles are dealt out in equal shares, and a tile
cut between two CTAs is summed by the one that comes second.  Whole numbers: the bits are those of the plain form, tolerance
none (the MLP's is derived in test_gpu_experts.py)."""

import pytest
import torch

from test_gpu_experts import _check_mlp, _linear, _quantise, _rows, _stack

pytestmark = pytest.mark.gpu

K, BLOCKS = 2816, 300     # 300 channel blocks on 2 x 148 CTAs: one round and a hundredth


@pytest.fixture(scope="module")
def moe():
    from liquidgemm_b200 import moe as _moe
    return _moe


@pytest.fixture(scope="module")
def stack(moe):
    return _stack(moe, 2, 128 * BLOCKS - 40, K, True, 5)     # the last block has 88 channels


def _choices(how, T):
    ids = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    if how == "two":
        ids[::2] = 1
    elif how == "other":
        ids[:] = 1
    elif how == "holes":
        ids[1::2] = -1
    elif how == "none":
        ids[:] = 2
    return ids


@pytest.mark.parametrize("T", [1, 2, 9, 16, 17, 20])
@pytest.mark.parametrize("how", ["one", "two", "other", "holes", "none"])
def test_bits(moe, stack, T, how):
    layer, q, s1 = stack
    ids = _choices(how, T)
    for dtype in (torch.bfloat16, torch.float32):
        x = _rows((T, K), dtype, T)
        xq, scale = _quantise(x)
        want = _linear(xq, scale, ids, q, s1, False, dtype)
        for _ in range(4):       # which of two CTAs comes second changes from call to call
            assert torch.equal(moe.experts_linear(x, ids, layer), want)


def test_replayed_with_other_choices(moe, stack):
    """One captured call: dealt out evenly or not, as the ids of each replay have it; the counts of the joins start afresh."""
    layer, q, s1 = stack
    T = 20
    x, ids = _rows((T, K), torch.bfloat16, 1), _choices("one", T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moe.experts_linear(x, ids, layer)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moe.experts_linear(x, ids, layer)
    for n, how in enumerate(("one", "two", "none", "holes", "other", "one")):
        ids.copy_(_choices(how, T))
        x.copy_(_rows((T, K), torch.bfloat16, 10 + n))
        y.fill_(7.0)
        graph.replay()
        xq, scale = _quantise(x)
        assert torch.equal(y, _linear(xq, scale, ids, q, s1, False, torch.bfloat16))


def test_two_streams(moe, stack):
    layer, q, s1 = stack
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [_rows((9, K), torch.bfloat16, 30 + i) for i in range(2)]
    ids = _choices("two", 9)
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i].append(moe.experts_linear(xs[i], ids, layer))
    torch.cuda.synchronize()
    for i in range(2):
        xq, scale = _quantise(xs[i])
        want = _linear(xq, scale, ids, q, s1, False, torch.bfloat16)
        assert all(torch.equal(y, want) for y in out[i])


@pytest.mark.parametrize("T,how", [(1, "random"), (4, "random"), (10, "one")])
def test_mlp(moe, T, how):
    # 2 x 160 blocks of 22 k-steps in the first product
    _check_mlp(moe, T, 2, 2, 2816, 10240, True, how, torch.bfloat16, T)


def test_many_experts(moe):
    """More pairs than the placing kernel sorts by itself; every tile is another expert's."""
    T, k, E, K = 300, 8, 300, 3584
    layer, q, s1 = _stack(moe, E, 128, K, True, 8)
    x = _rows((T, K), torch.float16, 3)
    xq, scale = _quantise(x)
    ids = torch.stack([(torch.arange(E, device="cuda") * 7 + 41 * j) % E for j in range(k)], dim=1).to(torch.int32)   # eight rows each
    want = _linear(xq, scale, ids, q, s1, False, torch.float16)
    for _ in range(3):
        assert torch.equal(moe.experts_linear(x, ids, layer), want)
