"""What the mixture-of-experts entry points refuse before anything reaches a device: the C calls by status code, the Python
checks by message.  The pointers below are never followed."""

import pytest
import torch

from liquidgemm_b200 import moe
from liquidgemm_b200._lib import lib

BAD_ARG, SHAPE, WORKSPACE = -1, -2, -3
P, BIG = 4096, 1 << 50


def _route(logits=P, dtype=0, bias=None, w=P, ids=P, T=4, E=64, topk=4, scoring=0, n_group=1, topk_group=1, group_score=0):
    return lib.lq_moe_route(logits, dtype, bias, w, ids, T, E, topk, scoring, n_group, topk_group, group_score, 1, 1.0, None)


@pytest.mark.parametrize("change", [dict(logits=None), dict(w=None), dict(ids=None), dict(dtype=3), dict(dtype=-1), dict(T=0),
                                    dict(E=0), dict(topk=0), dict(scoring=2), dict(n_group=0), dict(topk_group=0), dict(group_score=2)])
def test_route_bad_arguments(change):
    assert _route(**change) == BAD_ARG


@pytest.mark.parametrize("change", [dict(E=513), dict(topk=33), dict(n_group=3), dict(n_group=8, topk_group=9),
                                    dict(n_group=32, topk_group=1), dict(E=3)])
def test_route_bad_shapes(change):
    assert _route(**change) == SHAPE


def _linear(x=P, x_dtype=0, x_scale=None, ids=P, w=P, kind=0, s1=P, y=P, out=0, T=4, topk=2, E=8, N=256, K=256, scratch=P, nbytes=BIG):
    return lib.lq_experts_linear(x, x_dtype, x_scale, 0, ids, w, kind, s1, y, out, T, topk, E, N, K, scratch, nbytes, None)


@pytest.mark.parametrize("change", [dict(x=None), dict(ids=None), dict(w=None), dict(s1=None), dict(y=None), dict(x_dtype=4),
                                    dict(x_dtype=3), dict(x_scale=P), dict(kind=2), dict(out=3), dict(T=0), dict(topk=0), dict(E=0),
                                    dict(N=0), dict(K=0)])
def test_linear_bad_arguments(change):
    assert _linear(**change) == BAD_ARG


@pytest.mark.parametrize("change", [dict(K=192), dict(topk=33), dict(E=513), dict(T=1 << 24), dict(x=P + 8), dict(w=P + 4),
                                    dict(E=512, N=1 << 23), dict(K=131072)])
def test_linear_bad_shapes(change):
    assert _linear(**change) == SHAPE


@pytest.mark.parametrize("kind", [0, 1])
def test_linear_scratch(kind):
    need = lib.lq_experts_linear_scratch_bytes(4, 2, 8, 256, 256, kind)
    assert need > 4 * 2 * 256
    for scratch, nbytes in ((None, BIG), (P, need - 1), (P + 8, BIG)):
        assert _linear(kind=kind, scratch=scratch, nbytes=nbytes) == WORKSPACE
    for bad in ((0, 2, 8, 256, 256), (4, 33, 8, 256, 256), (4, 2, 513, 256, 256), (4, 2, 8, 256, 200), (4, 2, 8, 0, 256)):
        assert lib.lq_experts_linear_scratch_bytes(*bad, kind) == 0
    assert lib.lq_experts_linear_scratch_bytes(4, 2, 8, 256, 256, 2) == 0


def _mlp(x=P, x_dtype=0, weights=P, ids=P, w13=P, s13=P, w2=P, s2=P, kind=0, y=P, out=0, T=4, topk=2, E=8, H=256, inner=256,
         scratch=P, nbytes=BIG):
    return lib.lq_experts_mlp(x, x_dtype, weights, ids, w13, s13, w2, s2, kind, y, out, T, topk, E, H, inner, scratch, nbytes, None)


@pytest.mark.parametrize("change", [dict(x=None), dict(weights=None), dict(ids=None), dict(w13=None), dict(s13=None), dict(w2=None),
                                    dict(s2=None), dict(y=None), dict(x_dtype=3), dict(kind=-1), dict(out=3), dict(T=0), dict(E=0)])
def test_mlp_bad_arguments(change):
    assert _mlp(**change) == BAD_ARG


@pytest.mark.parametrize("change", [dict(H=200), dict(inner=192), dict(H=131072), dict(inner=131072), dict(topk=33), dict(E=513), dict(T=1 << 24), dict(inner=1 << 30),
                                    dict(x=P + 8), dict(w13=P + 8), dict(w2=P + 8), dict(s13=P + 4), dict(s2=P + 4),
                                    dict(y=P + 8)])
def test_mlp_bad_shapes(change):
    assert _mlp(**change) == SHAPE


def test_mlp_scratch():
    need = lib.lq_experts_mlp_scratch_bytes(4, 2, 8, 256, 384, 0)
    assert need > 4 * 2 * (256 + 384)
    for scratch, nbytes in ((None, BIG), (P, need - 1), (P + 8, BIG)):
        assert _mlp(inner=384, scratch=scratch, nbytes=nbytes) == WORKSPACE
    assert lib.lq_experts_mlp_scratch_bytes(4, 2, 8, 256, 100, 0) == 0 and lib.lq_experts_mlp_scratch_bytes(4, 2, 8, 256, 384, 2) == 0


# ---- Python checks that need no device -----------------------------------------------------------------------------

def test_python_checks_on_cpu_tensors():
    """CPU tensors reach no kernel, directly or through the operators."""
    x, ids = torch.zeros(4, 256), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        moe._moe_route(x, None, 2, 0, 1, 1, 0, True, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        moe.quantize_experts(torch.zeros(2, 128, 128))
    with pytest.raises(RuntimeError, match="CUDA"):
        moe._experts_linear(x, None, ids, torch.zeros(1, dtype=torch.uint8), torch.zeros(8, 128), 128, 256, 0)
    with pytest.raises((RuntimeError, NotImplementedError)):
        moe.route(x, 2)


def test_python_checks_of_names_and_layers():
    x, ids = torch.zeros(4, 256), torch.zeros(4, 2, dtype=torch.int32)
    gated, plain = {"gated": True, "w": x, "s1": x, "N": 2, "K": 2}, {"gated": False, "w": x, "s1": x, "N": 2, "K": 2}
    with pytest.raises(RuntimeError, match="scoring"):
        moe.route(x, 2, scoring="relu")
    with pytest.raises(RuntimeError, match="group_score"):
        moe.route(x, 2, group_score="mean")
    with pytest.raises(RuntimeError, match="gated"):
        moe.experts_linear(x, ids, gated)
    with pytest.raises(RuntimeError, match="gated"):
        moe.experts_mlp(x, x, ids, plain, plain)
    with pytest.raises(RuntimeError, match="out_dtype"):
        moe.experts_linear(x, ids, plain, out_dtype=torch.float64)


def test_fake_kernels_give_the_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        logits = torch.empty(5, 16, device="cuda")
        w, ids = torch.ops.liquidgemm.moe_route(logits, None, 3, 0, 1, 1, 0, True, 1.0)
        assert w.shape == ids.shape == (5, 3) and w.dtype == torch.float32 and ids.dtype == torch.int32
        x = torch.empty(5, 256, device="cuda", dtype=torch.bfloat16)
        q = torch.empty(16, 2, 2, moe.TILE_BYTES, dtype=torch.uint8, device="cuda")
        s = torch.empty(16, 256, device="cuda")
        y = torch.ops.liquidgemm.experts_linear(x, None, ids, q, s, 256, 256, 1)
        assert y.shape == (5, 3, 256) and y.dtype == torch.float16
        z = torch.ops.liquidgemm.experts_mlp(x, w, ids, q, s, q, s, 0)
        assert z.shape == (5, 256) and z.dtype == torch.bfloat16
        # the entry points themselves, on tensors that are not ordinary ones
        layer = {"w": q, "s1": s, "N": 256, "K": 256, "gated": False}
        w, ids = moe.route(logits, 3, scoring="sigmoid")
        assert w.shape == (5, 3)
        assert moe.experts_linear(x, ids, layer).shape == (5, 3, 256)
        assert moe.experts_mlp(x, w, ids, dict(layer, gated=True), layer).shape == (5, 256)
