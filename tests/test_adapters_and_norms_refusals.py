"""What the adapters' and the norms' entry points refuse before anything reaches a device: the C calls by status code, the Python
checks by message.  The pointers below are never followed."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from liquidgemm_b200 import adapters, norms
from liquidgemm_b200._lib import lib

BAD_ARG, SHAPE, WORKSPACE = -1, -2, -3
P, BIG = 4096, 1 << 50


def _add(x=P, dtype=0, ldx=256, a=P, b=P, ranks=P, scales=P, ids=P, ids_64=0, y=P, ldy=128, y_f32=0, out=P, ldo=128, T=4, K=256, L=3,
         rank=16, widths=(64, 64), scratch=P, nbytes=BIG):
    w = None if widths is None else (ctypes.c_int * len(widths))(*widths)
    return lib.lq_adapters_add(x, dtype, ldx, a, b, ranks, scales, ids, ids_64, y, ldy, y_f32, out, ldo, T, K, L, rank, w,
                               0 if widths is None else len(widths), scratch, nbytes, None)


@pytest.mark.parametrize("change", [dict(x=None), dict(a=None), dict(b=None), dict(ranks=None), dict(scales=None), dict(ids=None),
                                    dict(y=None), dict(out=None), dict(widths=None), dict(dtype=2), dict(dtype=-1), dict(T=0), dict(K=0),
                                    dict(L=0), dict(rank=0), dict(widths=()), dict(widths=(64, 0)), dict(widths=(-8, 136))])
def test_add_bad_arguments(change):
    assert _add(**change) == BAD_ARG


@pytest.mark.parametrize("change", [dict(K=252), dict(rank=12), dict(rank=264), dict(L=4097), dict(T=(1 << 24) + 1), dict(K=(1 << 20) + 8),
                                    dict(widths=(8,) * 9), dict(widths=(64, 60)), dict(widths=(1 << 25, 64)), dict(x=P + 2), dict(a=P + 8),
                                    dict(b=P + 4), dict(y=P + 8), dict(out=P + 2), dict(ldx=252), dict(ldx=-256), dict(ldy=132),
                                    dict(ldo=132), dict(ldy=120), dict(ldo=64), dict(y_f32=1, ldy=130), dict(ldy=-128)])
def test_add_bad_shapes(change):
    assert _add(**change) == SHAPE


def test_add_scratch():
    need = lib.lq_adapters_scratch_bytes(4, 256, 3, 16, 2)
    assert need >= 4 * 32 * 4
    for scratch, nbytes in ((None, BIG), (P, need - 1), (P + 8, BIG)):
        assert _add(scratch=scratch, nbytes=nbytes) == WORKSPACE
    for bad in ((0, 256, 3, 16, 2), (4, 250, 3, 16, 2), (4, 256, 4097, 16, 2), (4, 256, 3, 15, 2), (4, 256, 3, 16, 9), (4, 256, 3, 264, 2)):
        assert lib.lq_adapters_scratch_bytes(*bad) == 0


def _norm(x=P, x_dtype=0, residual=P, stream_dtype=0, gate=None, gate_dtype=0, gate_step=1, weight=P, weight_dtype=0, post=None,
          post_dtype=0, z=P, q=None, q_scale=None, h=P, rows=4, inner=4, H=256, eps=1e-6):
    return lib.lq_block_norm(x, x_dtype, 0, 256, residual, stream_dtype, 0, 256, gate, gate_dtype, 0, 256, gate_step, weight,
                             weight_dtype, post, post_dtype, z, q, q_scale, h, rows, inner, H, eps, 1.0, 1.0, 0.0, None)


@pytest.mark.parametrize("change", [dict(x=None), dict(z=None), dict(q=P), dict(q=P, z=None), dict(q_scale=P), dict(rows=0), dict(inner=0),
                                    dict(H=0), dict(x_dtype=3), dict(x_dtype=-1), dict(stream_dtype=1), dict(residual=None, stream_dtype=2),
                                    dict(x_dtype=2), dict(weight_dtype=1), dict(gate=P, gate_dtype=1), dict(post=P, post_dtype=1),
                                    dict(gate=P, gate_step=2), dict(eps=-1.0), dict(eps=float("nan"))])
def test_norm_bad_arguments(change):
    assert _norm(**change) == BAD_ARG


def test_norm_too_wide():
    assert _norm(H=32769) == SHAPE


def test_stack_sizes():
    stack = adapters.make_stack(3, 12, 64, (16, 24), device="cpu")
    assert stack["a"].shape == (3, 2, 16, 64) and stack["b"].shape == (3, 40, 16) and stack["N"] == 40
    assert stack["rank"].tolist() == [[0, 0]] * 3
    for bad in ((0, 8, 64, 8), (4097, 8, 64, 8), (1, 0, 64, 8), (1, 257, 64, 8), (1, 8, 60, 8), (1, 8, 0, 8), (1, 8, 64, 12),
                (1, 8, 64, (8,) * 9), (1, 8, 64, ()), (1, 8, 64, (8, 0)), (1, 8, 1 << 21, 8)):
        with pytest.raises(RuntimeError):
            adapters.make_stack(*bad, device="cpu")
    with pytest.raises(RuntimeError, match="dtype"):
        adapters.make_stack(1, 8, 64, 8, dtype=torch.float32, device="cpu")


def test_load_and_unload():
    stack = adapters.make_stack(2, 12, 64, (16, 24), device="cpu")
    a, b = [torch.randn(5, 64), torch.randn(12, 64)], [torch.randn(16, 5), torch.randn(24, 12)]
    adapters.load(stack, 1, a, b, 0.5)
    assert stack["rank"].tolist() == [[0, 0], [5, 12]] and stack["scale"].tolist() == [0.0, 0.5]
    assert torch.equal(stack["a"][1, 0, :5], a[0].to(torch.bfloat16)) and not stack["a"][1, 0, 5:].any()
    assert torch.equal(stack["b"][1, 16:, :12], b[1].to(torch.bfloat16)) and not stack["b"][1, :16, 5:].any()
    adapters.load(stack, 1, [a[0], None], [b[0], None], 1.0)   # nothing of the adapter before is left
    assert stack["rank"].tolist() == [[0, 0], [5, 0]] and not stack["a"][1, 1].any() and not stack["b"][1, 16:].any()
    adapters.unload(stack, 1)
    assert not stack["rank"].any()
    for slot, aa, bb in ((2, a, b), (-1, a, b), (0, a[:1], b[:1]), (0, a, b[:1]), (0, [a[0], None], b), (0, b, a),
                         (0, [torch.randn(17, 64), a[1]], [torch.randn(16, 17), b[1]]), (0, [torch.randn(5, 56), a[1]], b)):
        with pytest.raises(RuntimeError):
            adapters.load(stack, slot, aa, bb)
    assert not stack["rank"].any()


def test_nothing_runs_on_the_cpu():
    stack = adapters.make_stack(2, 8, 64, 16, device="cpu")
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        adapters.add(torch.zeros(3, 16, dtype=torch.bfloat16), x, stack, torch.zeros(3, dtype=torch.int32))
    with pytest.raises((RuntimeError, NotImplementedError)):
        norms.block_norm(x, None)
    with pytest.raises(RuntimeError, match="another linear"):
        adapters.linear(x, {"N": 24, "K": 64}, stack, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="bf16 or fp16"):
        adapters.linear(x.float(), {"N": 16, "K": 64}, stack, torch.zeros(3, dtype=torch.int32))


def _cuda(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _like_stack(L=2, S=1, r=8, K=64, N=16, dtype=torch.bfloat16):
    return dict(a=_cuda(L, S, r, K, dtype=dtype), b=_cuda(L, N, r, dtype=dtype), rank=_cuda(L, S, dtype=torch.int32),
                scale=_cuda(L, dtype=torch.float32), widths=[N])


@pytest.mark.parametrize("change,match", [
    (dict(x=(3, 64, torch.float32)), "bf16 or fp16"), (dict(x=(3, 64, torch.float16)), "type of x"), (dict(x=(3, 56, torch.bfloat16)), "x must be"),
    (dict(y=(3, 24, torch.bfloat16)), "y must be"), (dict(y=(4, 16, torch.bfloat16)), "y must be"), (dict(y=(3, 16, torch.float16)), "y must be"),
    (dict(ids=(4, torch.int32)), "ids must"), (dict(ids=(3, torch.int16)), "ids must"), (dict(widths=[8]), "widths"), (dict(widths=[8, 8]), "widths"),
    (dict(widths=[12, 4]), "widths"), (dict(r=12), "multiples of 8"), (dict(K=60, x=(3, 60, torch.bfloat16)), "multiples of 8"), (dict(rank=(2, 2)), "rank must"),
])
def test_add_python_checks(change, match):
    with FakeTensorMode():
        args = _like_stack(r=change.get("r", 8), K=change.get("K", 64))
        if "rank" in change:
            args["rank"] = _cuda(*change["rank"], dtype=torch.int32)
        *shape, dtype = change.get("x", (3, 64, torch.bfloat16))
        x = _cuda(*shape, dtype=dtype)
        *shape, dtype = change.get("y", (3, 16, torch.bfloat16))
        y = _cuda(*shape, dtype=dtype)
        n, dtype = change.get("ids", (3, torch.int32))
        with pytest.raises(RuntimeError, match=match):
            adapters._run(y, x, args["a"], args["b"], args["rank"], args["scale"], _cuda(n, dtype=dtype),
                          change.get("widths", args["widths"]), False)


@pytest.mark.parametrize("change,match", [
    (dict(shape=(64,)), "x must be"), (dict(shape=(2, 3, 4, 64)), "x must be"), (dict(dtype=torch.float64), "x must be"),
    (dict(shape=(3, 0)), "H must be"), (dict(shape=(3, 32769)), "H must be"), (dict(weight=(63,)), "weight must be"),
    (dict(weight=(64,), weight_dtype=torch.float16), "weight must be"), (dict(post=(1, 64)), "post_weight must be"),
    (dict(residual=(3, 63)), "residual must be"), (dict(residual=(3, 64), residual_dtype=torch.float16), "residual must be"),
    (dict(gate=(2, 64)), "does not broadcast"), (dict(gate=(1, 3, 64)), "does not broadcast"), (dict(gate=(3, 64), gate_dtype=torch.float16), "gate must be"),
    (dict(eps=-1e-6), "eps"),
])
def test_norm_python_checks(change, match):
    with FakeTensorMode():
        def made(name):
            return _cuda(*change[name], dtype=change.get(name + "_dtype", torch.bfloat16)) if name in change else None
        x = _cuda(*change.get("shape", (3, 64)), dtype=change.get("dtype", torch.bfloat16))
        with pytest.raises(RuntimeError, match=match):
            norms._block_norm(x, made("weight"), made("residual"), made("post"), made("gate"), change.get("eps", 1e-6), 1.0, 1.0, 0.0, True)


def test_traced_shapes():
    with FakeTensorMode():
        args = _like_stack()
        y = torch.ops.liquidgemm.adapters_add(_cuda(3, 16, dtype=torch.float32), _cuda(3, 64), args["a"], args["b"], args["rank"], args["scale"],
                                              _cuda(3, dtype=torch.int64), args["widths"])
        assert y.shape == (3, 16) and y.dtype == torch.float32
        for quantize in (False, True):
            z, scale, h = torch.ops.liquidgemm.block_norm(_cuda(2, 3, 64), None, _cuda(2, 3, 64, dtype=torch.float32), None, None, 1e-6, 1.0, 1.0,
                                                          0.0, quantize)
            assert z.shape == (2, 3, 64) and z.dtype == (torch.int8 if quantize else torch.bfloat16)
            assert scale.shape == ((2, 3) if quantize else (0,)) and h.dtype == torch.float32 and h.shape == (2, 3, 64)
        assert norms.block_norm(_cuda(3, 64), None)[0].shape == (3, 64)
