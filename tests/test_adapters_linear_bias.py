"""The bias of a linear with adapters: [N] in the output type for both weight kinds, refused before anything runs otherwise."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from liquidgemm_b200 import adapters

N, K = 256, 512


def _bias(shape, dtype, device="cuda"):
    return torch.zeros(shape, dtype=dtype, device=device)


BAD = [((N,), torch.float32, None), ((N,), torch.float16, None), ((N,), torch.bfloat16, torch.float32), ((1,), torch.bfloat16, None),
       ((), torch.bfloat16, None), ((N - 8,), torch.bfloat16, None), ((3, N), torch.bfloat16, None), ((3, 1), torch.bfloat16, None)]


@pytest.mark.parametrize("w4", [True, False])
@pytest.mark.parametrize("shape,dtype,out_dtype", BAD)
def test_refused(shape, dtype, out_dtype, w4):
    with FakeTensorMode():
        layer = {"s1": torch.ones(N, device="cuda"), "N": N, "K": K}
        if w4:
            layer.update(rs=torch.zeros(N // 128, K // 128, 8704, dtype=torch.uint8, device="cuda"),
                         s_u8=torch.zeros(N, K // 64, dtype=torch.uint8, device="cuda"),
                         offset_a=torch.zeros(N, K // 64, dtype=torch.uint8, device="cuda"))
        else:
            layer["w_i8"] = torch.zeros(N, K, dtype=torch.int8, device="cuda")
        stack = adapters.make_stack(2, 8, K, N)
        x, ids = torch.zeros(3, K, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
        with pytest.raises(RuntimeError, match="bias must be"):
            adapters.linear(x, layer, stack, ids, bias=_bias(shape, dtype), out_dtype=out_dtype)
        with pytest.raises(RuntimeError, match="bias must be"):
            adapters.linear(x, layer, stack, ids, bias=_bias((N,), torch.bfloat16, "cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("w4", [True, False])
def test_both_weight_kinds(w4):
    """The same answers and refusals; a bias of [1, N] or with a step is N elements like any other."""
    from liquidgemm_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = (torch.randn(N, K, device="cuda", generator=gen) * 0.05).to(torch.bfloat16)
    q, blob = ops.quantize_weight_cuda(w, want_codes=True, want_blob=True)
    layer = {"s1": q.s1, "N": N, "K": K}
    layer.update({"rs": blob, "s_u8": q.s_u8, "offset_a": q.offset_a} if w4 else {"w_i8": ops.dequant_weight_i8(q)})
    stack = adapters.make_stack(2, 8, K, N)
    adapters.load(stack, 1, torch.randn(8, K, device="cuda", generator=gen) * 0.05, torch.randn(N, 8, device="cuda", generator=gen))
    for T in (1, 5, 200):
        x = torch.randn(T, K, device="cuda", generator=gen).to(torch.bfloat16)
        ids = torch.arange(T, device="cuda") % 3 - 1
        rows, scales = torch.ops.liquidgemm.quant_per_token(x)
        for out_dtype, code in ((torch.bfloat16, 0), (torch.float32, 2)):
            wide = torch.randn(2 * N, device="cuda", generator=gen).to(out_dtype)
            keep = wide.clone()
            y = torch.ops.liquidgemm.w4a8_linear_bias(rows, blob, scales, q.s1, None, N, K, code) + wide[::2]
            want = adapters.add(y, x, stack, ids)
            for bias in (wide[::2], wide[::2].contiguous()[None]):
                got = adapters.linear(x, layer, stack, ids, bias=bias, out_dtype=out_dtype)
                assert got.dtype == out_dtype and torch.equal(got, want)
            assert torch.equal(wide, keep)
        for shape, dtype, out_dtype in BAD:
            with pytest.raises(RuntimeError, match="bias must be"):
                adapters.linear(x, layer, stack, ids, bias=_bias(shape, dtype), out_dtype=out_dtype)
    assert adapters.linear(x[:0], layer, stack, ids[:0], bias=wide[::2].to(torch.bfloat16)).shape == (0, N)
