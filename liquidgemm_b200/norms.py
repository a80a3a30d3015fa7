"""Norms around a block, fused with its gate, its scales and the residual, in front of the linears.

One pass over the rows of a block's output ``x``:

    ``p = x * (mean(x^2) + eps)^-1/2 * (post_weight + weight_offset)``      (``x`` without ``post_weight``)
    ``h = residual_scale * residual + scale * gate * p``                    (the new residual stream)
    ``z = h * (mean(h^2) + eps)^-1/2 * (weight + weight_offset)``           (what the next block reads)

* :func:`block_norm`        ``z`` in the type of ``x``;
* :func:`block_norm_quant`  ``z`` as INT8 rows with one scale each, as ``torch.ops.liquidgemm.w4a8_wgmma_rs_fused``,
                            ``w4a8_linear_bias`` and ``i8_gemm_scaled`` take them.

The operator behind both is ``torch.ops.liquidgemm.block_norm``, with a fake kernel.  Like the dense operators it validates its
arguments in Python, allocates its outputs with torch, enqueues on the current stream of the tensors' device, synchronises nothing and can be
captured into a CUDA graph.  Inference only.

The reference has no counterpart: its linears quantise what a norm has rounded to 16 bits (liquidgemm/vllm_plugin.py:183-196).
Like :mod:`liquidgemm_b200.ops` this module is not imported by the package ``__init__``.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._lib import check, lib
from .moe import _plain_call, _refuse, _same_device
from .ops import _DTYPE_CODES, _dev_ctx, _impl, _libdef

MAX_WIDTH = 32768

_libdef.define("block_norm(Tensor x, Tensor? weight, Tensor? residual, Tensor? post_weight, Tensor? gate, float eps, float scale, "
               "float residual_scale, float weight_offset, bool quantize) -> (Tensor, Tensor, Tensor)")


def _joins(residual, post_weight, gate, scale) -> bool:
    return residual is not None or post_weight is not None or gate is not None or scale != 1.0


@torch.library.register_fake("liquidgemm::block_norm")
def _f_norm(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, quantize):
    z = x.new_empty(x.shape, dtype=torch.int8 if quantize else x.dtype)
    q_scale = x.new_empty(x.shape[:-1] if quantize else (0,), dtype=torch.float32)
    stream = x if residual is None else residual
    return z, q_scale, stream.new_empty(x.shape if _joins(residual, post_weight, gate, scale) else (0,))


def _strides(t: torch.Tensor, nd: int):
    """(t, outer, inner) of [T, H] or [B, S, H] rows whose elements are neighbours."""
    strides = t.stride()
    if strides[-1] != 1 and t.shape[-1] != 1:
        t = t.contiguous()
        strides = t.stride()
    return (t, 0, strides[0]) if nd == 2 else (t, strides[0], strides[1])


def _vector(w, name, H, dtype, device):
    w.is_cuda and w.dim() == 1 and w.shape[0] == H and (w.dtype is dtype or w.dtype is torch.float32) or \
        _refuse(f"{name} must be a CUDA [{H}] tensor in the type of x or float32")
    w.device == device or _refuse(f"{name} must be on the device of x, {device}")
    return w if w.is_contiguous() else w.contiguous()


def _run(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, quantize):
    """(z, scales or None, h or None): the checks of a call cost the host more than a small one's kernel takes, so each value is asked for once."""
    dtype, shape, device = x.dtype, x.shape, x.device
    code = _DTYPE_CODES.get(dtype)
    nd = len(shape)
    code is not None and (nd == 2 or nd == 3) and x.is_cuda or _refuse("x must be a CUDA [T, H] or [B, S, H] tensor of bf16, fp16 or fp32")
    H = shape[-1]
    1 <= H <= MAX_WIDTH or _refuse(f"H must be 1..{MAX_WIDTH}")
    rows = shape[0] if nd == 2 else shape[0] * shape[1]
    rows < 1 << 31 or _refuse("fewer than 2^31 rows required")
    eps >= 0.0 or _refuse("eps must not be negative")
    joins = scale != 1.0
    stream, stream_code = dtype, code
    r = g = w = p = None
    ro = ri = go = gi = step = g_code = w_code = p_code = 0
    if residual is not None:
        joins, stream = True, residual.dtype
        residual.is_cuda and residual.shape == shape and (stream is dtype or stream is torch.float32) or \
            _refuse("residual must be a CUDA tensor of x's shape, in the type of x or float32")
        residual.device == device or _same_device(x, residual)
        stream_code = _DTYPE_CODES[stream]
        residual, ro, ri = _strides(residual, nd)
        r = residual.data_ptr()
    if weight is not None:
        weight = _vector(weight, "weight", H, dtype, device)
        w, w_code = weight.data_ptr(), _DTYPE_CODES[weight.dtype]
    if post_weight is not None:
        joins = True
        post_weight = _vector(post_weight, "post_weight", H, dtype, device)
        p, p_code = post_weight.data_ptr(), _DTYPE_CODES[post_weight.dtype]
    if gate is not None:
        joins = True
        gate.is_cuda and (gate.dtype is dtype or gate.dtype is torch.float32) or \
            _refuse("gate must be a CUDA tensor in the type of x or float32")
        gate.dim() <= nd and all(a == 1 or a == n for a, n in zip(reversed(gate.shape), reversed(shape))) or \
            _refuse(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
        gate.device == device or _same_device(x, gate)
        per_row = gate.dim() == 0 or (gate.shape[-1] == 1 and H > 1)
        if not per_row and H > 1 and gate.stride(-1) != 1:
            gate = gate.contiguous()
        wide = gate.expand(shape)
        go, gi = (wide.stride(0), wide.stride(1)) if nd == 3 else (0, wide.stride(0))
        g, g_code, step = gate.data_ptr(), _DTYPE_CODES[gate.dtype], 0 if per_row else 1
    z = torch.empty(shape, dtype=torch.int8 if quantize else dtype, device=device)
    q_scale = torch.empty(shape[:-1], dtype=torch.float32, device=device) if quantize else None
    h = torch.empty(shape, dtype=stream, device=device) if joins else None
    if rows == 0:
        return z, q_scale, h
    x, xo, xi = _strides(x, nd)
    pz = z.data_ptr()
    with _dev_ctx(x):
        code = lib.lq_block_norm(x.data_ptr(), code, xo, xi, r, stream_code, ro, ri, g, g_code, go, gi, step, w, w_code, p, p_code,
                                 None if quantize else pz, pz if quantize else None, q_scale.data_ptr() if quantize else None,
                                 h.data_ptr() if joins else None, rows, rows if nd == 2 else shape[1], H, eps, scale,
                                 residual_scale, weight_offset, torch._C._cuda_getCurrentRawStream(device.index))
    if code:
        check(code, "block_norm")
    return z, q_scale, h


def _block_norm(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, quantize):
    z, q_scale, h = _run(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, quantize)
    stream = x if residual is None else residual
    return z, x.new_empty(0, dtype=torch.float32) if q_scale is None else q_scale, stream.new_empty(0) if h is None else h


_impl.impl("block_norm", _block_norm)


# --------------------------------------------------------------------------------------
# Python entry points
# --------------------------------------------------------------------------------------

def _call(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, quantize):
    args = (x, weight, residual, post_weight, gate, float(eps), float(scale), float(residual_scale), float(weight_offset), quantize)
    if _plain_call(x, weight, residual, post_weight, gate):
        z, q_scale, h = _run(*args)
        return z, q_scale, x if h is None else h
    z, q_scale, h = torch.ops.liquidgemm.block_norm(*args)
    return z, q_scale, h if _joins(residual, post_weight, gate, scale) else x


def block_norm(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None,
               post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, eps: float = 1e-6, scale: float = 1.0,
               residual_scale: float = 1.0, weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(z, h)`` of a block's output ``x`` [T, H] or [B, S, H] (bf16, fp16 or fp32; H up to 32768): the rows that the next block
    reads, in the type of ``x``, and the new residual stream, in the type of ``residual`` (that of ``x``, or float32).

    ``weight`` and ``post_weight`` are [H] in the type of ``x`` or float32, plus ``weight_offset`` each (1 where a checkpoint stores them
    around 0); ``weight`` None: no weights.  ``gate`` broadcasts to ``x``: one number for a channel, a row, a sequence ([B, 1, H]) or
    every element.  Everything is float32 in between; ``h`` is rounded to its type where it is stored, and ``z`` is the norm of
    that.  Without ``residual``, ``post_weight``, ``gate`` and ``scale`` there is nothing to join: ``h`` is ``x`` itself.
    Sums of squares that float32 does not hold, too large or (where ``eps`` does not stand above them) too small, are taken in 64 bits; a
    row of zeros stays zeros, with ``eps`` 0 as well."""
    z, _, h = _call(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, False)
    return z, h


def block_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None,
                     post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     scale: float = 1.0, residual_scale: float = 1.0,
                     weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(rows int8, scales float32, h)``: :func:`block_norm` with ``z`` as INT8 rows and one scale for each.

    With ``t = h * (weight + weight_offset)`` in float32 the codes of a row are ``round(127 t / max|t|)``, exactly (ties to even): ``z`` is
    not rounded to 16 bits on the way and the root, a factor of the whole row, is in the scale alone.  A row of zeros has
    scale 0, whatever ``eps``; one that holds an infinity or a NaN has scale NaN."""
    return _call(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, True)
