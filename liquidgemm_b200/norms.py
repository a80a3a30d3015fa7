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
from .ops import _DTYPE_CODES, _dev_ctx, _impl, _libdef, _stream

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


def _strides(t: torch.Tensor):
    """(t, outer, inner) of [T, H] or [B, S, H] rows whose elements are neighbours."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    return (t, t.stride(0), t.stride(1)) if t.dim() == 3 else (t, 0, t.stride(0))


def _vector(w, name, H, dtype):
    w.is_cuda and w.shape == (H,) and (w.dtype is dtype or w.dtype is torch.float32) or \
        _refuse(f"{name} must be a CUDA [{H}] tensor in the type of x or float32")
    return w.contiguous()


def _block_norm(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, quantize):
    dtype = x.dtype
    x.is_cuda and x.dim() in (2, 3) and dtype in _DTYPE_CODES or _refuse("x must be a CUDA [T, H] or [B, S, H] tensor of bf16, fp16 or fp32")
    shape = x.shape
    H = shape[-1]
    rows = x.numel() // H if H else 0
    1 <= H <= MAX_WIDTH or _refuse(f"H must be 1..{MAX_WIDTH}")
    rows < 1 << 31 or _refuse("fewer than 2^31 rows required")
    eps >= 0.0 or _refuse("eps must not be negative")
    if residual is not None:
        residual.is_cuda and residual.shape == shape and (residual.dtype is dtype or residual.dtype is torch.float32) or \
            _refuse("residual must be a CUDA tensor of x's shape, in the type of x or float32")
    if weight is not None:
        weight = _vector(weight, "weight", H, dtype)
    if post_weight is not None:
        post_weight = _vector(post_weight, "post_weight", H, dtype)
    if gate is not None:
        gate.is_cuda and (gate.dtype is dtype or gate.dtype is torch.float32) or \
            _refuse("gate must be a CUDA tensor in the type of x or float32")
        gate.dim() <= len(shape) and all(g in (1, n) for g, n in zip(reversed(gate.shape), reversed(shape))) or \
            _refuse(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    _same_device(x, residual, weight, post_weight, gate)
    stream = x if residual is None else residual
    joins = _joins(residual, post_weight, gate, scale)
    device = x.device
    z = torch.empty(shape, dtype=torch.int8 if quantize else dtype, device=device)
    q_scale = torch.empty(shape[:-1] if quantize else (0,), dtype=torch.float32, device=device)
    h = torch.empty(shape if joins else (0,), dtype=stream.dtype, device=device)
    if rows == 0:
        return z, q_scale, h
    inner = shape[1] if len(shape) == 3 else rows
    x, xo, xi = _strides(x)
    r, ro, ri, g, go, gi, step = None, 0, 0, None, 0, 0, 0
    if residual is not None:
        residual, ro, ri = _strides(residual)
        r = residual.data_ptr()
    if gate is not None:
        per_row = gate.dim() == 0 or (gate.shape[-1] == 1 and H > 1)
        if not per_row and gate.stride(-1) != 1 and H > 1:
            gate = gate.contiguous()
        wide = gate.expand(shape)
        go, gi = (wide.stride(0), wide.stride(1)) if len(shape) == 3 else (0, wide.stride(0))
        g, step = gate.data_ptr(), 0 if per_row else 1
    with _dev_ctx(x):
        check(lib.lq_block_norm(x.data_ptr(), _DTYPE_CODES[dtype], xo, xi, r, _DTYPE_CODES[stream.dtype], ro, ri, g,
                                0 if gate is None else _DTYPE_CODES[gate.dtype], go, gi, step,
                                None if weight is None else weight.data_ptr(), 0 if weight is None else _DTYPE_CODES[weight.dtype],
                                None if post_weight is None else post_weight.data_ptr(),
                                0 if post_weight is None else _DTYPE_CODES[post_weight.dtype],
                                None if quantize else z.data_ptr(), z.data_ptr() if quantize else None,
                                q_scale.data_ptr() if quantize else None, h.data_ptr() if joins else None, rows, inner, H,
                                eps, scale, residual_scale, weight_offset, _stream()), "block_norm")
    return z, q_scale, h


_impl.impl("block_norm", _block_norm)


# --------------------------------------------------------------------------------------
# Python entry points
# --------------------------------------------------------------------------------------

def _call(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, quantize):
    run = _block_norm if _plain_call(x, weight, residual, post_weight, gate) else torch.ops.liquidgemm.block_norm
    z, q_scale, h = run(x, weight, residual, post_weight, gate, float(eps), float(scale), float(residual_scale),
                        float(weight_offset), quantize)
    return z, q_scale, h if _joins(residual, post_weight, gate, scale) else x


def block_norm(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None,
               post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, eps: float = 1e-6, scale: float = 1.0,
               residual_scale: float = 1.0, weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(z, h)`` of a block's output ``x`` [T, H] or [B, S, H] (bf16, fp16 or fp32; H up to 32768): the rows that the next block
    reads, in the type of ``x``, and the new residual stream, in the type of ``residual`` (that of ``x``, or float32).

    ``weight`` and ``post_weight`` are [H] in the type of ``x`` or float32, plus ``weight_offset`` each (1 where a checkpoint stores them
    around 0); ``weight`` None: no weights.  ``gate`` broadcasts to ``x``: one number for a channel, a row, a sequence ([B, 1, H]) or
    every element.  Everything is float32 in between; ``h`` is rounded to its type where it is stored, and ``z`` is the norm of
    that.  Without ``residual``, ``post_weight``, ``gate`` and ``scale`` there is nothing to join: ``h`` is ``x`` itself."""
    z, _, h = _call(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, False)
    return z, h


def block_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None,
                     post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     scale: float = 1.0, residual_scale: float = 1.0,
                     weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(rows int8, scales float32, h)``: :func:`block_norm` with ``z`` as INT8 rows and one scale for each.

    With ``t = h * (weight + weight_offset)`` in float32 the codes of a row are ``round(127 t / max|t|)``, exactly (ties to even): ``z`` is
    not rounded to 16 bits on the way and the root, a factor of the whole row, is in the scale alone.  A row of zeros has
    scale 0; one that holds an infinity or a NaN has scale NaN."""
    return _call(x, weight, residual, post_weight, gate, eps, scale, residual_scale, weight_offset, True)
