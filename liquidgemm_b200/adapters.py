"""Low-rank adapters of many requests at once beside a linear.

A stack holds the adapters that a server keeps on the GPU, one per slot; every row of a batch names the slot of its request, or none:

    ``y[t, n] + scale[l] * sum_j B[l, n, j] (sum_k A[l, s, j, k] x[t, k])``,  l = ids[t], s = the slice that column n belongs to.

* :func:`make_stack`, :func:`load`, :func:`unload`   the stack and its slots;
* :func:`add`      the adapters' part of a projection, added to its output ``y``;
* :func:`linear`   a W4A8 or INT8 linear with the adapters beside it.

A fused projection (q, k and v; gate and up) has one slice per part, each with matrices of its own.  The operators behind these are
``torch.ops.liquidgemm.adapters_add`` and ``adapters_add_`` (in place), with fake kernels.  Like the dense operators they validate
their arguments in Python, allocate outputs and scratch with torch, enqueue on the current stream of the tensors' device, synchronise
nothing and can be captured into a CUDA graph; which slots a batch reaches is known on the device only, and nothing depends on it on the
host, so a captured step may be replayed with other ids and after slots were loaded anew.  Inference only.

The reference has no counterpart: its plugin quantises plain linears only (liquidgemm/vllm_plugin.py:101-108).
Like :mod:`liquidgemm_b200.ops` this module is not imported by the package ``__init__``.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Sequence, Union

import torch

from ._lib import check, lib
from .moe import _aligned, _any_requires_grad, _plain_call, _refuse, _same_device
from .ops import _DTYPE_CODES, _dev_ctx, _i8_gemm_scaled, _impl, _libdef, _linear, _quant_per_token, _req

_is_alias_of, _increment_version = torch._C._is_alias_of, torch.autograd.graph.increment_version

MAX_SLOTS = 4096
MAX_RANK = 256
MAX_SLICES = 8
MAX_ROWS = 1 << 24
MAX_K = 1 << 20
MAX_CHANNELS = 1 << 22

_ARGS = "Tensor x, Tensor a, Tensor b, Tensor rank, Tensor scale, Tensor ids, int[] widths"
_libdef.define(f"adapters_add(Tensor y, {_ARGS}) -> Tensor")
_libdef.define(f"adapters_add_(Tensor(a!) y, {_ARGS}) -> ()")


@torch.library.register_fake("liquidgemm::adapters_add")
def _f_add(y, x, a, b, rank, scale, ids, widths):
    return y.new_empty(y.shape)


@torch.library.register_fake("liquidgemm::adapters_add_")
def _f_add_(y, x, a, b, rank, scale, ids, widths):
    return None


@lru_cache(maxsize=256)
def _c_widths(widths):
    return (ctypes.c_int * len(widths))(*widths)


@lru_cache(maxsize=1024)
def _scratch_bytes(device, T, K, L, r, S):   # (of the current device, whose number keeps devices apart)
    return lib.lq_adapters_scratch_bytes(T, K, L, r, S)


@lru_cache(maxsize=256)
def _stack_sizes(a_shape, b_shape, widths):
    """(L, S, r, K, N) of a stack's matrices; refused where they do not fit each other."""
    len(a_shape) == 4 and len(b_shape) == 3 or _refuse("the stack's matrices must be [L, S, rank, K] and [L, N, rank]")
    L, S, r, K = a_shape
    N = b_shape[1]
    1 <= L <= MAX_SLOTS and 1 <= S <= MAX_SLICES and 8 <= r <= MAX_RANK and r % 8 == 0 and 8 <= K <= MAX_K and K % 8 == 0 or \
        _refuse(f"1..{MAX_SLOTS} slots, 1..{MAX_SLICES} slices, a rank of 8..{MAX_RANK} and K up to {MAX_K}, both multiples of 8, required")
    b_shape[0] == L and b_shape[2] == r or _refuse("the stack's matrices do not fit each other")
    len(widths) == S and sum(widths) == N <= MAX_CHANNELS and all(w > 0 and w % 8 == 0 for w in widths) or \
        _refuse(f"widths must be {S} multiples of 8 whose sum is {N}")
    return L, S, r, K, N


def _rows(t: torch.Tensor, size: int):
    """(t, pitch) of ``t`` [T, n] with neighbours next to each other, rows and first element on 16-byte boundaries (copied where it is not)."""
    T, n = t.shape
    pitch, step = t.stride()
    if T == 1:
        pitch = n   # a single row has no next
    if step == 1 and pitch >= n and pitch * size % 16 == 0 and t.data_ptr() % 16 == 0:
        return t, pitch
    return _aligned(t), n


def _run(y, x, a, b, rank, scale, ids, widths, inplace):
    dtype, device = x.dtype, x.device
    (dtype is torch.bfloat16 or dtype is torch.float16) and x.is_cuda and x.dim() == 2 or _refuse("x must be a 2-D CUDA tensor of bf16 or fp16")
    a.dtype is dtype and b.dtype is dtype and a.is_contiguous() and b.is_contiguous() or \
        _refuse("the stack's matrices must be contiguous and in the type of x")
    widths = tuple(widths)
    L, S, r, K, N = _stack_sizes(a.shape, b.shape, widths)
    T = x.shape[0]
    x.shape[1] == K or _refuse(f"x must be [T, {K}]")
    y_f32 = y.dtype is torch.float32
    y.is_cuda and y.dim() == 2 and y.shape[0] == T and y.shape[1] == N and (y_f32 or y.dtype is dtype) or \
        _refuse(f"y must be CUDA [{T}, {N}] in the type of x or float32")
    rank.dtype is torch.int32 and scale.dtype is torch.float32 and rank.shape == (L, S) and scale.shape == (L,) and \
        rank.is_contiguous() and scale.is_contiguous() or _refuse(f"rank must be int32 [{L}, {S}] and scale float32 [{L}]")
    wide = ids.dtype is torch.int64
    ids.is_cuda and ids.dim() == 1 and ids.shape[0] == T and (wide or ids.dtype is torch.int32) or \
        _refuse(f"ids must be a CUDA [{T}] tensor of int32 or int64")
    T <= MAX_ROWS or _refuse(f"at most {MAX_ROWS} rows")
    _same_device(x, y, a, b, rank, scale, ids)
    pa, pb = a.data_ptr(), b.data_ptr()
    (pa | pb) % 16 == 0 or _refuse("the stack's matrices must start on 16-byte boundaries")
    if T == 0:
        return y if inplace else torch.empty_like(y, memory_format=torch.contiguous_format)
    yr, ldy = _rows(y, 4 if y_f32 else 2)
    if inplace:
        yr is y or _refuse("y is changed in place: neighbours next to each other, rows on 16-byte boundaries required")
        out, ldo = y, ldy
    else:
        out, ldo = torch.empty((T, N), dtype=y.dtype, device=device), N
    x, ldx = _rows(x, 2)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    with _dev_ctx(x):
        nbytes = _scratch_bytes(device.index, T, K, L, r, S)
        nbytes > 0 or _refuse("sizes out of range")
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
        code = lib.lq_adapters_add(x.data_ptr(), _DTYPE_CODES[dtype], ldx, pa, pb, rank.data_ptr(), scale.data_ptr(), ids.data_ptr(), wide,
                                   yr.data_ptr(), ldy, y_f32, out.data_ptr(), ldo, T, K, L, r, _c_widths(widths), S, scratch.data_ptr(),
                                   nbytes, torch._C._cuda_getCurrentRawStream(device.index))
    if code:
        check(code, "adapters_add")
    if inplace:
        _increment_version(y)   # autograd may have kept y
    return out


def _add(y, x, a, b, rank, scale, ids, widths):
    return _run(y, x, a, b, rank, scale, ids, widths, False)


def _add_(y, x, a, b, rank, scale, ids, widths):
    torch.is_grad_enabled() and _any_requires_grad(y, x, a, b, scale) and \
        _refuse("the adapters have no gradients to give: y cannot be changed in place where they are asked for (torch.no_grad, or out of place)")
    _run(y, x, a, b, rank, scale, ids, widths, True)


_impl.impl("adapters_add", _add)
_impl.impl("adapters_add_", _add_)


# --------------------------------------------------------------------------------------
# Python entry points
# --------------------------------------------------------------------------------------

def make_stack(slots: int, rank: int, K: int, widths: Union[int, Sequence[int]], dtype: torch.dtype = torch.bfloat16,
               device="cuda") -> dict:
    """An empty stack for adapters of a linear with inputs of ``K`` and slices of ``widths`` output channels (one number: one
    slice): ``slots`` of them, of ranks up to ``rank`` (rounded up to a multiple of 8), in ``dtype`` (bf16 or fp16, the activations' type).

    ``{"a" [slots, S, R, K], "b" [slots, N, R], "rank" [slots, S] int32, "scale" [slots] float32, "widths", "K", "N"}`` with R the rank
    rounded up to a multiple of 8.  The tensors keep their addresses; an empty slot has ranks 0."""
    widths = (int(widths),) if isinstance(widths, int) else tuple(int(w) for w in widths)
    _req(1 <= slots <= MAX_SLOTS, f"1..{MAX_SLOTS} slots")
    _req(1 <= rank <= MAX_RANK, f"rank must be 1..{MAX_RANK}")
    _req(8 <= K <= MAX_K and K % 8 == 0, f"K must be a multiple of 8 up to {MAX_K}")
    _req(1 <= len(widths) <= MAX_SLICES and all(w > 0 and w % 8 == 0 for w in widths) and sum(widths) <= MAX_CHANNELS,
         f"1..{MAX_SLICES} slices of widths that are multiples of 8 (up to {MAX_CHANNELS} channels) required")
    _req(dtype in (torch.bfloat16, torch.float16), "dtype must be bfloat16 or float16")
    r = (rank + 7) // 8 * 8
    N = sum(widths)
    return {"a": torch.zeros((slots, len(widths), r, K), dtype=dtype, device=device),
            "b": torch.zeros((slots, N, r), dtype=dtype, device=device),
            "rank": torch.zeros((slots, len(widths)), dtype=torch.int32, device=device),
            "scale": torch.zeros(slots, dtype=torch.float32, device=device), "widths": widths, "K": int(K), "N": N}


def load(stack: dict, slot: int, a, b, scale: float = 1.0) -> None:
    """Put an adapter into ``slot``: ``a`` [r, K] and ``b`` [N, r] (a list of such pairs' halves, one for each slice, for a fused
    projection; ranks may differ, ``None`` for a slice without one), its part multiplied by ``scale`` (``alpha / r``).  The
    matrices may be the stack's own (copied aside first).  Enqueued on the current stream: work on other streams that reads the slot has
    to be ordered by the caller."""
    widths = stack["widths"]
    a, b = ([t] if isinstance(t, torch.Tensor) else list(t) for t in (a, b))
    _req(0 <= slot < stack["rank"].shape[0], f"slot must be 0..{stack['rank'].shape[0] - 1}")
    _req(len(a) == len(widths) and len(b) == len(widths), f"{len(widths)} pairs of matrices required, one for each slice")
    most, K = stack["a"].shape[2], stack["K"]
    ranks = []
    for s, w in enumerate(widths):
        _req((a[s] is None) == (b[s] is None), "a slice has both matrices or none")
        if a[s] is None:
            ranks.append(0)
            continue
        _req(a[s].dim() == 2 and a[s].shape[1] == K and 1 <= a[s].shape[0] <= most, f"a must be [1..{most}, {K}]")
        _req(tuple(b[s].shape) == (w, a[s].shape[0]), f"b must be [{w}, {a[s].shape[0]}]")
        ranks.append(a[s].shape[0])
    def aside(t):   # (the slot is cleared first)
        return t.clone() if t is not None and (_is_alias_of(t, stack["a"]) or _is_alias_of(t, stack["b"])) else t

    a, b = [aside(t) for t in a], [aside(t) for t in b]
    with torch.no_grad():
        stack["a"][slot].zero_()
        stack["b"][slot].zero_()
        at = 0
        for s, w in enumerate(widths):
            if ranks[s]:
                stack["a"][slot, s, :ranks[s]].copy_(a[s])
                stack["b"][slot, at:at + w, :ranks[s]].copy_(b[s])
            at += w
        stack["scale"][slot] = float(scale)
        for s, n in enumerate(ranks):
            stack["rank"][slot, s] = n


def unload(stack: dict, slot: int) -> None:
    """Empty ``slot``: rows that name it are left as they are."""
    _req(0 <= slot < stack["rank"].shape[0], f"slot must be 0..{stack['rank'].shape[0] - 1}")
    stack["rank"][slot].zero_()


def add(y: torch.Tensor, x: torch.Tensor, stack: dict, ids: torch.Tensor, inplace: bool = False) -> torch.Tensor:
    """``y`` [T, N] plus what the adapters of its rows make of ``x`` [T, K] (bf16 or fp16), in the type of ``y`` (that of ``x``, or
    float32): a new tensor, or ``y`` itself, changed, with ``inplace``.

    ``ids`` [T] (int32 or int64) names the slot of every row; an id outside the slots, or an empty slot, leaves its row as it is.
    Both products are summed in float32 and the result is rounded once.  Between them a row goes on as two 16-bit numbers for each sum,
    which keep 16 bits of it (bf16; fp16: 22): beside a float32 ``y`` the result is off by that, 2^-16 of what a bf16 adapter adds.
    In place is refused where gradients are asked for."""
    args = (y, x, stack["a"], stack["b"], stack["rank"], stack["scale"], ids)
    if inplace:
        (_add_ if _plain_call(*args) else torch.ops.liquidgemm.adapters_add_)(*args, stack["widths"])
        return y
    return (_add if _plain_call(*args) else torch.ops.liquidgemm.adapters_add)(*args, stack["widths"])


def linear(x: torch.Tensor, layer: dict, stack: dict, ids: torch.Tensor, bias: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A linear with the adapters of its rows beside it: [T, N] in ``out_dtype`` (default: that of ``x``).

    ``layer`` holds a layer's device tensors: 4-bit weights as :func:`liquidgemm_b200.ops.w4a8_linear` takes them (``rs, s_u8, offset_a,
    s1, N, K``), or ``w_i8`` [N, K] with ``s1`` in place of the first three.  The linear quantises ``x``, the adapters read it
    as it is; their part joins the linear's rounded output (like ``bias`` [N], in ``out_dtype``, does), so the result is that of the linear
    and :func:`add`, bit for bit.  With 16-bit outputs that rounds twice (three times with a bias), by half a step at most each time:
    1.4 times the root-mean-square error of one rounding.  ``out_dtype=torch.float32``, rounded by the caller, rounds once."""
    out_dtype = out_dtype or x.dtype
    _req(x.dtype in (torch.bfloat16, torch.float16) and out_dtype in (x.dtype, torch.float32),
         "x must be bf16 or fp16, out_dtype its type or float32")
    _req(layer["N"] == stack["N"] and layer["K"] == stack["K"], "the stack is for another linear (N and K)")
    if bias is not None:   # (one contract for both weight kinds: no broadcast, no promotion of the result)
        bias.is_cuda and bias.dtype == out_dtype and bias.numel() == layer["N"] or \
            _refuse(f"bias must be a CUDA [{layer['N']}] tensor of the output type, {out_dtype}")
        _same_device(x, bias)
        bias = bias.reshape(-1)
    code = _DTYPE_CODES[out_dtype]
    blob = layer.get("rs")
    # (in place only where nothing transforms the call or asks for gradients, the stack's among them: y may be what is not batched)
    plain = _plain_call(x, blob if blob is not None else layer["w_i8"], layer["s1"], bias, stack["a"], stack["b"], stack["rank"], stack["scale"],
                        ids)
    if blob is not None:
        run = _linear if plain else torch.ops.liquidgemm.w4a8_linear
        y = run(x, blob, layer["s_u8"], layer["offset_a"], layer["s1"], bias, layer["N"], layer["K"], 64, code)
    else:
        quantise, product = (_quant_per_token, _i8_gemm_scaled) if plain else \
            (torch.ops.liquidgemm.quant_per_token, torch.ops.liquidgemm.i8_gemm_scaled)
        rows, scales = quantise(x)
        y = product(rows, layer["w_i8"], scales, layer["s1"], code)
        if bias is not None:
            y = y.add_(bias) if plain else y + bias
    if plain:
        return _run(y, x, stack["a"], stack["b"], stack["rank"], stack["scale"], ids, stack["widths"], True)
    return add(y, x, stack, ids)
