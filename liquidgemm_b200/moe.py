"""Mixture-of-experts layers in 8-bit integers: router, products grouped by expert, gated MLP.

The expert weights are those of the dense linears (:mod:`liquidgemm_b200.ops`), stacked: 4-bit tile blobs or INT8 rows
with one scale per channel, activations in INT8 with one scale per row, exact int32 sums.

* :func:`route`            router logits -> weights and ids of the chosen experts;
* :func:`quantize_experts` stacked bf16 / fp16 / fp32 weights -> the form the products read, once per model load;
* :func:`experts_linear`   one product for every (token, chosen expert) pair;
* :func:`experts_mlp`      gate/up product, ``silu(gate) * up``, quantisation, down product, weighted sum.

The operators behind them are ``torch.ops.liquidgemm.moe_route``, ``experts_linear`` and ``experts_mlp``, with fake
kernels, so that they can be traced.  Like the dense operators they validate their arguments in Python, allocate outputs and scratch
with torch, enqueue on the current stream of the tensors' device, synchronise nothing and can be captured into a CUDA graph.  How
many rows an expert gets is known on the device only; nothing depends on it on the host.

The reference has no counterpart: its plugin quantises plain linears only (liquidgemm/vllm_plugin.py:101-108).
Like :mod:`liquidgemm_b200.ops` this module is not imported by the package ``__init__``.
"""

from __future__ import annotations

from typing import Optional

import torch

from ._lib import check, lib
from .ops import _DTYPE_CODES, _OUT_DTYPES, TILE_BYTES, _dev_ctx, _impl, _libdef, _ptr, _req, _stream

MAX_EXPERTS = 512
MAX_TOPK = 32
MAX_PAIRS = 1 << 24
_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}

_libdef.define("moe_route(Tensor logits, Tensor? bias, int topk, int scoring, int n_group, int topk_group, int group_score, "
               "bool renormalize, float scale) -> (Tensor, Tensor)")
_libdef.define("experts_linear(Tensor x, Tensor? ascale, Tensor ids, Tensor w, Tensor s1, int N, int K, int out_dtype) -> Tensor")
_libdef.define("experts_mlp(Tensor x, Tensor weights, Tensor ids, Tensor w13, Tensor s13, Tensor w2, Tensor s2, int out_dtype) "
               "-> Tensor")


@torch.library.register_fake("liquidgemm::moe_route")
def _f_route(logits, bias, topk, scoring, n_group, topk_group, group_score, renormalize, scale):
    shape = (logits.shape[0], topk)
    return logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32)


@torch.library.register_fake("liquidgemm::experts_linear")
def _f_linear(x, ascale, ids, w, s1, N, K, out_dtype):
    return x.new_empty((*ids.shape, N), dtype=_OUT_DTYPES[int(out_dtype)])


@torch.library.register_fake("liquidgemm::experts_mlp")
def _f_mlp(x, weights, ids, w13, s13, w2, s2, out_dtype):
    return x.new_empty(x.shape, dtype=_OUT_DTYPES[int(out_dtype)])


def _refuse(msg: str):
    raise RuntimeError(msg)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and on a 16-byte boundary (a view may start anywhere in its storage)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _same_device(first, *others):
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:
            _refuse(f"every tensor must be on the device of the first argument, {first.device} (one is on {t.device})")


def _ids(ids: torch.Tensor) -> torch.Tensor:
    _req(ids.is_cuda and ids.dim() == 2 and ids.dtype in (torch.int32, torch.int64), "ids must be a CUDA [T, topk] tensor of int32 or int64")
    # (messages with values are put together only where one is raised: a call of these costs the host as much as a kernel)
    1 <= ids.shape[1] <= MAX_TOPK or _refuse(f"topk must be 1..{MAX_TOPK}")
    ids.numel() <= MAX_PAIRS or _refuse(f"at most {MAX_PAIRS} (token, expert) pairs")
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, MAX_EXPERTS).to(torch.int32)   # what is no expert stays none
    return ids.contiguous()


def _weights(w: torch.Tensor, s1: torch.Tensor, N: int, K: int, name: str):
    """(kind, w, s1, E) of one stack of expert matrices [E, N, K]."""
    dtype = w.dtype
    w.is_cuda and (dtype is torch.uint8 or dtype is torch.int8) or \
        _refuse(f"{name} must be a CUDA tensor: uint8 tile blobs or int8 rows")
    s1.is_cuda and s1.dtype is torch.float32 and s1.dim() == 2 and s1.shape[1] == N or \
        _refuse(f"the scales of {name} must be CUDA float32 [E, {N}]")
    E = s1.shape[0]
    1 <= E <= MAX_EXPERTS or _refuse(f"1..{MAX_EXPERTS} experts")
    1 <= N < 1 << 30 and K >= 128 and K % 128 == 0 or _refuse(f"{name}: N below 2^30 and K % 128 == 0 required")
    K < 131072 or _refuse(f"{name}: K below 131072 required (int32 sums)")
    if dtype is torch.uint8:
        need = E * ((N + 127) // 128) * (K // 128) * TILE_BYTES
        w.numel() == need or _refuse(f"{name} must hold {E} tile blobs for N={N}, K={K} ({need} bytes, got {w.numel()})")
        return 0, _aligned(w), _aligned(s1), E
    w.numel() == E * N * K or _refuse(f"{name} must be int8 [{E}, {N}, {K}]")
    return 1, _aligned(w), _aligned(s1), E


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    _req(nbytes > 0, "sizes out of range")
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


def _moe_route(logits, bias, topk, scoring, n_group, topk_group, group_score, renormalize, scale):
    logits.is_cuda and logits.dim() == 2 and logits.dtype in _DTYPE_CODES or _refuse("logits must be a 2-D CUDA tensor of bf16, fp16 or fp32")
    T, E = logits.shape
    1 <= E <= MAX_EXPERTS or _refuse(f"1..{MAX_EXPERTS} experts")
    T < 1 << 31 or _refuse("fewer than 2^31 tokens required")   # (a C int, which ctypes would cut)
    scoring in (0, 1) and group_score in (0, 1) or _refuse("scoring and group_score must be 0 or 1")
    n_group >= 1 and E % n_group == 0 or _refuse("n_group must divide the number of experts")
    1 <= topk_group <= n_group or _refuse("topk_group must be 1..n_group")
    1 <= topk <= MAX_TOPK and topk <= topk_group * (E // n_group) or \
        _refuse(f"topk must be 1..{MAX_TOPK} and at most the experts of topk_group groups")
    if bias is not None:
        _req(bias.is_cuda and bias.dtype == torch.float32 and bias.shape == (E,), "bias must be a CUDA float32 [E] tensor")
        _same_device(logits, bias)
        bias = bias.contiguous()
    logits = logits.contiguous()
    device = logits.device
    weights = torch.empty(T, topk, dtype=torch.float32, device=device)
    ids = torch.empty(T, topk, dtype=torch.int32, device=device)
    if T:
        with _dev_ctx(logits):
            check(lib.lq_moe_route(logits.data_ptr(), _DTYPE_CODES[logits.dtype], None if bias is None else bias.data_ptr(),
                                   weights.data_ptr(), ids.data_ptr(), T, E, topk, scoring, n_group, topk_group, group_score,
                                   int(renormalize), scale, torch._C._cuda_getCurrentRawStream(device.index)), "moe_route")
    return weights, ids


def _experts_linear(x, ascale, ids, w, s1, N, K, out_dtype):
    ids = _ids(ids)
    T, topk = ids.shape
    shape = x.shape
    per_pair = len(shape) == 3
    x.is_cuda and (per_pair or len(shape) == 2) and shape[-1] == K or _refuse(f"x must be a CUDA [T, {K}] or [T, topk, {K}] tensor")
    shape[0] == T and (not per_pair or shape[1] == topk) or _refuse("x and ids must have the same tokens (and slots)")
    _req(int(out_dtype) in _OUT_DTYPES, "out_dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)")
    if ascale is None:
        _req(x.dtype in _DTYPE_CODES, "x must be bfloat16, float16 or float32 (or int8 with ascale)")
        code = _DTYPE_CODES[x.dtype]
    else:
        _req(x.dtype == torch.int8, "ascale comes with int8 rows")
        _req(ascale.is_cuda and ascale.dtype == torch.float32 and ascale.numel() == x.numel() // K, "ascale must be CUDA float32 with one scale for each row of x")
        ascale = ascale.contiguous()
        code = 3
    kind, w, s1, E = _weights(w, s1, N, K, "w")
    _same_device(x, ids, w, s1, ascale)
    y = torch.empty(T, topk, N, dtype=_OUT_DTYPES[int(out_dtype)], device=x.device)
    if T == 0:
        return y
    x = _aligned(x)
    with _dev_ctx(x):
        scratch = _scratch(lib.lq_experts_linear_scratch_bytes(T, topk, E, N, K, kind), x)
        check(lib.lq_experts_linear(_ptr(x), code, None if ascale is None else _ptr(ascale), int(per_pair), _ptr(ids), _ptr(w),
                                    kind, _ptr(s1), _ptr(y), int(out_dtype), T, topk, E, N, K, _ptr(scratch), scratch.numel(),
                                    _stream()), "experts_linear")
    return y


def _experts_mlp(x, weights, ids, w13, s13, w2, s2, out_dtype):
    ids = _ids(ids)
    T, topk = ids.shape
    _req(x.is_cuda and x.dim() == 2 and x.dtype in _DTYPE_CODES, "x must be a 2-D CUDA tensor of bf16, fp16 or fp32")
    _req(x.shape[0] == T, "x and ids must have the same tokens")
    _req(weights.is_cuda and weights.dtype == torch.float32 and weights.shape == ids.shape, "weights must be CUDA float32 [T, topk]")
    _req(int(out_dtype) in _OUT_DTYPES, "out_dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)")
    H = x.shape[1]
    _req(s13.dim() == 2 and s13.shape[1] % 2 == 0, "the scales of w13 must be [E, 2 I]")
    inner = s13.shape[1] // 2
    kind, w13, s13, E = _weights(w13, s13, 2 * inner, H, "w13")
    kind2, w2, s2, E2 = _weights(w2, s2, H, inner, "w2")
    _req(kind == kind2 and E == E2, "w13 and w2 must be of the same kind and have the same experts")
    _same_device(x, ids, weights, w13, s13, w2, s2)
    y = torch.empty(T, H, dtype=_OUT_DTYPES[int(out_dtype)], device=x.device)
    if T == 0:
        return y
    x, weights = _aligned(x), weights.contiguous()
    with _dev_ctx(x):
        scratch = _scratch(lib.lq_experts_mlp_scratch_bytes(T, topk, E, H, inner, kind), x)
        check(lib.lq_experts_mlp(_ptr(x), _DTYPE_CODES[x.dtype], _ptr(weights), _ptr(ids), _ptr(w13), _ptr(s13), _ptr(w2),
                                 _ptr(s2), kind, _ptr(y), int(out_dtype), T, topk, E, H, inner, _ptr(scratch),
                                 scratch.numel(), _stream()), "experts_mlp")
    return y


_ORDINARY = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))
_is_compiling, _dispatch_modes, _tracing_state, _transform = (torch.compiler.is_compiling, torch._C._len_torch_dispatch_stack,
                                                              torch._C._get_tracing_state, torch._C._functorch.peek_interpreter_stack)
_any_requires_grad, _forward_ad = torch._C._any_requires_grad, torch.autograd.forward_ad


def _plain_call(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether an operator may be called without torch's dispatcher: ordinary CUDA tensors that no gradient is asked of, and nothing
    that traces, transforms or intercepts (under ``vmap`` and its like a wrapped tensor looks ordinary).  The dispatcher's way into
    a Python kernel costs 4.5 us of the host's 17 for a router call, which is all that a small one takes."""
    if _is_compiling() or _dispatch_modes() or _tracing_state() is not None or _transform() is not None or _forward_ad._current_level >= 0:
        return False
    if not _ORDINARY.issuperset(map(type, tensors)) or (_any_requires_grad(*tensors) and torch.is_grad_enabled()):
        return False
    return tensors[0].is_cuda


_impl.impl("moe_route", _moe_route)
_impl.impl("experts_linear", _experts_linear)
_impl.impl("experts_mlp", _experts_mlp)


# --------------------------------------------------------------------------------------
# Python entry points
# --------------------------------------------------------------------------------------

def route(logits: torch.Tensor, topk: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, n_group: int = 1,
          topk_group: int = 1, group_score: str = "max", renormalize: bool = True, scale: float = 1.0):
    """``(weights [T, topk] float32, ids [T, topk] int32)`` of the experts chosen for each row of ``logits`` [T, E].

    Scores are ``softmax(logits)`` or ``sigmoid(logits)``; experts are chosen by score plus ``bias`` [E], the largest first and the
    lowest index among equals.  With ``n_group`` > 1 only experts of the ``topk_group`` best groups of E / n_group neighbours
    can be chosen; a group ranks by its largest key (``group_score="max"``) or the sum of its two largest (``"top2"``).
    Weights are the scores without the bias, divided by their sum with ``renormalize``, times ``scale``: those of 64-bit scores, however
    small, and 0 where none of the chosen has one.  A logit of -inf or NaN takes its expert out; slots for which no expert is left have
    id -1 and weight 0 (the products skip them)."""
    scoring in _SCORING or _refuse("scoring must be 'softmax' or 'sigmoid'")
    group_score in _GROUP_SCORE or _refuse("group_score must be 'max' or 'top2'")
    run = _moe_route if _plain_call(logits, bias) else torch.ops.liquidgemm.moe_route
    return run(logits, bias, int(topk), _SCORING[scoring], int(n_group), int(topk_group), _GROUP_SCORE[group_score], bool(renormalize),
               float(scale))


def quantize_experts(w: torch.Tensor, w4: bool = True, gated: bool = False, group_size: int = 64) -> dict:
    """Expert weights ``w`` [E, N, K] (CUDA; bf16, fp16 or fp32) in the form the products read: ``{"w", "s1", "E", "N", "K",
    "gated"}`` with ``w`` the tile blobs of the 4-bit codes [E, ceil(N/128), K/128, 8704] (``w4``) or the INT8 values they stand for
    [E, N, K], the two weight forms of the dense linears, and ``s1`` [E, N] the channel scales.  ``gated``: N = 2 I rows, the I gate
    rows first and the I up rows behind them, as :func:`experts_mlp` takes them; they are stored in turn."""
    _req(w.is_cuda and w.dim() == 3 and w.dtype in _DTYPE_CODES, "w must be a 3-D CUDA tensor of bf16, fp16 or fp32")
    E, N, K = w.shape
    _req(1 <= E <= MAX_EXPERTS and N >= 1, f"1..{MAX_EXPERTS} experts with at least one row")
    _req(K >= 128 and K % 128 == 0 and group_size in (64, 128), "K % 128 == 0 and group_size 64 or 128 required")
    _req(not gated or N % 2 == 0, "gated weights have as many up rows as gate rows")
    dev = w.device
    s1 = torch.empty((E, N), dtype=torch.float32, device=dev)
    if w4:
        out = torch.empty((E, (N + 127) // 128, K // 128, TILE_BYTES), dtype=torch.uint8, device=dev)
    else:
        out = torch.empty((E, N, K), dtype=torch.int8, device=dev)
    with _dev_ctx(w):
        s_u8 = torch.empty((N, K // group_size), dtype=torch.uint8, device=dev)
        off = torch.empty_like(s_u8)
        codes = None if w4 else torch.empty((N, K), dtype=torch.uint8, device=dev)
        for e in range(E):   # one expert at a time: the reordered copy of a gated stack stays small
            rows = w[e].detach()
            if gated:
                rows = rows.view(2, N // 2, K).transpose(0, 1).reshape(N, K) if rows.is_contiguous() else \
                    torch.stack([rows[:N // 2], rows[N // 2:]], dim=1).view(N, K)
            rows = rows.contiguous()
            check(lib.lq_quantize_weight(_ptr(rows), _DTYPE_CODES[w.dtype], N, K, group_size, _ptr(s1[e]), _ptr(s_u8), _ptr(off),
                                         _ptr(codes) if codes is not None else None, _ptr(out[e]) if w4 else None, _stream()),
                  "quantize_experts")
            if not w4:
                check(lib.lq_dequant_weight(_ptr(codes), _ptr(s_u8), _ptr(off), _ptr(out[e]), N, K, group_size, _stream()),
                      "quantize_experts")
    return {"w": out, "s1": s1, "E": E, "N": N, "K": K, "gated": bool(gated)}


def experts_linear(x: torch.Tensor, ids: torch.Tensor, layer: dict, ascale: Optional[torch.Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``y[t, j] = W[ids[t, j]] x[t]`` (or ``x[t, j]``): [T, topk, N] in ``out_dtype`` (default: that of ``x``, bf16 for INT8 rows).

    ``x`` is [T, K], or [T, topk, K] with a row for every pair, in bf16, fp16 or fp32 (each row is quantised on the way) or
    in INT8 with ``ascale``, one scale per row.  ``layer`` comes from :func:`quantize_experts`.  The values are those of the dense
    linear, bit for bit; an id outside the experts gives a row of zeros."""
    _req(not layer["gated"], "a gated stack is stored for experts_mlp")
    out_dtype = out_dtype or (torch.bfloat16 if x.dtype == torch.int8 else x.dtype)
    _req(out_dtype in _DTYPE_CODES, "out_dtype must be bfloat16, float16 or float32")
    w, s1 = layer["w"], layer["s1"]
    run = _experts_linear if _plain_call(x, ascale, ids, w, s1) else torch.ops.liquidgemm.experts_linear
    return run(x, ascale, ids, w, s1, layer["N"], layer["K"], _DTYPE_CODES[out_dtype])


def experts_mlp(x: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor, w13: dict, w2: dict,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``y[t] = sum_j weights[t, j] * W2[e] (silu(gate) * up)`` with gate and up from ``W13[e] x[t]``, e = ids[t, j]: [T, H] in
    ``out_dtype`` (default: that of ``x``).

    ``x`` [T, H] in bf16, fp16 or fp32 and the hidden rows are quantised to INT8 with one scale per row; everything between the
    integer sums is float32 and the result is rounded once.  ``w13`` and ``w2`` come from :func:`quantize_experts` (``w13`` with
    ``gated=True``); an id outside the experts adds nothing."""
    _req(w13["gated"] and not w2["gated"], "w13 must be quantised with gated=True and w2 without")
    out_dtype = out_dtype or x.dtype
    _req(out_dtype in _DTYPE_CODES, "out_dtype must be bfloat16, float16 or float32")
    args = (x, weights, ids, w13["w"], w13["s1"], w2["w"], w2["s1"])
    run = _experts_mlp if _plain_call(*args) else torch.ops.liquidgemm.experts_mlp
    return run(*args, _DTYPE_CODES[out_dtype])
