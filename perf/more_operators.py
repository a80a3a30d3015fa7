"""What stands around the linears of a served layer, as cases that can be timed and compared.

* ``add``          low-rank adapters of many requests at once on a projection's output (``adapters.add``): every row has an
                   adapter of its own choice or none, ``y + scale * B (A x)``; a fused projection has several slices, each with
                   a pair of matrices of its own;
* ``linear``       the W4A8 or INT8 linear with the adapters beside it (``adapters.linear``);
* ``norm``         the norm of a block's output, gate, scales, residual and the norm before the next block in one pass
                   (``norms.block_norm``): the new residual stream and its normalised rows;
* ``norm_linear``  the same with INT8 rows and scales (``norms.block_norm_quant``) and the linear that reads them.

Weights have the package's values: INT8 with a scale per channel, re-coded in groups of 64 as 4-bit codes with an integer
step and offset.  Shapes are those of this repository's benchmark (the linears of the 8B layer, shards of the 70B layer) and
generic ones.
"""

import torch

own = False   # whether `run` goes through the package's own operators (their plain forms otherwise)

GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5

# the largest listed case, which drawn ones stay below
MAX_ROWS_BYTES = 8192 * (4096 + 2 * 28672)     # elements of x, y and the result
MAX_PRODUCT = 4096 * 28672 * 4096              # of the linears


def _add(name, T, K, slices, L, rank, dtype, used=None, none=0, sorted_ids=True):
    """`slices`: the widths of a fused projection's parts, as a text; `used`: how many of the L slots the batch reaches;
    `none`: rows without an adapter; `sorted_ids`: the rows of a request are neighbours."""
    return dict(name=name, kind="add", T=T, K=K, slices=slices, L=L, rank=rank, dtype=dtype, used=used or L, none=none,
                sorted_ids=sorted_ids)


def _linear(name, T, K, slices, L, rank, dtype, w4, none=0):
    return dict(name=name, kind="linear", T=T, K=K, slices=slices, L=L, rank=rank, dtype=dtype, used=L, none=none,
                sorted_ids=True, w4=w4)


def _norm(name, T, H, dtype, stream="same", post=False, gate="none", scale=1.0, rscale=1.0, offset=0.0):
    """`stream`: type of the residual ("same" as the block's output, "fp32", or "none": the rows themselves are normalised);
    `gate`: "none", one number per "channel", per "row", or for "all" elements."""
    return dict(name=name, kind="norm", T=T, H=H, dtype=dtype, stream=stream, post=post, gate=gate, scale=scale, rscale=rscale,
                offset=offset)


def _norm_linear(name, T, H, N, dtype, w4, **more):
    return dict(_norm(name, T, H, dtype, **more), kind="norm_linear", N=N, w4=w4)


def listed():
    return [
        # One token of one request: the adapter of the 8B layer's `o` projection.
        _add("add_t1", 1, 4096, "4096", 4, 16, "bf16", used=1),
        # A decode batch, every request with an adapter of its own; q, k and v have their own matrices.
        _add("add_t32_qkv", 32, 4096, "4096,1024,1024", 48, 16, "bf16", used=32, sorted_ids=False),
        # A mixed batch of odd size, a few long requests, some rows without an adapter, an odd rank.
        _add("add_t333", 333, 8192, "1280", 16, 12, "fp16", used=7, none=41),
        # Prefill through `down`: long requests of eight adapters.
        _add("add_t8192", 8192, 14336, "4096", 8, 16, "bf16"),
        # The largest: prefill through gate_up with a high rank.
        _add("add_t8192_r64", 8192, 4096, "14336,14336", 8, 64, "bf16", none=100),
        # A decode batch through the whole projection, 4-bit weights.
        _linear("linear_w4_t16", 16, 4096, "4096,1024,1024", 16, 16, "bf16", True),
        # Prefill through the whole projection, INT8 weights, rows without an adapter.
        _linear("linear_int8_t2000", 2000, 4096, "4096", 12, 32, "fp16", False, none=200),
        # One token: residual and the next block's norm.
        _norm("norm_t1", 1, 4096, "bf16"),
        # An odd batch and width: norms on both sides of the block, a gate per channel, a scaled branch.
        _norm("norm_t777_sandwich", 777, 5001, "fp16", post=True, gate="channel", scale=0.5, offset=1.0),
        # Prefill with a residual stream in 32 bits and a gate for every element.
        _norm("norm_t16384", 16384, 8192, "bf16", stream="fp32", gate="all"),
        # A decode batch: norm, INT8 rows and the qkv projection, 4-bit weights.
        _norm_linear("norm_linear_t16", 16, 4096, 6144, "bf16", True),
        # Prefill: norm, INT8 rows and the gate_up projection, INT8 weights.
        _norm_linear("norm_linear_t4096", 4096, 4096, 28672, "bf16", False, post=True, rscale=0.9),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choices(["add", "linear", "norm", "norm_linear"], [40, 20, 25, 15])[0]
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind in ("add", "linear"):
        K = 128 * _log_uniform(rng, 2, 112)
        parts = [64 * _log_uniform(rng, 2, 160) for _ in range(rng.choice([1, 1, 2, 3]))]
        L = _log_uniform(rng, 1, 64)
        rank = rng.choice([8, 16, 16, 32, 64, 128, rng.randint(1, 64)])
        top = min(8192, MAX_ROWS_BYTES // (K + 2 * sum(parts)))
        if kind == "linear":
            top = min(top, MAX_PRODUCT // (K * sum(parts)))
        # the plain form lets every adapter see every row
        top = max(1, min(top, (1 << 38) // (L * rank * len(parts) * (K + sum(parts)))))
        T = _log_uniform(rng, 1, top)
        none = rng.choice([0, 0, T // 7])
        case = dict(kind=kind, T=T, K=K, slices=",".join(map(str, parts)), L=L, rank=rank, dtype=dtype,
                    used=rng.randint(1, L), none=none, sorted_ids=rng.random() < 0.7)
        return dict(case, w4=rng.random() < 0.6) if kind == "linear" else case
    case = dict(kind=kind, dtype=rng.choice([dtype, "fp32"]) if kind == "norm" else dtype,
                stream=rng.choice(["same", "same", "fp32", "none"]), post=rng.random() < 0.4,
                gate=rng.choice(["none", "none", "channel", "row", "all"]), scale=rng.choice([1.0, 0.22]),
                rscale=rng.choice([1.0, 1.0, 0.7]), offset=rng.choice([0.0, 1.0]))
    if kind == "norm":
        H = _log_uniform(rng, 64, 16384)
        return dict(case, H=H, T=_log_uniform(rng, 1, min(16384, 16384 * 8192 // H // 2)))
    H, N = 128 * _log_uniform(rng, 4, 64), 64 * _log_uniform(rng, 8, 448)
    return dict(case, H=H, N=N, T=_log_uniform(rng, 1, min(4096, MAX_PRODUCT // (H * N))), w4=rng.random() < 0.6)


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------

def _parts(case):
    return [int(s) for s in case["slices"].split(",")]


def _weight(N, K, gen):
    """Gaussian weights in bf16 with one entry in a thousand twenty times larger."""
    w = torch.randn(N, K, device="cuda", generator=gen).mul_(0.02)
    return w.mul_(torch.where(torch.rand(N, K, device="cuda", generator=gen) < 1e-3, 20.0, 1.0)).to(torch.bfloat16)


def _int8_values(w):
    """(q [N,K] int8, s1 [N] fp32) that the bf16 weights stand for once they are quantised at load time."""
    r = w.float()
    s1 = r.abs().amax(1).clamp_min(1e-12) / torch.full((), 119.0, device=w.device)
    c = torch.round(r / s1[:, None]).clamp_(-119, 119).view(w.shape[0], -1, GROUP)
    lo, hi = c.amin(2, keepdim=True), c.amax(2, keepdim=True)
    step = torch.floor((hi - lo + 14) * (1 / 15 + 1e-5)).clamp_(1, 16)   # ceil(range / 15) of whole numbers up to 238
    code = torch.round((c - lo) / step).clamp_(0, 15)
    return (code * step + lo).view(w.shape[0], -1).to(torch.int8), s1


def _activations(T, K, dtype, gen):
    """Gaussian activations with one channel in a hundred ten times larger."""
    hot = torch.where(torch.rand(K, device="cuda", generator=gen) < 0.01, 10.0, 1.0)
    return (torch.randn(T, K, device="cuda", generator=gen) * hot).to(dtype)


def _requests(case, gen):
    """Slot of every row, -1 for none: as many requests as slots reached, of uneven lengths."""
    T, L, used = case["T"], case["L"], min(case["used"], case["T"])
    slots = torch.sort(torch.rand(L, device="cuda", generator=gen)).indices[:used]
    cuts = torch.rand(max(T - used, 0), device="cuda", generator=gen).square().mul(used).long().clamp_max(used - 1)
    order = torch.cat([torch.arange(used, device="cuda"), cuts])
    order = torch.sort(order).values if case["sorted_ids"] else order[torch.sort(torch.rand(T, device="cuda", generator=gen)).indices]
    ids = slots[order].to(torch.int32)
    if case["none"]:
        ids[T - case["none"]:] = -1
    return ids


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, T = DTYPES[case["dtype"]], case["T"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    got = {}
    if case["kind"] in ("add", "linear"):
        K, parts, L, r = case["K"], _parts(case), case["L"], case["rank"]
        got["x"] = _activations(T, K, dtype, gen)
        got["a"] = (randn(L, len(parts), r, K) / K ** 0.5).to(dtype)
        got["b"] = (randn(L, sum(parts), r) * 0.3 / r ** 0.5).to(dtype)
        got["scales"] = 0.5 + torch.rand(L, device="cuda", generator=gen)
        got["ids"] = _requests(case, gen)
        if case["kind"] == "add":
            got["y"] = (1.5 * randn(T, sum(parts))).to(dtype)
        else:
            got["w"] = _weight(sum(parts), K, gen)
        return got
    H = case["H"]
    got["x"] = _activations(T, H, dtype, gen)
    stream = {"same": dtype, "fp32": torch.float32, "none": None}[case["stream"]]
    got["residual"] = None if stream is None else (4.0 * _activations(T, H, torch.float32, gen)).to(stream)
    one = 1.0 - case["offset"]
    got["weight"] = (one + 0.2 * randn(H)).to(dtype)
    got["post"] = (one + 0.2 * randn(H)).to(dtype) if case["post"] else None
    shape = {"none": None, "channel": (H,), "row": (T, 1), "all": (T, H)}[case["gate"]]
    got["gate"] = None if shape is None else (0.7 + 0.3 * randn(*shape)).to(dtype)
    if case["kind"] == "norm_linear":
        got["w"] = _weight(case["N"], H, gen)
    return got


def prepare(case, seed):
    """The inputs, and weights and adapters in the form a serving program keeps them in once they are loaded."""
    state = _inputs(case, seed)
    state["case"] = case
    if "w" in state:
        w = state.pop("w")
        if own:
            from liquidgemm_b200 import ops
            q, blob = ops.quantize_weight_cuda(w, want_codes=not case["w4"], want_blob=case["w4"])
            state["layer"] = {"s1": q.s1, "N": q.N, "K": q.K}
            if case["w4"]:
                state["layer"].update(rs=blob, s_u8=q.s_u8, offset_a=q.offset_a)
            else:
                state["layer"]["w_i8"] = ops.dequant_weight_i8(q)
        else:
            state["layer"] = _int8_values(w)
        del w
    if not own and "a" in state:   # 1 where a column is the slice's
        parts = torch.tensor(_parts(case), device="cuda")
        ends, columns = torch.cumsum(parts, 0)[:, None], torch.arange(sum(_parts(case)), device="cuda")
        state["in_slice"] = ((columns < ends) & (columns >= ends - parts[:, None])).float()
    if own and "a" in state:
        from liquidgemm_b200 import adapters
        parts, a, b = _parts(case), state.pop("a"), state.pop("b")
        stack = adapters.make_stack(case["L"], case["rank"], case["K"], parts, dtype=a.dtype, device=a.device)
        for slot, scale in enumerate(state.pop("scales").tolist()):
            adapters.load(stack, slot, list(a[slot]), list(b[slot].split(parts)), scale)
        state["stack"] = stack
    return state


# --------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------

def _quantise(x):
    scale = x.abs().amax(-1, keepdim=True).clamp_min(1e-12) / torch.full((), 127.0, device=x.device)
    return torch.round(x / scale).clamp(-127, 127), scale


def _product(x, scale, layer):
    q, s1 = layer
    return torch.matmul(x, q.float().t()) * scale * s1


def _delta(state):
    """What the adapters add, in float32: every adapter sees every row, and the rows' own are kept."""
    case, ids = state["case"], state["ids"].long()
    T, L, r, parts = case["T"], case["L"], case["rank"], _parts(case)
    S, N = len(parts), sum(parts)
    v = torch.matmul(state["x"].float(), state["a"].float().view(L * S * r, -1).t()).view(T, L, S * r)
    mine = torch.arange(L, device=ids.device) == ids[:, None]
    v = torch.where(mine[:, :, None], v * state["scales"][:, None], 0.0)
    b = state["b"].float().transpose(1, 2)[:, None] * state["in_slice"][:, None, :]   # zero outside a slice's own columns
    return torch.matmul(v.view(T, L * S * r), b.reshape(L * S * r, N))


def _plain_norm(state):
    """(stream as stored, its rows times the norm's weight, the inverse root) in float32."""
    case, x = state["case"], state["x"].float()
    if case["post"]:
        x = x / torch.sqrt(x.square().mean(1, keepdim=True) + EPS) * (state["post"].float() + case["offset"])
    if state["gate"] is not None:
        x = x * state["gate"].float()
    h = x * case["scale"]
    if state["residual"] is not None:
        h = h + state["residual"].float() * case["rscale"]
    h = h.to(state["x"].dtype if state["residual"] is None else state["residual"].dtype)
    t = h.float() * (state["weight"].float() + case["offset"])
    return h, t, 1.0 / torch.sqrt(h.float().square().mean(1, keepdim=True) + EPS)


def _plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "add":
        return (state["y"].float() + _delta(state)).to(dtype)
    if case["kind"] == "linear":
        return (_product(*_quantise(state["x"].float()), state["layer"]) + _delta(state)).to(dtype)
    h, t, root = _plain_norm(state)
    if case["kind"] == "norm":
        return h, (t * root).to(dtype)
    top = t.abs().amax(1, keepdim=True)
    codes = torch.round(t.double() * 127.0 / top.double().clamp_min(1e-300)).float()   # 64 bits: quotients next to a border
    return h, _product(codes, top * root / 127.0, state["layer"]).to(dtype)


def run(state):
    if not own:
        return _plain(state)
    case = state["case"]
    if case["kind"] == "add":
        from liquidgemm_b200 import adapters
        return adapters.add(state["y"], state["x"], state["stack"], state["ids"])
    if case["kind"] == "linear":
        from liquidgemm_b200 import adapters
        return adapters.linear(state["x"], state["layer"], state["stack"], state["ids"])
    from liquidgemm_b200 import norms
    more = dict(residual=state["residual"], post_weight=state["post"], gate=state["gate"], eps=EPS, scale=case["scale"],
                residual_scale=case["rscale"], weight_offset=case["offset"])
    if case["kind"] == "norm":
        z, h = norms.block_norm(state["x"], state["weight"], **more)
        return h, z
    from liquidgemm_b200 import ops
    rows, scales, h = norms.block_norm_quant(state["x"], state["weight"], **more)
    layer, code = state["layer"], {"bf16": 0, "fp16": 1}[case["dtype"]]
    if case["w4"]:
        return h, torch.ops.liquidgemm.w4a8_wgmma_rs_fused(rows, layer["rs"], layer["s_u8"], layer["offset_a"], scales,
                                                           layer["s1"], layer["N"], layer["K"], 64, code)
    return h, torch.ops.liquidgemm.i8_gemm_scaled(rows, layer["w_i8"], scales, layer["s1"], code)


# --------------------------------------------------------------------------------------------------

def _weight_bytes(case, n, k):   # codes with a step and an offset for each group, or INT8; a scale for each channel
    return (n * k // 2 + 2 * n * (k // GROUP) if case["w4"] else n * k) + 4 * n


def work(case):
    T = case["T"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] in ("add", "linear"):
        K, parts, r = case["K"], _parts(case), case["rank"]
        N, S, rows = sum(parts), len(parts), T - case["none"]
        reached = min(case["used"], max(rows, 0))
        adapters = reached * r * (S * K + N) * size + 4 * T
        flops = 2 * rows * r * (S * K + N)
        if case["kind"] == "add":
            return {"bytes": adapters + T * K * size + 2 * T * N * size, "flops": flops + T * N}
        return {"bytes": adapters + _weight_bytes(case, N, K) + T * (K + N) * size, "flops": flops + 2 * T * N * K}
    H = case["H"]
    stream = {"same": size, "fp32": 4, "none": 0}[case["stream"]]
    joins = case["stream"] != "none" or case["post"] or case["gate"] != "none" or case["scale"] != 1.0
    gate = {"none": 0, "channel": H, "row": T, "all": T * H}[case["gate"]] * size
    moved = T * H * (size + 2 * stream + (size if joins and not stream else 0)) + gate + H * size * (2 if case["post"] else 1)
    if case["kind"] == "norm":
        return {"bytes": moved + T * H * size, "flops": 12 * T * H}
    return {"bytes": moved + _weight_bytes(case, case["N"], H) + T * case["N"] * size, "flops": 2 * T * H * case["N"] + 12 * T * H}


# --------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# --------------------------------------------------------------------------------------------------

def _exact_rows(x):
    # scales and quotients are float32 numbers by definition: half the largest magnitude lies between two codes
    scale = (x.abs().amax(1).clamp_min(1e-12) / 127.0).float().double()
    return torch.round((x / scale[:, None]).float().double()), scale


def exact(case, seed):
    got = _inputs(case, seed)
    T = case["T"]
    if case["kind"] in ("add", "linear"):
        x, ids = got["x"].double(), got["ids"].tolist()
        if case["kind"] == "add":
            y = got["y"].double()
        else:
            q, s1 = _int8_values(got.pop("w"))
            rows, scale = _exact_rows(x)
            y = (rows @ q.double().t()) * scale[:, None] * s1.double()
        for slot in sorted(set(ids) - {-1}):
            mine = torch.tensor([t for t in range(T) if ids[t] == slot], device=x.device)
            at = 0
            for s, n in enumerate(_parts(case)):
                v = x[mine] @ got["a"][slot, s].double().t()
                y[mine, at:at + n] += got["scales"][slot].double() * (v @ got["b"][slot, at:at + n].double().t())
                at += n
        return y
    p = got["x"].double()
    if got["post"] is not None:
        p = p * torch.rsqrt((p * p).sum(1, keepdim=True) / case["H"] + EPS) * (got["post"].double() + case["offset"])
    if got["gate"] is not None:
        p = got["gate"].double() * p
    stream = case["scale"] * p + (0.0 if got["residual"] is None else case["rscale"] * got["residual"].double())
    h = stream.to(got["x"].dtype if got["residual"] is None else got["residual"].dtype).double()   # rounded where it is stored
    w = got["weight"].double() + case["offset"]
    root = torch.rsqrt((h * h).sum(1, keepdim=True) / case["H"] + EPS)
    if case["kind"] == "norm":
        return h, h * root * w
    t = (h * w).float().double()   # a float32 number by definition
    top = t.abs().amax(1, keepdim=True)
    q, s1 = _int8_values(got.pop("w"))
    return h, (torch.round(127.0 * t / top.clamp_min(1e-300)) @ q.double().t()) * (top * root / 127.0) * s1.double()
