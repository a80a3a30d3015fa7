"""The operators of a mixture-of-experts layer, as cases that can be timed and compared.

* ``route``   router logits to the chosen experts and their weights (``moe.route``);
* ``linear``  one product in 8-bit integers for every (token, expert) pair, with a scale for each row of activations and
              each output channel (``moe.experts_linear``): 4-bit or INT8 weights, activations given in 16 bits (and
              quantised on the way) or in INT8, one row per token or one per pair;
* ``mlp``     the gated MLP of the chosen experts: gate and up product, ``silu(gate) * up``, quantisation of each row,
              down product, weighted sum over a token's experts (``moe.experts_mlp``).

Expert weights have the package's values: INT8 with a scale per channel, re-coded in groups of 64 as 4-bit codes with an
integer step and offset.  Activations are INT8 with one scale per row, the largest magnitude over 127, both for the input and
for the gated hidden rows.  Shapes are those of this repository's benchmark (the gate/up and down projections of the 8B
layer, the eight-way shards of the 70B layer) as experts, and generic fine-grained experts.
"""

import torch

own = False   # whether `run` goes through the package's own operators (its plain forms otherwise)

GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# the largest listed case, which drawn ones stay below: its weights, and what its plain form computes and holds
MAX_WEIGHTS = 8 * 3 * 4096 * 14336
MAX_DENSE = 8192 * MAX_WEIGHTS
MAX_HELD = 8 * 8192 * 28672


def _route(name, T, E, k, dtype, scoring="softmax", bias=False, n_group=1, topk_group=1, group_score="max", renorm=True,
           scale=1.0, masked=False):
    return dict(name=name, kind="route", T=T, E=E, k=k, dtype=dtype, scoring=scoring, bias=bias, n_group=n_group,
                topk_group=topk_group, group_score=group_score, renorm=renorm, scale=scale, masked=masked)


def _linear(name, T, E, k, N, K, dtype, w4, int8_in=False, per_pair=False):
    return dict(name=name, kind="linear", T=T, E=E, k=k, N=N, K=K, dtype=dtype, w4=w4, int8_in=int8_in, per_pair=per_pair)


def _mlp(name, T, E, k, H, I, dtype, w4, padded=0):
    return dict(name=name, kind="mlp", T=T, E=E, k=k, H=H, I=I, dtype=dtype, w4=w4, padded=padded)


def listed():
    return [
        # One decode step of a few users on a layer with few experts.
        _route("route_decode", 4, 8, 2, "bf16"),
        # A mixed batch, fine-grained experts, some of them masked out and some rows padding.
        _route("route_mixed", 777, 64, 6, "fp32", renorm=False, masked=True),
        # Prefill with sigmoid scores, a balancing bias, groups and a scale on the weights.
        _route("route_grouped", 8192, 192, 8, "bf16", scoring="sigmoid", bias=True, n_group=8, topk_group=4,
               group_score="top2", scale=2.5),
        # One product of a decode step: the gate/up matrices of the 8B layer, one token.
        _linear("linear_w4_m1", 1, 8, 2, 28672, 4096, "bf16", True),
        # One rank's shard in a mixed batch of odd size; rows already quantised.
        _linear("linear_w4_m333", 333, 16, 3, 1024, 8192, "fp16", True, int8_in=True),
        # INT8 weights, a row of its own for every pair (a down projection), prefill.
        _linear("linear_int8_m2000", 2000, 8, 2, 4096, 14336, "bf16", False, per_pair=True),
        # One token through large experts; a decode batch; the same with padding rows in INT8-weights mode.
        _mlp("mlp_w4_m1", 1, 8, 2, 4096, 14336, "bf16", True),
        _mlp("mlp_w4_m16", 16, 8, 2, 4096, 14336, "fp16", True),
        _mlp("mlp_int8_m48_pad", 48, 32, 4, 4096, 1792, "bf16", False, padded=5),
        # Fine-grained experts, a decode batch that reaches nearly all of them.
        _mlp("mlp_w4_fine_m64", 64, 64, 6, 2048, 1024, "bf16", True),
        # Prefill of a ragged length over fine-grained experts, INT8 weights.
        _mlp("mlp_int8_m3333", 3333, 32, 4, 4096, 1792, "fp16", False),
        # The largest: prefill through large experts.
        _mlp("mlp_w4_m8192", 8192, 8, 2, 4096, 14336, "bf16", True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choices(["route", "linear", "mlp"], [25, 30, 45])[0]
    if kind == "route":
        scoring = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log_uniform(rng, 2 if groups > 1 else 4, 512 // groups)
        kept = rng.randint(1, groups)
        bias = rng.random() < 0.5
        return dict(kind=kind, T=_log_uniform(rng, 1, 16384), E=E, k=rng.randint(1, min(10, kept * (E // groups))),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), scoring=scoring, bias=bias, n_group=groups,
                    topk_group=kept, group_score=rng.choice(["max", "top2"]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), masked=rng.random() < 0.4)
    E = rng.choice([4, 8, 16, 32, 64, _log_uniform(rng, 3, 128)])
    k = rng.randint(1, min(8, E))
    dtype, w4 = rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.6
    weights = MAX_WEIGHTS if w4 else MAX_WEIGHTS // 2
    if kind == "linear":
        K = 128 * _log_uniform(rng, 2, 112)
        N = 64 * _log_uniform(rng, 2, max(3, min(448, weights // (3 * E * K * 64))))
        dense, held = E * N * K, E * N
    else:
        H = 128 * _log_uniform(rng, 4, 64)
        inner = 128 * _log_uniform(rng, 2, max(3, min(112, weights // (3 * E * H * 128))))
        dense, held = 3 * E * H * inner, E * max(2 * inner, H)
    T = _log_uniform(rng, 1, max(2, min(6000, MAX_DENSE // (2 * dense), MAX_HELD // held)))
    if kind == "linear":
        per_pair = rng.random() < 0.4
        T = max(1, T // k) if per_pair else T
        return dict(kind=kind, T=T, E=E, k=k, N=N, K=K, dtype=dtype, w4=w4, int8_in=rng.random() < 0.4, per_pair=per_pair)
    return dict(kind=kind, T=T, E=E, k=k, H=H, I=inner, dtype=dtype, w4=w4, padded=rng.choice([0, 0, T // 5]))


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------

def _weights(E, N, K, gen):
    """Gaussian expert weights in bf16 with one entry in a thousand twenty times larger."""
    w = torch.empty(E, N, K, device="cuda", dtype=torch.bfloat16)
    for e in range(E):
        r = torch.randn(N, K, device="cuda", generator=gen).mul_(0.02)
        r.mul_(torch.where(torch.rand(N, K, device="cuda", generator=gen) < 1e-3, 20.0, 1.0))
        w[e] = r
    return w


def _int8_values(w):
    """(q [E,N,K] int8, s1 [E,N] fp32) that the bf16 weights stand for once they are quantised at load time."""
    q = torch.empty(w.shape, device=w.device, dtype=torch.int8)
    s1 = torch.empty(w.shape[:2], device=w.device)
    for e in range(w.shape[0]):
        r = w[e].float()
        s1[e] = r.abs().amax(1).clamp_min(1e-12) / torch.full((), 119.0, device=w.device)
        c = torch.round(r / s1[e][:, None]).clamp_(-119, 119).view(w.shape[1], -1, GROUP)
        lo, hi = c.amin(2, keepdim=True), c.amax(2, keepdim=True)
        step = torch.floor((hi - lo + 14) * (1 / 15 + 1e-5)).clamp_(1, 16)   # ceil(range / 15) of whole numbers up to 238
        code = torch.round((c - lo) / step).clamp_(0, 15)
        q[e] = (code * step + lo).view(w.shape[1], -1).to(torch.int8)
    return q, s1


def _activations(shape, dtype, gen):
    """Gaussian activations with one channel in a hundred ten times larger."""
    hot = torch.where(torch.rand(shape[-1], device="cuda", generator=gen) < 0.01, 10.0, 1.0)
    return (torch.randn(*shape, device="cuda", generator=gen) * hot).to(dtype)


def _rows_int8(x):
    """Rows in INT8 with their scales, as a producer that quantises them leaves them."""
    scale = x.float().abs().amax(-1).clamp_min(1e-12) / 127.0
    return torch.round(x.float() / scale[..., None]).clamp_(-127, 127).to(torch.int8), scale


def _choice(T, E, k, padded, gen):
    """Experts and weights of a router whose experts are not equally popular; the last rows are padding."""
    logits = torch.randn(T, E, device="cuda", generator=gen) + 0.7 * torch.randn(E, device="cuda", generator=gen)
    top, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    weights, ids = torch.softmax(top[:, :k], 1), ids[:, :k].to(torch.int32)
    if padded:
        ids[T - padded:] = -1
        weights[T - padded:] = 0
    return weights.contiguous(), ids.contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, T, E, k = DTYPES[case["dtype"]], case["T"], case["E"], case["k"]
    if case["kind"] == "route":
        logits = 1.5 * torch.randn(T, E, device="cuda", generator=gen)
        if case["masked"]:
            logits[torch.rand(T, E, device="cuda", generator=gen) < 0.1] = -float("inf")
            logits[torch.rand(T, device="cuda", generator=gen) < 0.05] = -float("inf")
        bias = 0.1 * torch.randn(E, device="cuda", generator=gen) if case["bias"] else None
        return {"logits": logits.to(dtype), "bias": bias}
    got = {}
    if case["kind"] == "linear":
        got["w"] = _weights(E, case["N"], case["K"], gen)
        got["x"] = _activations((T, k, case["K"]) if case["per_pair"] else (T, case["K"]), dtype, gen)
        got["ascale"] = None
        if case["int8_in"]:
            got["x"], got["ascale"] = _rows_int8(got["x"])
        got["ids"] = _choice(T, E, k, 0, gen)[1]
        return got
    got["w13"] = _weights(E, 2 * case["I"], case["H"], gen)
    got["w2"] = _weights(E, case["H"], case["I"], gen)
    got["x"] = _activations((T, case["H"]), dtype, gen)
    got["weights"], got["ids"] = _choice(T, E, k, case["padded"], gen)
    return got


def prepare(case, seed):
    """The inputs, and the weights in the form a serving program keeps them in once the model is loaded."""
    state = _inputs(case, seed)
    state["case"] = case
    for name in ("w", "w13", "w2"):
        if name in state:
            w = state.pop(name)
            if own:
                from liquidgemm_b200 import moe
                state[name] = moe.quantize_experts(w, w4=case["w4"], gated=name == "w13")
            else:
                state[name] = _int8_values(w)
            del w
    return state


# --------------------------------------------------------------------------------------------------
# plain forms: every expert sees every row, and the chosen rows are picked
# --------------------------------------------------------------------------------------------------

def _plain_route(state):
    case = state["case"]
    T, E, k, G = case["T"], case["E"], case["k"], case["n_group"]
    # 64 bits: keys next to one another decide whole numbers
    l = state["logits"].double()
    can = l > -float("inf")
    if case["scoring"] == "softmax":
        top = torch.where(can, l, -float("inf")).amax(1, keepdim=True)
        p = torch.where(can, torch.exp(l - top), 0.0)
        s = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        s = torch.where(can, 1.0 / (1.0 + torch.exp(-l)), 0.0)
    key = torch.where(can, l if state["bias"] is None else s + state["bias"].double(), -float("inf"))
    if G > 1:
        choice = s if state["bias"] is None else key
        if case["group_score"] == "max":
            score = key.view(T, G, -1).amax(2)
        else:
            two = torch.sort(torch.where(can, choice, -float("inf")).view(T, G, -1), dim=2, descending=True).values[..., :2]
            score = torch.where(two[..., 1] > -float("inf"), two[..., 0] + two[..., 1], two[..., 0])
        kept = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :case["topk_group"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        key = torch.where(keep[:, :, None].expand(T, G, E // G).reshape(T, E), key, -float("inf"))
    top, ids = torch.sort(key, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    w = torch.where(top > -float("inf"), torch.gather(s, 1, ids), 0.0)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    return (w * case["scale"]).float(), torch.where(top > -float("inf"), ids, -1).to(torch.int32)


def _quantise(x):
    scale = x.abs().amax(-1, keepdim=True).clamp_min(1e-12) / torch.full((), 127.0, device=x.device)
    return torch.round(x / scale).clamp(-127, 127), scale


def _product(x, scale, weight):
    """[E, rows, N] of the quantised rows [rows, K] or [E, rows, K] and all experts' weights."""
    q, s1 = weight
    return torch.matmul(x, q.float().transpose(1, 2)) * scale * s1[:, None, :]


def _plain_linear(state):
    x, ids, out = state["x"], state["ids"], DTYPES[state["case"]["dtype"]]
    T, k = ids.shape
    if state["ascale"] is None:
        x, scale = _quantise(x.float())
    else:
        x, scale = x.float(), state["ascale"][..., None]
    per_pair = x.dim() == 3
    rows = torch.arange(T * k, device=x.device)
    y = _product(x.flatten(0, -2), scale.flatten(0, -2), state["w"])
    y = y[ids.flatten().long().clamp_min(0), rows if per_pair else rows // k]
    return torch.where(ids.flatten()[:, None] >= 0, y, 0.0).view(T, k, -1).to(out)


def _plain_mlp(state):
    ids, weights = state["ids"].long(), state["weights"]
    T, k = ids.shape
    gate_up = _product(*_quantise(state["x"].float()), state["w13"])
    gate, up = gate_up.chunk(2, 2)
    y = _product(*_quantise(gate / (1.0 + torch.exp(-gate)) * up), state["w2"])
    y = y[ids.clamp_min(0), torch.arange(T, device=y.device)[:, None]]   # [T, k, H]
    return (torch.where(ids >= 0, weights, 0.0)[:, :, None] * y).sum(1).to(DTYPES[state["case"]["dtype"]])


def run(state):
    case = state["case"]
    if not own:
        return {"route": _plain_route, "linear": _plain_linear, "mlp": _plain_mlp}[case["kind"]](state)
    from liquidgemm_b200 import moe
    if case["kind"] == "route":
        return moe.route(state["logits"], case["k"], scoring=case["scoring"], bias=state["bias"], n_group=case["n_group"],
                         topk_group=case["topk_group"], group_score=case["group_score"], renormalize=case["renorm"],
                         scale=case["scale"])
    if case["kind"] == "linear":
        return moe.experts_linear(state["x"], state["ids"], state["w"], ascale=state["ascale"],
                                  out_dtype=DTYPES[case["dtype"]])
    return moe.experts_mlp(state["x"], state["weights"], state["ids"], state["w13"], state["w2"])


# --------------------------------------------------------------------------------------------------

def _reached(case):
    """Experts that a pass reads: the expected number of different ones among the pairs of equally popular experts."""
    pairs = case["T"] - case.get("padded", 0)
    return max(min(case["k"], case["E"]), round(case["E"] * (1 - (1 - case["k"] / case["E"]) ** pairs)))


def work(case):
    T, E, k = case["T"], case["E"], case["k"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "route":
        return {"bytes": T * E * size + (4 * E if case["bias"] else 0) + 8 * T * k, "flops": 10 * T * E}

    def matrix(n, kk):   # codes with a step and an offset for each group, or INT8; a scale for each channel
        return (n * kk // 2 + 2 * n * (kk // GROUP) if case["w4"] else n * kk) + 4 * n

    if case["kind"] == "linear":
        N, K = case["N"], case["K"]
        rows = T * k if case["per_pair"] else T
        return {"bytes": _reached(case) * matrix(N, K) + rows * (K + 4 if case["int8_in"] else K * size) + 4 * T * k +
                T * k * N * size, "flops": 2 * T * k * N * K}
    H, inner = case["H"], case["I"]
    return {"bytes": _reached(case) * (matrix(2 * inner, H) + matrix(H, inner)) + 2 * T * H * size + 8 * T * k,
            "flops": 2 * (T - case["padded"]) * k * 3 * H * inner}


# --------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# --------------------------------------------------------------------------------------------------

def _exact_route(case, got):
    """Row by row on the host."""
    import numpy as np
    logits = got["logits"].double().cpu().numpy()
    bias = None if got["bias"] is None else got["bias"].double().cpu().numpy()
    T, E = logits.shape
    k, size = case["k"], E // case["n_group"]
    weights, ids = np.zeros((T, k)), np.full((T, k), -1, dtype=np.int32)
    for t in range(T):
        row = logits[t]
        live = [e for e in range(E) if row[e] > -np.inf]
        if not live:
            continue
        score = np.zeros(E)
        if case["scoring"] == "softmax":
            score[live] = np.exp(row[live] - max(row[live]))
            score /= score.sum()
        else:
            score[live] = 1.0 / (1.0 + np.exp(-row[live]))
        key = row if bias is None else score + bias
        if case["n_group"] > 1:
            by = []
            for g in range(case["n_group"]):
                mine = [e for e in live if e // size == g]
                if not mine:
                    by.append(-np.inf)
                elif case["group_score"] == "max":
                    by.append(max(key[mine]))
                else:
                    by.append(sum(sorted((score if bias is None else key)[mine], reverse=True)[:2]))
            kept = sorted(range(case["n_group"]), key=lambda g: (-by[g], g))[:case["topk_group"]]
            live = [e for e in live if e // size in kept]
        chosen = sorted(live, key=lambda e: (-key[e], e))[:k]
        ids[t, :len(chosen)] = chosen
        w = score[chosen]
        if case["renorm"] and w.sum() > 0:
            w = w / w.sum()
        weights[t, :len(chosen)] = w * case["scale"]
    return torch.from_numpy(weights), torch.from_numpy(ids)


def _exact_rows(x):
    # scales and quotients are float32 numbers by definition: half the largest magnitude lies between two codes
    scale = (x.abs().amax(1).clamp_min(1e-12) / 127.0).float().double()
    return torch.round((x / scale[:, None]).float().double()), scale


def exact(case, seed):
    got = _inputs(case, seed)
    T, E, k = case["T"], case["E"], case["k"]
    if case["kind"] == "route":
        return _exact_route(case, got)
    names = ("w",) if case["kind"] == "linear" else ("w13", "w2")
    coded = {n: _int8_values(got.pop(n)) for n in names}
    ids = got["ids"].flatten().long()
    x = got["x"].double()
    if case["kind"] == "linear":
        x = x.reshape(-1, x.shape[-1])
        x, scale = (x, got["ascale"].double().flatten()) if case["int8_in"] else _exact_rows(x)
        y = torch.zeros(T * k, case["N"], dtype=torch.float64, device=x.device)
        for e in range(E):
            mine = (ids == e).nonzero().flatten()
            q, s1 = coded["w"][0][e].double(), coded["w"][1][e].double()
            rows = mine if case["per_pair"] else mine // k
            y[mine] = (x[rows] @ q.t()) * scale[rows, None] * s1
        return y.view(T, k, case["N"])
    x, scale = _exact_rows(x)
    y = torch.zeros(T, case["H"], dtype=torch.float64, device=x.device)
    for e in range(E):
        mine = (ids == e).nonzero().flatten()
        (q13, s13), (q2, s2) = [(coded[n][0][e].double(), coded[n][1][e].double()) for n in names]
        rows = mine // k
        gate, up = ((x[rows] @ q13.t()) * scale[rows, None] * s13).split(case["I"], 1)
        h, hs = _exact_rows(gate * torch.sigmoid(gate) * up)
        y.index_add_(0, rows, (h @ q2.t()) * hs[:, None] * s2 * got["weights"].flatten()[mine].double()[:, None])
    return y
