"""The registered operators of the adapters and the norms on the device, and the entry points wherever these have to go through them:
compiled, traced and transformed calls, gradients asked for.  The results are the entry points' own, bit for bit."""

import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu

T, K, N, R = 21, 256, 192, 12


def _randn(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.fixture(scope="module")
def data():
    from liquidgemm_b200 import adapters, norms, ops   # (norms: its operator is registered there)
    stack = adapters.make_stack(4, R, K, (128, 64))
    for slot in range(3):
        adapters.load(stack, slot, [_randn(slot, R, K) * 0.1, _randn(9 + slot, 5, K) * 0.1], [_randn(4 + slot, 128, R), _randn(6 + slot, 64, 5)], 0.5 + slot)
    q, blob = ops.quantize_weight_cuda(_randn(1, N, K) * 0.05, want_codes=True, want_blob=True)
    return {"x": _randn(2, T, K), "y": _randn(3, T, N), "ids": torch.arange(T, device="cuda") % 5 - 1, "stack": stack, "bias": _randn(4, N),
            "w4": {"rs": blob, "s_u8": q.s_u8, "offset_a": q.offset_a, "s1": q.s1, "N": N, "K": K},
            "int8": {"w_i8": ops.dequant_weight_i8(q), "s1": q.s1, "N": N, "K": K}, "weight": _randn(5, K),
            "residual": _randn(6, T, K, dtype=torch.float32), "gate": _randn(7, T, 1)}


def _stack_args(d):
    s = d["stack"]
    return s["a"], s["b"], s["rank"], s["scale"], d["ids"], list(s["widths"])


def _in_place(d, x):
    from liquidgemm_b200 import adapters
    y = d["y"] * 1.0
    assert adapters.add(y, x, d["stack"], d["ids"], inplace=True) is y
    return y


def _entries(d):
    """(name, entry point of x)"""
    from liquidgemm_b200 import adapters, norms
    more = dict(residual=d["residual"], post_weight=d["weight"], gate=d["gate"], scale=0.5, eps=1e-5)
    return [
        ("add", lambda x: adapters.add(d["y"], x, d["stack"], d["ids"])),
        ("linear", lambda x: adapters.linear(x, d["w4"], d["stack"], d["ids"], bias=d["bias"])),
        ("linear_int8", lambda x: adapters.linear(x, d["int8"], d["stack"], d["ids"], bias=d["bias"])),
        ("linear_int8_wide", lambda x: adapters.linear(x, d["int8"], d["stack"], d["ids"], out_dtype=torch.float32)),
        ("norm", lambda x: norms.block_norm(x, d["weight"], **more)),
        ("norm_quant", lambda x: norms.block_norm_quant(x, d["weight"], **more)),
        ("norm_alone", lambda x: norms.block_norm(x, None)[0]),
    ]


def _operators(d):
    return [
        ("add", torch.ops.liquidgemm.adapters_add, (d["y"], d["x"], *_stack_args(d))),
        ("norm", torch.ops.liquidgemm.block_norm, (d["x"], d["weight"], d["residual"], d["weight"], d["gate"], 1e-5, 0.5, 1.0, 0.0, False)),
        ("norm_quant", torch.ops.liquidgemm.block_norm, (d["x"], d["weight"], None, None, None, 1e-5, 1.0, 1.0, 0.0, True)),
    ]


def _same(a, b):
    a, b = (a, b) if isinstance(a, (tuple, list)) else ((a,), (b,))
    return len(a) == len(b) and all(torch.equal(u, v) and u.dtype == v.dtype for u, v in zip(a, b))


def test_operators_pass_the_checks_of_torch(data):
    """Schema, fake kernels and tracing."""
    for _, op, args in _operators(data):
        torch.library.opcheck(op.default, args)
    torch.library.opcheck(torch.ops.liquidgemm.adapters_add_.default, (data["y"].clone(), data["x"], *_stack_args(data)))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(data, backend):
    for name, entry in _entries(data) + [("in place", lambda x: _in_place(data, x))]:
        torch._dynamo.reset()
        assert _same(torch.compile(entry, backend=backend, fullgraph=True)(data["x"]), entry(data["x"])), name


def test_traced(data):
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, entry in _entries(data) + [("in place", lambda x: _in_place(data, x))]:
        graph = make_fx(entry)(data["x"])
        assert any(str(n.target).startswith("liquidgemm.") for n in graph.graph.nodes), name
        assert _same(graph(data["x"]), entry(data["x"])), name


def test_vmap(data):
    """A batch of calls: torch runs the operators once for each."""
    from liquidgemm_b200 import adapters
    x = torch.stack([data["x"], data["x"].flip(0), data["x"].roll(3, 0)])
    ids = torch.stack([data["ids"], data["ids"].flip(0)])
    bias = torch.stack([data["bias"], -data["bias"]])
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        for name, entry in _entries(data):
            if name.startswith("linear_int8"):   # the token quantiser gives a list, for which torch makes no loop: refused
                with pytest.raises(RuntimeError, match="quant_per_token"):
                    torch.vmap(entry)(x)
                continue
            want = [entry(b) for b in x]
            want = tuple(torch.stack(w) for w in zip(*want)) if isinstance(want[0], tuple) else torch.stack(want)
            assert _same(torch.vmap(entry)(x), want), name
        # what is batched is not the rows
        for layer in ("w4", "int8"):
            def call(i, b):
                return adapters.linear(data["x"], data[layer], data["stack"], i, bias=b)
            assert _same(torch.vmap(lambda i: call(i, None))(ids), torch.stack([call(i, None) for i in ids])), layer
            assert _same(torch.vmap(lambda b: call(data["ids"], b))(bias), torch.stack([call(data["ids"], b) for b in bias])), layer


def _outcome(call):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        try:
            out = call()
        except Exception as e:
            return type(e), str(e).split("\n")[0]
    return [(t.requires_grad, t.grad_fn is not None) for t in torch.utils._pytree.tree_leaves(out) if t.is_floating_point()]


def test_derivatives_as_the_registered_operators_have_them(data):
    """There are none: asked for, the entry points answer (or refuse) as the operators do, and the values are the same."""
    calls = {name: (op, args) for name, op, args in _operators(data)}
    at = {"add": 1, "norm": 0}
    for name, entry in _entries(data):
        want = entry(data["x"])
        leaf = data["x"].clone().requires_grad_()
        if name in at:
            op, args = calls[name]
            def direct(t):
                out = op(*args[:at[name]], t, *args[at[name] + 1:])
                return out if name == "add" else (out[0], out[2])
            assert _outcome(lambda: entry(leaf)) == _outcome(lambda: direct(leaf)), name
            assert _outcome(lambda: torch.func.jvp(entry, (data["x"],), (data["x"],))) == \
                _outcome(lambda: torch.func.jvp(direct, (data["x"],), (data["x"],))), name
        assert all(asks for asks, _ in _outcome(lambda: entry(leaf))), name   # (nothing passes for independent of x: backward says that there is no kernel)
        with torch.no_grad():
            assert _same(entry(leaf), want), name


@pytest.mark.parametrize("layer", ["w4", "int8"])
@pytest.mark.parametrize("what", ["a", "b", "scale"])
def test_gradients_of_the_stack_are_not_passed_over(data, layer, what):
    from liquidgemm_b200 import adapters
    stack = dict(data["stack"], **{what: data["stack"][what].clone().requires_grad_()})
    want = adapters.linear(data["x"], data[layer], data["stack"], data["ids"])
    got = adapters.linear(data["x"], data[layer], stack, data["ids"])
    assert got.requires_grad and torch.equal(got, want)
    with torch.no_grad():
        assert torch.equal(adapters.linear(data["x"], data[layer], stack, data["ids"]), want)
