"""The registered operators of the expert layers on the device, and the entry points wherever these have to go through them: compiled,
traced and transformed calls, gradients asked for.  The results are the entry points' own, bit for bit."""

import warnings

import pytest
import torch

from test_gpu_experts import _gen, _ids, _layer, _rows, _stack

pytestmark = pytest.mark.gpu

T, E, K, H, INNER = 21, 6, 2, 256, 128


@pytest.fixture(scope="module")
def moe():
    from liquidgemm_b200 import moe as _moe
    return _moe


@pytest.fixture(scope="module")
def data(moe):
    w13, w2 = _layer(moe, E, H, INNER, True, 3)
    d = {"logits": torch.randn(T, E, device="cuda", generator=_gen(1)), "bias": torch.randn(E, device="cuda", generator=_gen(2)) * 0.1,
         "x": _rows((T, H), torch.bfloat16, 4), "ids": _ids(T, E, K, 5), "weights": torch.rand(T, K, device="cuda", generator=_gen(6)),
         "w13": w13, "w2": w2, "one": _stack(moe, E, 192, H, False, 7)[0]}
    d["xq"] = torch.randint(-127, 128, (T, H), device="cuda", generator=_gen(8)).to(torch.int8)
    d["ascale"] = torch.rand(T, device="cuda", generator=_gen(9))
    return d


def _calls(moe, d):
    """(name, entry point of its first argument, registered operator of all, the operator's arguments)"""
    one, w13, w2 = d["one"], d["w13"], d["w2"]
    ops = torch.ops.liquidgemm
    return [
        ("route", lambda l: moe.route(l, K, scoring="sigmoid", bias=d["bias"], n_group=3, topk_group=2, group_score="top2", scale=2.5),
         ops.moe_route, (d["logits"], d["bias"], K, 1, 3, 2, 1, True, 2.5)),
        ("linear", lambda x: moe.experts_linear(x, d["ids"], one), ops.experts_linear,
         (d["x"], None, d["ids"], one["w"], one["s1"], one["N"], one["K"], 0)),
        ("linear_int8", lambda x: moe.experts_linear(x, d["ids"], one, ascale=d["ascale"], out_dtype=torch.float32), ops.experts_linear,
         (d["xq"], d["ascale"], d["ids"], one["w"], one["s1"], one["N"], one["K"], 2)),
        ("mlp", lambda x: moe.experts_mlp(x, d["weights"], d["ids"], w13, w2), ops.experts_mlp,
         (d["x"], d["weights"], d["ids"], w13["w"], w13["s1"], w2["w"], w2["s1"], 0)),
    ]


def _same(a, b):
    a, b = (a, b) if isinstance(a, (tuple, list)) else ((a,), (b,))
    return len(a) == len(b) and all(torch.equal(u, v) and u.dtype == v.dtype for u, v in zip(a, b))


def test_registered_operators(moe, data):
    for name, entry, op, args in _calls(moe, data):
        assert _same(entry(args[0]), op(*args)), name


def test_operators_pass_the_checks_of_torch(moe, data):
    """Schema, fake kernels and tracing."""
    for _, _, op, args in _calls(moe, data):
        torch.library.opcheck(op.default, args)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(moe, data, backend):
    for name, entry, _, args in _calls(moe, data):
        torch._dynamo.reset()
        assert _same(torch.compile(entry, backend=backend, fullgraph=True)(args[0]), entry(args[0])), name


def test_traced(moe, data):
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, entry, op, args in _calls(moe, data):
        graph = make_fx(entry)(args[0])
        assert op.default in [n.target for n in graph.graph.nodes], name
        assert _same(graph(args[0]), entry(args[0])), name


def test_vmap(moe, data):
    """A batch of calls: torch runs the operator once for each."""
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        for name, entry, _, args in _calls(moe, data):
            batch = torch.stack([args[0], args[0].flip(0), args[0].roll(3, 0)])
            got, want = torch.vmap(entry)(batch), [entry(b) for b in batch]
            if name == "route":
                want = tuple(torch.stack([w[i] for w in want]) for i in range(2))
            else:
                want = torch.stack(want)
            assert _same(got, want), name
        # what is batched is another argument than the first
        weights = torch.stack([data["weights"], data["weights"] * 2])
        got = torch.vmap(lambda w: moe.experts_mlp(data["x"], w, data["ids"], data["w13"], data["w2"]))(weights)
        assert _same(got, torch.stack([moe.experts_mlp(data["x"], w, data["ids"], data["w13"], data["w2"]) for w in weights]))


def _outcome(call):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        try:
            out = call()
        except Exception as e:
            return type(e), str(e).split("\n")[0]
    return [(t.requires_grad, t.grad_fn is not None) for t in torch.utils._pytree.tree_leaves(out) if t.is_floating_point()]


def test_derivatives_as_the_registered_operators_have_them(moe, data):
    """There are none: asked for, the entry points answer (or refuse) as the operators do, and the values are the same."""
    for name, entry, op, args in _calls(moe, data):
        if not args[0].is_floating_point():
            continue
        want = entry(args[0])
        leaf = args[0].clone().requires_grad_()
        assert _outcome(lambda: entry(leaf)) == _outcome(lambda: op(leaf, *args[1:])), name
        with torch.no_grad():
            assert _same(entry(leaf), want), name
        assert _outcome(lambda: torch.func.jvp(entry, (args[0],), (args[0],))) == \
            _outcome(lambda: torch.func.jvp(lambda t: op(t, *args[1:]), (args[0],), (args[0],))), name


def test_parameters_are_ordinary(moe, data):
    layer = dict(data["one"], w=torch.nn.Parameter(data["one"]["w"], requires_grad=False), s1=torch.nn.Parameter(data["one"]["s1"], requires_grad=False))
    assert moe._plain_call(data["x"], layer["w"], layer["s1"], None)
    assert torch.equal(moe.experts_linear(data["x"], data["ids"], layer), moe.experts_linear(data["x"], data["ids"], data["one"]))
