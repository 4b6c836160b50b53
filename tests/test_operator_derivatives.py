"""Derivatives of the long-sequence operators by other ways than one plain backward pass: graphs of gradients over operands that
share a tensor or depend on each other, forward-mode differentiation, ``torch.func`` transforms, batched gradients.

Bounds: ``u`` = 2^-24.  Both sides of a comparison are f32 sums of at most ``n`` terms of size at most one step of the formula; the
tests take operands of order one and allow ``1e-4`` of the largest gradient, thousands of ``u`` for sums of a hundred terms, where a
doubled path is an error of the gradient's own size.  In 64 bits the bound is ``1e-12``.
"""
import pytest
import torch
import torch.autograd.forward_ad as fw


def _ties(x, y, z):
    """Operand triples of one shape: apart, shared, and computed from one another."""
    return {"apart": (x, y, z), "q is k": (x, x, z), "k is v": (x, y, y), "all": (x, x, x), "v of k": (x, y, (2 * y).tanh()),
            "k of q": (x, x * x + y, z), "chain": (x, x.sin(), x.sin().exp())}


@pytest.mark.parametrize("tie", list(_ties(*torch.zeros(3, 1))))
def test_formula_gradients_belong_to_their_places(tie):
    """What autograd adds up over the places of shared operands is the plain gradient, and so is what it differentiates again."""
    from mitune.ops import lib as L
    from mitune.ops.attention import SequencePack, packed_attention_reference
    pack = SequencePack([3, 0, 4], device="cpu")
    formula = lambda q, k, v: packed_attention_reference(q, k, v, pack, True, 0.5)          # noqa: E731

    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v):
            ctx.save_for_backward(q, k, v)
            return formula(q, k, v)

        @staticmethod
        def backward(ctx, g):
            return tuple(L.grads_by_formula(formula, ctx.saved_tensors, g))

    g = torch.Generator().manual_seed(1)
    leaves = [torch.randn(7, 2, 4, dtype=torch.float64, generator=g).requires_grad_() for _ in range(3)]
    dy, dg = (torch.randn(7, 2, 4, dtype=torch.float64, generator=g) for _ in range(2))
    results = []
    for op in (formula, Op.apply):
        out = op(*_ties(*leaves)[tie])
        first = torch.autograd.grad(out, leaves, dy, create_graph=True, allow_unused=True)
        second = torch.autograd.grad(first[0], leaves, dg, allow_unused=True)
        results.append([t for t in first + second if t is not None])
    assert len(results[0]) == len(results[1])
    for a, b in zip(*results):
        assert (a - b).abs().max().item() <= 1e-12


def _same_with_and_without_a_graph(call, leaves, dy):
    with_graph = torch.autograd.grad(call(*leaves), leaves, dy, create_graph=True)
    without = torch.autograd.grad(call(*leaves), leaves, dy)
    for a, b in zip(with_graph, without):
        assert (a - b).abs().max().item() <= 1e-4 * b.abs().max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("tie", list(_ties(*torch.zeros(3, 1))))
def test_shared_operands_of_attention(tie):
    from mitune.ops.attention import SequencePack, packed_attention
    g = torch.Generator(device="cuda").manual_seed(2)
    leaves = [torch.randn(50, 2, 16, device="cuda", generator=g).requires_grad_() for _ in range(3)]
    used = {"q is k": (0, 2), "k is v": (0, 1), "all": (0,), "v of k": (0, 1), "chain": (0,)}.get(tie, (0, 1, 2))
    pack = SequencePack([30, 17], rows=50)
    dy = torch.randn(50, 2, 16, device="cuda", generator=g)

    def call(*mine):
        full = list(leaves)
        for i, t in zip(used, mine):
            full[i] = t
        return packed_attention(*_ties(*full)[tie], pack, causal=True)

    _same_with_and_without_a_graph(call, [leaves[i] for i in used], dy)


@pytest.mark.gpu
def test_shared_operands_of_the_norm_and_the_dense_layer():
    from mitune.ops.layernorm import layer_norm
    from mitune.ops.linear import linear
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randn(40, 40, device="cuda", generator=g).requires_grad_() for _ in range(2))
    b = torch.randn(40, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(40, 40, device="cuda", generator=g)
    _same_with_and_without_a_graph(lambda x, b: layer_norm(x, b, b), [x, b], dy)
    _same_with_and_without_a_graph(lambda x: layer_norm(x, x[0], x.mean(0)), [x], dy)
    _same_with_and_without_a_graph(lambda x: linear(x, x, activation="gelu"), [x], dy)
    _same_with_and_without_a_graph(lambda x, w: linear(x, x @ w, w[0], activation="gelu", residual=x), [x, w], dy)
    _same_with_and_without_a_graph(lambda w: linear(w.tanh(), w, w.sum(1), residual=w), [w], dy)


@pytest.mark.filterwarnings("ignore:.torch.jit:DeprecationWarning")
def test_transforms_are_seen():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from mitune.ops.lib import transformed
    x, seen = torch.randn(3), []

    def look(t):
        seen.append(transformed(None, t))
        return t * 2

    assert not transformed(x, None) and not transformed(x.clone().requires_grad_())
    torch.func.vmap(look)(torch.randn(2, 3))
    torch.func.jvp(look, (x,), (x,))
    torch.func.grad(lambda t: look(t).sum())(x)
    torch.func.hessian(lambda t: (look(t) ** 3).sum())(x)
    torch.jit.trace(look, x, check_trace=False)
    with FakeTensorMode():
        look(torch.empty(3))
    with fw.dual_level():
        look(fw.make_dual(x, x))
        assert not transformed(x)
    with torch.no_grad(), fw.dual_level():
        look(fw.make_dual(x, x))
    assert len(seen) == 8 and all(seen)
    assert not transformed(x)


def _tangent(f, args, at):
    with fw.dual_level():
        out = f(*(fw.make_dual(a, t) for a, t in zip(args, at)))
        return fw.unpack_dual(out).tangent


@pytest.mark.parametrize("way", ["tangent", "batched"])
def test_formula_gradients_of_transformed_gradients(way):
    """The gradients are linear in the upstream gradient: their tangent along ``t`` is the gradient for ``t``."""
    from mitune.ops import lib as L
    formula = lambda q, k, v: (torch.tanh(q @ k.T) @ v)          # noqa: E731

    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, *t):
            ctx.save_for_backward(*t)
            return formula(*t)

        @staticmethod
        def backward(ctx, g):
            assert not torch.is_grad_enabled() and L.formula_backward(g)
            return tuple(L.grads_by_formula(formula, ctx.saved_tensors, g))

    leaves = [torch.randn(5, 5, dtype=torch.float64).requires_grad_() for _ in range(3)]
    dys = torch.randn(3, 5, 5, dtype=torch.float64)
    want = [torch.autograd.grad(formula(*leaves), leaves, dy) for dy in dys]
    if way == "batched":
        got = torch.autograd.grad(Op.apply(*leaves), leaves, dys, is_grads_batched=True)
        for i, w in enumerate(want):
            assert all((a[i] - b).abs().max().item() <= 1e-12 for a, b in zip(got, w))
    else:
        with fw.dual_level():
            got = torch.autograd.grad(Op.apply(*leaves), leaves, fw.make_dual(dys[0], dys[1]))
            parts = [fw.unpack_dual(t) for t in got]
        for p, a, b in zip(parts, *want[:2]):
            assert not p.primal.requires_grad
            assert (p.primal - a).abs().max().item() <= 1e-12 and (p.tangent - b).abs().max().item() <= 1e-12


def _calls():
    """(call on operands, its operands' shapes) of every operator that goes through plain torch under a transform; the first two were
    plain torch before their kernels were there."""
    from mitune.ops.attention import SequencePack, packed_attention, self_attention
    from mitune.ops.layernorm import layer_norm, residual_layer_norm
    return {
        "self_attention": (lambda qk, v: self_attention(qk, v, 2), [(2, 150, 32), (2, 150, 16)]),
        "residual_layer_norm": (residual_layer_norm, [(20, 2050), (20, 2050), (2050,), (2050,)]),
        "packed_attention": (lambda q, k, v: packed_attention(q, k, v, SequencePack([30, 17], rows=50, device=q.device), True),
                             [(50, 4, 16), (50, 2, 16), (50, 2, 16)]),
        "layer_norm": (layer_norm, [(20, 50), (50,), (50,)]),
    }


def _operands(shapes, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g) for s in shapes]


def _near(a, b):
    assert a.shape == b.shape
    assert (a.cpu().double() - b.double()).abs().max().item() <= 1e-4 * b.abs().max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(_calls()))
def test_forward_mode_and_func_transforms(name):
    """Against the CPU's plain form in 64 bits, under every transform."""
    call, shapes = _calls()[name]
    xs, ts = _operands(shapes, 4), _operands(shapes, 5)
    cpu = [[t.double() for t in group] for group in (xs, ts)]
    gpu = [[t.cuda() for t in group] for group in (xs, ts)]
    want = _tangent(call, *cpu)
    _near(_tangent(call, *gpu), want)
    _near(torch.func.jvp(call, *map(tuple, gpu))[1], want)
    with torch.no_grad():
        _near(_tangent(call, *gpu), want)
    one = lambda args: lambda *first: call(*first, *args[1:]).square().sum()          # noqa: E731
    _near(torch.func.grad(one(gpu[0]))(gpu[0][0]), torch.func.grad(one(cpu[0]))(cpu[0][0]))
    over = lambda group: torch.func.vmap(lambda t: call(t, *group[0][1:]))(torch.stack([group[0][0], group[1][0]]))          # noqa: E731
    _near(over(gpu), over(cpu))
    weights = [t.clone().requires_grad_() for t in gpu[0]]          # leaves beside the transformed operand
    _near(torch.func.vmap(lambda t: call(t, *weights[1:]))(torch.stack([gpu[0][0], gpu[1][0]])).detach(), over(cpu))


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(_calls()) + ["linear"])
def test_transformed_upstream_gradients(name):
    """Gradients are linear in the upstream gradient, one by one, batched, or along a tangent."""
    from mitune.ops.linear import linear
    calls = _calls()
    calls["linear"] = (lambda x, w, b, r: linear(x, w, b, activation="gelu", residual=r), [(20, 50), (30, 50), (30,), (20, 30)])
    call, shapes = calls[name]
    leaves = [t.cuda().requires_grad_() for t in _operands(shapes, 6)]
    out = call(*leaves)
    dys = torch.randn(3, *out.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
    want = [torch.autograd.grad(out, leaves, dy, retain_graph=True) for dy in dys]
    got = torch.autograd.grad(out, leaves, dys, is_grads_batched=True, retain_graph=True)
    for i, w in enumerate(want):
        for a, b in zip(got, w):
            _near(a[i], b.cpu())
    with fw.dual_level():
        for d, a, b in zip(torch.autograd.grad(out, leaves, fw.make_dual(dys[0], dys[1])), *want[:2]):
            primal, tangent = fw.unpack_dual(d)
            _near(primal, a.cpu())
            _near(tangent, b.cpu())


@pytest.mark.gpu
def test_dense_layers_refuse_transforms():
    from mitune.ops.linear import linear
    x, w, r = (t.cuda() for t in _operands([(20, 50), (30, 50), (20, 30)], 8))
    for kwargs in ({}, {"activation": "relu"}, {"residual": r}, {"activation": "gelu", "residual": r}):
        call = lambda t: linear(t, w, **kwargs)          # noqa: E731,B023
        with pytest.raises(NotImplementedError, match="jvp"):
            _tangent(call, [x], [x])
        with pytest.raises(RuntimeError, match="functorch transforms"):
            torch.func.jvp(call, (x,), (x,))
        with pytest.raises(RuntimeError, match="functorch transforms"):
            torch.func.vmap(lambda t: call(t[None])[0] if "residual" not in kwargs else linear(t, w, residual=r[0]))(x)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:.torch.jit:DeprecationWarning", "ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", list(_calls()))
def test_a_traced_call_computes(name):
    call, shapes = _calls()[name]
    first, second = ([t.cuda() for t in _operands(shapes, seed)] for seed in (9, 10))
    with torch.no_grad():
        traced = torch.jit.trace(call, tuple(first), check_trace=False)
        _near(traced(*second), call(*second).cpu())


def test_formula_gradients_under_autocast_keep_their_precision():
    """Under autocast a product of f32 matrices would be rounded to bf16: 2^-9 of its terms instead of 2^-24."""
    from mitune.ops import lib as L
    formula = lambda a, b: torch.tanh(a @ b)          # noqa: E731
    a, b = (torch.randn(20, 20, generator=torch.Generator().manual_seed(s)).requires_grad_() for s in (1, 2))
    dy = torch.ones(20, 20)
    want = L.grads_by_formula(formula, (a, b), dy)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = L.grads_by_formula(formula, (a, b), dy)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
def test_second_derivatives_and_tangents_under_autocast():
    from mitune.ops.attention import SequencePack, packed_attention
    g = torch.Generator(device="cuda").manual_seed(12)
    ops, ts = ([torch.randn(50, 2, 16, device="cuda", generator=g) for _ in range(3)] for _ in range(2))
    pack = SequencePack([30, 20])
    call = lambda *t: packed_attention(*t, pack, causal=True)          # noqa: E731
    leaves = [t.clone().requires_grad_() for t in ops]
    dy = torch.randn(50, 2, 16, device="cuda", generator=g)
    want, tangent = torch.autograd.grad(call(*leaves), leaves, dy, create_graph=True), _tangent(call, ops, ts)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got, other = torch.autograd.grad(call(*leaves), leaves, dy, create_graph=True), _tangent(call, ops, ts)
    for a, b in zip((*got, other), (*want, tangent)):
        _near(a.detach(), b.detach().cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["self_attention", "residual_layer_norm"])
def test_compiled_calls_stay_one_graph(name):
    call, shapes = _calls()[name]
    args = [t.cuda() for t in _operands(shapes, 11)]
    torch._dynamo.reset()
    _near(torch.compile(call, backend="eager", fullgraph=True)(*args), call(*args).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_types_are_refused_under_transforms_too(dtype):
    from mitune.ops.layernorm import layer_norm
    x = torch.randn(3, 8, device="cuda").to(dtype)
    for call in (layer_norm, torch.func.vmap(layer_norm), lambda t: torch.func.jvp(layer_norm, (t,), (t,))):
        with pytest.raises(TypeError, match="f32 or bf16"):
            call(x)
