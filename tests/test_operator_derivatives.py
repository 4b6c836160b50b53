"""Derivatives of the long-sequence operators by other ways than one plain backward pass: graphs of gradients over operands that
share a tensor or depend on each other.

Bounds: ``u`` = 2^-24.  Both sides of a comparison are f32 sums of at most ``n`` terms of size at most one step of the formula; the
tests take operands of order one and allow ``1e-4`` of the largest gradient, thousands of ``u`` for sums of a hundred terms, where a
doubled path is an error of the gradient's own size.  In 64 bits the bound is ``1e-12``.
"""
import pytest
import torch


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
