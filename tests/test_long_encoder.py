"""The encoder-block operators as they are used together, and the models that reach them past the short kernels' 128 tokens.

f32 tolerances: one product over K terms is off by at most (K + 3) 2^-24 of its absolute sum, 1.6e-5 at K = 256, and by about
sqrt(K) 2^-24 = 1e-6 of its value as errors of either sign add up; ten such operations in a row stay below 2e-5 of a tensor's norm.
bf16: every operation rounds its result, and p, ds and dz inside, by at most 2^-8, 1.7e-3 on average; ten in a row, adding as
squares, 5.4e-3, and gradients pass forward and backward: 1.6e-2 of a tensor's norm is three times what both together come to."""
import math

import pytest
import torch

NAMES = ("w_n1", "b_n1", "w_qkv", "b_qkv", "w_o", "b_o", "w_n2", "b_n2", "w_up", "b_up", "w_down", "b_down")


def _block(x, P, pack, h, hk, d, norm, linear, attention):
    """A pre-norm block with grouped heads on packed rows, written once for both sides."""
    y = norm(x, P["w_n1"], P["b_n1"])
    qkv = linear(y, P["w_qkv"], P["b_qkv"], None, None)
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], dim=1))
    o = attention(q, k, v, pack).reshape(x.shape[0], h * d)
    x = linear(o, P["w_o"], P["b_o"], None, x)
    y = norm(x, P["w_n2"], P["b_n2"])
    return linear(linear(y, P["w_up"], P["b_up"], "gelu", None), P["w_down"], P["b_down"], None, x)


def _plain_norm(x, w, b):
    c = x - x.mean(-1, keepdim=True)
    return c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * w + b


def _plain_linear(x, w, b, act, r):
    z = x @ w.T + b
    z = 0.5 * z * (1 + torch.erf(z / math.sqrt(2))) if act == "gelu" else z
    return z if r is None else z + r


def _plain_attention(lengths):
    def run(q, k, v, _):
        out, at = [], 0
        group = q.shape[1] // k.shape[1]
        for n in lengths:
            Q, K, V = (t[at:at + n].transpose(0, 1) for t in (q, k, v))
            s = Q @ K.repeat_interleave(group, 0).transpose(1, 2) / math.sqrt(q.shape[2])
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
            out.append((torch.softmax(s, -1) @ V.repeat_interleave(group, 0)).transpose(0, 1))
            at += n
        return torch.cat(out)
    return run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 1.6e-2)])
@pytest.mark.parametrize("lengths,h,hk,d,ff", [([200, 3, 129, 1], 4, 2, 32, 256), ([500, 77], 4, 4, 64, 200)])
def test_a_block_of_the_operators(dtype, tol, lengths, h, hk, d, ff):
    from mitune.ops.attention import SequencePack, packed_attention
    from mitune.ops.layernorm import layer_norm
    from mitune.ops.linear import linear
    g = torch.Generator(device="cuda").manual_seed(len(lengths))
    E, rows = h * d, sum(lengths)
    new = lambda *s, k=1.0: (torch.randn(*s, device="cuda", generator=g) * k).to(dtype)          # noqa: E731
    W = (h + 2 * hk) * d
    shapes = [(E,), (E,), (W, E), (W,), (E, E), (E,), (E,), (E,), (ff, E), (ff,), (E, ff), (E,)]
    P = {n: (new(*s, k=s[1] ** -0.5) if len(s) == 2 else new(*s, k=0.1)) for n, s in zip(NAMES, shapes)}
    P["w_n1"], P["w_n2"] = P["w_n1"] + 1, P["w_n2"] + 1
    x, dy = new(rows, E), new(rows, E)

    def run(cast, *ops):
        leaves = [cast(x).detach().requires_grad_()] + [cast(P[n]).detach().requires_grad_() for n in NAMES]
        y = _block(leaves[0], dict(zip(NAMES, leaves[1:])), SequencePack(lengths), h, hk, d, *ops)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, cast(dy)))

    own = run(lambda t: t, layer_norm, lambda a, w, b, act, r: linear(a, w, b, activation=act, residual=r),
              lambda q, k, v, p: packed_attention(q, k, v, p, causal=True))
    ref = run(lambda t: t.double(), _plain_norm, _plain_linear, _plain_attention(lengths))
    for name, a, e in zip(("y", "x") + NAMES, own, ref):
        if name == "b_qkv":       # a key bias moves every score of a row alike: its gradient is zero up to rounding
            a, e = (torch.cat([t[:h * d], t[(h + hk) * d:]]) for t in (a, e))
        assert ((a.double() - e).norm() / e.norm()).item() < tol, name


@pytest.mark.gpu
@pytest.mark.parametrize("S", [100, 200, 333])
def test_the_configurable_model_past_128_tokens(S):
    """f32 on the kernels against the same module in f64 on the CPU, output and every gradient."""
    from mitune.models.transformer import TransformerModel
    torch.manual_seed(3)
    m = TransformerModel(input_size=9, num_heads=2, num_encoder_layers=2, d_model=256 if S == 100 else 64, dim_feedforward=128,
                         dropout=0.0, key_dim_scaling=0.5)
    x = torch.randn(3, S, 9)
    ref = m.double()
    want = ref(x.double())
    want.sum().backward()
    grads = {n: p.grad.clone() for n, p in ref.named_parameters()}
    own = m.float().cuda()
    own.zero_grad()
    got = own(x.cuda())
    got.sum().backward()
    assert torch.allclose(got.double().cpu(), want, rtol=1e-4, atol=1e-5)
    scale = max(g.norm().item() for g in grads.values())
    for n, p in own.named_parameters():
        assert (p.grad.double().cpu() - grads[n]).norm().item() < 2e-4 * (grads[n].norm().item() + 1e-2 * scale), n


@pytest.mark.gpu
def test_long_self_attention_reaches_the_kernels():
    from mitune.ops.attention import attention_reference, self_attention, self_attention_qkv
    g = torch.Generator(device="cuda").manual_seed(2)
    B, S, h, dk, dv = 2, 300, 2, 16, 32
    qkv = torch.randn(B, S, h * (2 * dk + dv), device="cuda", generator=g, requires_grad=True)
    do = torch.randn(B, S, h * dv, device="cuda", generator=g)
    o = self_attention_qkv(qkv, h, dk)
    (a,) = torch.autograd.grad(o, qkv, do)
    q, k, v = qkv.detach().double().split([h * dk, h * dk, h * dv], -1)
    leaves = [t.unflatten(2, (h, -1)).transpose(1, 2).requires_grad_() for t in (q, k, v)]
    ref = attention_reference(*leaves)
    grads = torch.autograd.grad(ref, leaves, do.double().unflatten(2, (h, dv)).transpose(1, 2))
    want = torch.cat([t.transpose(1, 2).flatten(2) for t in grads], -1)
    assert torch.allclose(o.double(), ref.transpose(1, 2).flatten(2), rtol=1e-4, atol=1e-5)
    assert torch.allclose(a.double(), want, rtol=1e-4, atol=1e-4)
    qk, vv = qkv.detach().split([2 * h * dk, h * dv], -1)
    assert torch.equal(self_attention(qk, vv, h), o.detach())
    assert self_attention_qkv(qkv.detach(), h, dk, kind="relu").shape == o.shape          # the plain forms stay for the rest
    assert self_attention_qkv(qkv.detach(), h, dk, dropout_p=0.5).shape == o.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 96), (torch.float32, 2100), (torch.float32, 33)])
def test_residual_norms_outside_the_fused_kernels(dtype, d):
    from mitune.ops.layernorm import residual_layer_norm
    g = torch.Generator(device="cuda").manual_seed(d)
    x, r, w, b = (torch.randn(*s, device="cuda", generator=g).to(dtype).requires_grad_() for s in ((20, d), (20, d), (d,), (d,)))
    y = residual_layer_norm(x, r, w, b)
    assert y.dtype == dtype and "LayerNorm" in type(y.grad_fn).__name__ and "NativeLayerNorm" not in type(y.grad_fn).__name__
    ref = torch.nn.functional.layer_norm((x + r).double(), (d,), w.double(), b.double())
    assert torch.allclose(y.double(), ref, rtol=2 * torch.finfo(dtype).eps, atol=1e-2 if dtype == torch.bfloat16 else 1e-5)
    y.sum().backward()
    assert all(t.grad is not None for t in (x, r, w, b))


def _twice(f, inputs, a, b):
    """Gradients of b . (the gradients of a . f): second derivatives of every operand."""
    inputs = [t.detach().requires_grad_() for t in inputs]
    first = torch.autograd.grad(f(*inputs), inputs, a, create_graph=True)
    return torch.autograd.grad(sum((g * w).sum() for g, w in zip(first, b)), inputs, allow_unused=True)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["attention", "attention padded", "norm", "linear gelu", "linear relu"])
def test_gradients_of_gradients(what):
    """Penalties on a gradient differentiate the backward pass.  Sums of at most 40 terms, three inside one another: 3 x 43 x 2^-24
    = 8e-6 of their absolute sums, which are less than 30 times their values here: 2.4e-4 of a tensor's norm."""
    from mitune.ops.attention import SequencePack, packed_attention
    from mitune.ops.layernorm import layer_norm
    from mitune.ops.linear import linear
    g = torch.Generator().manual_seed(11)
    new = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).float().double()          # noqa: E731
    if what.startswith("attention"):
        d = 6 if what.endswith("padded") else 8
        make = lambda dev: (lambda q, k, v: packed_attention(q, k, v, SequencePack([5, 1, 9], rows=17, device=dev), True))     # noqa: E731
        inputs, out = (new(17, 4, d), new(17, 2, d), new(17, 2, d)), (17, 4, d)
    elif what == "norm":
        make = lambda dev: (lambda x, w, b: layer_norm(x, w, b))          # noqa: E731
        inputs, out = (new(7, 37), new(37), new(37)), (7, 37)
    else:
        make = lambda dev: (lambda x, w, b, r: linear(x, w, b, activation=what.split()[1], residual=r))          # noqa: E731
        inputs, out = (new(9, 33), new(19, 33), new(19), new(9, 19)), (9, 19)
    a, b = new(*out), [new(*t.shape) for t in inputs]
    want = _twice(make("cpu"), inputs, a, b)
    gpu = lambda t: t.float().cuda()          # noqa: E731
    got = _twice(make("cuda"), [gpu(t) for t in inputs], gpu(a), [gpu(t) for t in b])
    for x, y in zip(got, want):
        if y is None or y.norm() == 0:
            assert x is None or x.norm() == 0
        else:
            assert (x.double().cpu() - y).norm() <= 2.4e-4 * y.norm()
