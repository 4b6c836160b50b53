"""Layer norm alone: the kernels against the definition in 64 bits, element by element, within error bounds.

``u`` = 2^-24, ``r`` = 2^-8 for bf16 results, ``u`` for f32.  A row's sums add at most ``k`` terms in a chain (per thread, then
a tree).  mean: ``k u mean|x|``; the centred squares' sum: ``(k + 4) u`` relative plus the square of the mean's error; ``rstd``
half of that plus a few ``u``; the gradients' bounds follow from those by the product rule, see ``_bounds``.
"""
import pytest
import torch

U = 2.0 ** -24


def _bounds(x, w, b, dy, eps, bf16, w_bf16):
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    rows, d = x.shape
    k = 64 + -(-d // 1024)
    r, rw = (2.0 ** -8 if bf16 else U), (2.0 ** -8 if w_bf16 else U)
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = c.square().mean(1, keepdim=True)
    inv = 1 / torch.sqrt(var + eps)
    n = c * inv
    e_m = k * U * x.abs().mean(1, keepdim=True)
    e_r = 0.5 * ((k + 6) * U + e_m ** 2 / (var + eps)) + 4 * U
    e_n = inv * e_m + n.abs() * (e_r + 3 * U)
    y = n * w + b
    e_y = w.abs() * e_n + 2 * U * (n * w).abs() + (r + U) * (y.abs() + w.abs() * e_n)
    g = dy * w
    mg, mu = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    e_mg = (k + 2) * U * g.abs().mean(1, keepdim=True)
    e_mu = (k + 3) * U * (g * n).abs().mean(1, keepdim=True) + (g.abs() * e_n).mean(1, keepdim=True)
    dx = inv * (g - mg - n * mu)
    terms = g.abs() + mg.abs() + (n * mu).abs()
    e_dx = inv * (4 * U * terms + e_mg + e_n * mu.abs() + n.abs() * e_mu) + (e_r + 2 * U) * inv * terms
    e_dx = e_dx + r * (dx.abs() + e_dx)
    kr = 128                                  # rows per thread, groups of a workgroup, partial rows: at most 128 in all here
    dw, db = (dy * n).sum(0), dy.sum(0)
    e_dw = kr * U * (dy * n).abs().sum(0) + (dy.abs() * e_n).sum(0)
    e_db = kr * U * dy.abs().sum(0)
    return [(y, e_y), (dx, e_dx), (dw, e_dw + rw * (dw.abs() + e_dw)), (db, e_db + rw * (db.abs() + e_db))]


def _run(x, w, b, dy, eps=1e-5):
    from mitune.ops.layernorm import layer_norm
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    y = layer_norm(x, w, b, eps)
    return [y.detach()] + list(torch.autograd.grad(y, (x, w, b), dy))


def _check(got, bounds):
    for name, a, (v, e) in zip(("y", "dx", "dw", "db"), got, bounds):
        assert a.shape == v.shape
        worst = ((a.double() - v).abs() - e).max().item()
        assert worst <= 1e-37, (name, worst, e.max().item())


def _make(rows, d, dtype, pdtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + d)
    x = (torch.randn(rows, d, device="cuda", generator=g) * 2 + 1).to(dtype)
    w = (1 + 0.3 * torch.randn(d, device="cuda", generator=g)).to(pdtype)
    b = torch.randn(d, device="cuda", generator=g).to(pdtype)
    dy = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    return x, w, b, dy


KINDS = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pdtype", KINDS)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (7, 7), (70, 64), (5, 65), (33, 127), (4100, 96), (9, 255), (5000, 256), (17, 513),
                                    (2, 1024), (300, 1025), (65, 2048), (31, 2049), (12, 4100), (3, 8191), (5, 8193), (2, 16384),
                                    (3, 16385), (2, 32769), (70, 40001)])
def test_forward_and_gradients(dtype, pdtype, rows, d):
    x, w, b, dy = _make(rows, d, dtype, pdtype)
    _check(_run(x, w, b, dy), _bounds(x, w, b, dy, 1e-5, dtype == torch.bfloat16, pdtype == torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [96, 4100, 33000])
def test_a_large_mean_keeps_the_variance(d):
    """Rows of mean 1000 and unit spread: a difference of squares would lose the variance."""
    x, w, b, dy = _make(40, d, torch.float32, torch.float32)
    x = x + 1000
    _check(_run(x, w, b, dy), _bounds(x, w, b, dy, 1e-5, False, False))


@pytest.mark.gpu
def test_constant_rows_give_the_bias():
    from mitune.ops.layernorm import layer_norm
    for d in (5, 300, 3000):
        x = torch.full((3, d), 0.1, device="cuda")
        w, b = torch.randn(d, device="cuda"), torch.randn(d, device="cuda")
        y = layer_norm(x, w, b)
        # the mean is off by at most 64 u x, which 1 / sqrt(eps) magnifies
        assert (y - b).abs().max() <= 64 * U * 0.1 * 1e-5 ** -0.5 * w.abs().max() + 1e-6
        assert torch.equal(layer_norm(torch.zeros(2, d, device="cuda"), w, b), b.expand(2, d))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_missing_parameters_strides_and_shapes(dtype):
    from mitune.ops.layernorm import layer_norm
    x, w, b, dy = _make(60, 129, dtype, dtype)
    ones, zeros = torch.ones_like(w), torch.zeros_like(b)
    assert torch.equal(layer_norm(x), layer_norm(x, ones, zeros))
    assert torch.equal(layer_norm(x, w), layer_norm(x, w, zeros))
    assert torch.equal(layer_norm(x, None, b), layer_norm(x, ones, b))
    wide = torch.randn(60, 131, device="cuda").to(dtype)
    for view in (wide[:, 1:130], wide[:, :129], wide.t().contiguous().t()[:, :129], x.view(3, 4, 5, 129), x[0],
                 x[:1].expand(60, 129)):
        got = layer_norm(view, w, b)
        assert got.shape == view.shape and torch.equal(got, layer_norm(view.contiguous(), w, b))
    # an upstream gradient with rows apart, one whose columns are apart, and one expanded from a scalar
    ref = _run(x, w, b, dy)
    spread = torch.zeros(60, 140, device="cuda", dtype=dtype)
    spread[:, 3:132] = dy
    flipped = dy.t().contiguous().t()
    for other in (spread[:, 3:132], flipped):
        for a, e in zip(_run(x, w, b, other), ref):
            assert torch.equal(a, e)
    one = torch.ones((), device="cuda", dtype=dtype).expand(60, 129)
    for a, e in zip(_run(x, w, b, one), _run(x, w, b, one.contiguous())):
        assert torch.equal(a, e)


@pytest.mark.gpu
def test_only_the_wanted_gradients():
    from mitune.ops.layernorm import layer_norm
    x, w, b, dy = _make(50, 300, torch.float32, torch.float32)
    want = _run(x, w, b, dy)
    for flags in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(f)) for t, f in zip((x, w, b), flags)]
        layer_norm(*leaves).backward(dy)
        for leaf, f, e in zip(leaves, flags, want[1:]):
            assert (leaf.grad is not None) == bool(f) and (not f or torch.equal(leaf.grad, e))


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences in f32 with step 1e-2 along random directions: curvature e^2 and the sum's rounding over e, both well
    below 2e-3 of the function's norm."""
    from mitune.ops.layernorm import layer_norm
    x, w, b, dy = _make(20, 37, torch.float32, torch.float32)
    grads = _run(x, w, b, dy)[1:]
    g = torch.Generator(device="cuda").manual_seed(2)
    f = lambda a: (layer_norm(*a).double() * dy.double()).sum().item()          # noqa: E731
    size = (layer_norm(x, w, b).double() * dy.double()).norm().item()
    for i in range(3):
        step = torch.randn((x, w, b)[i].shape, device="cuda", generator=g)
        hi, lo = [x, w, b], [x, w, b]
        hi[i], lo[i] = hi[i] + 1e-2 * step, lo[i] - 1e-2 * step
        slope = (f(hi) - f(lo)) / 2e-2
        assert abs(slope - (grads[i].double() * step.double()).sum().item()) < 2e-3 * size * 37 ** 0.5


@pytest.mark.gpu
def test_rows_do_not_mix_and_results_repeat():
    x, w, b, dy = _make(4200, 200, torch.bfloat16, torch.float32)
    ref = _run(x, w, b, dy)
    for a, e in zip(_run(x, w, b, dy), ref):
        assert torch.equal(a, e)
    x[77], dy[78] = float("nan"), float("inf")
    got = _run(x, w, b, dy)
    keep = torch.ones(4200, dtype=torch.bool, device="cuda")
    keep[77:79] = False
    assert torch.equal(got[0][keep], ref[0][keep]) and torch.equal(got[1][keep], ref[1][keep])
    assert got[0][77].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", [(50, 96), (5000, 2100), (3, 40001)])
def test_captured_passes_replay_like_eager_ones(rows, d):
    from mitune.ops.layernorm import layer_norm
    x, w, b, dy = _make(rows, d, torch.float32, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
        y = y.detach()
    for seed in range(3):
        new = _make(rows, d, torch.float32, torch.float32, seed=seed + 5)
        for t, n in zip(leaves + [dy], new):
            t.data.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip([y] + list(grads), _run(*new)):
            assert torch.equal(a, e)


@pytest.mark.gpu
def test_empty_rows_and_gpu_refusals():
    from mitune.ops.layernorm import layer_norm
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == (0, 8) and grads[0].shape == (0, 8) and not grads[1].any() and not grads[2].any()
    with pytest.raises(TypeError):
        layer_norm(torch.zeros(2, 8, device="cuda", dtype=torch.float16))
    with pytest.raises(TypeError):
        layer_norm(torch.zeros(2, 8, device="cuda"), torch.ones(8))


def test_arguments_are_checked():
    from mitune.ops.layernorm import layer_norm
    x = torch.zeros(3, 8)
    for w, b in ((torch.ones(7), None), (None, torch.zeros(1, 8))):
        with pytest.raises(ValueError):
            layer_norm(x, w, b)
    with pytest.raises(TypeError):
        layer_norm(x, torch.ones(8, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        layer_norm(x.bfloat16(), torch.ones(8), torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(()))


def test_the_cpu_form_is_layer_norm():
    from mitune.ops.layernorm import layer_norm
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(5, 33, generator=g), torch.randn(33, generator=g), torch.randn(33, generator=g)
    assert torch.allclose(layer_norm(x, w, b), torch.nn.functional.layer_norm(x, (33,), w, b))
    y = layer_norm(x.bfloat16(), w, b)
    assert y.dtype == torch.bfloat16 and torch.allclose(y.float(), layer_norm(x.bfloat16().float(), w, b), atol=2.0 ** -6)
