"""The dense layer with its activation and residual in the epilogue, against the formulas in 64 bits within error bounds.

``u`` = 2^-24, ``r`` = 2^-8 for bf16 tensors.  ``z``: a chain of ``K`` products and the bias, ``(K + 3) u`` of the absolute sum.
``act`` has slope at most 1.13 (gelu) and its erf a few ``u``; ``y`` is rounded once.  ``act'`` changes by at most 0.8 per unit of
its argument, which is ``z`` rounded to the tensors' type; ``dz`` is rounded to that type; the gradients are sums of ``dz`` times
an operand, over ``N`` or ``M`` terms.  ReLU is tested on whole numbers, where ``z`` is exact and its sign never in doubt.
"""
import math

import pytest
import torch

U = 2.0 ** -24


def _formula(x, w, b, r, dy, act, bf16, param_bf16):
    x, w, dy = x.double(), w.double(), dy.double()
    b = torch.zeros(w.shape[0], device=x.device, dtype=torch.float64) if b is None else b.double()
    M, K = x.shape
    N = w.shape[0]
    q, qp = (2.0 ** -8 if bf16 else 0.0), (2.0 ** -8 if param_bf16 else U)
    out_q = q or U
    z = x @ w.T + b
    e_z = (K + 3) * U * (x.abs() @ w.abs().T + b.abs())
    if act == "relu":
        a, slope, e_slope = z.clamp(min=0), (z > 0).double(), torch.zeros_like(z)
    elif act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        a = z * cdf
        slope = cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        e_slope = 0.8 * (e_z + (q + U) * (z.abs() + e_z)) + 8 * U * (1 + z.abs())
    else:
        a, slope, e_slope = z, torch.ones_like(z), torch.zeros_like(z)
    e_a = 1.13 * e_z + 8 * U * z.abs()
    y = a if r is None else a + r.double()
    e_y = e_a + (out_q + U) * (y.abs() + e_a)
    dz = dy * slope
    e_dz = torch.zeros_like(dz) if act is None else dy.abs() * e_slope + (q + U) * (dz.abs() + dy.abs() * e_slope)
    dx, dw, db = dz @ w, dz.T @ x, dz.sum(0)
    e_dx = e_dz @ w.abs() + (N + 3) * U * ((dz.abs() + e_dz) @ w.abs())
    e_dw = e_dz.T @ x.abs() + (M + 130) * U * ((dz.abs() + e_dz).T @ x.abs())
    e_db = e_dz.sum(0) + (M + 130) * U * (dz.abs() + e_dz).sum(0)
    outs = [(y, e_y), (dx, e_dx + out_q * (dx.abs() + e_dx)), (dw, e_dw + qp * (dw.abs() + e_dw)),
            (db, e_db + qp * (db.abs() + e_db))]
    return outs + ([(dy, torch.zeros_like(dy))] if r is not None else [])


def _run(x, w, b, r, dy, act):
    from mitune.ops.linear import linear
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    b = None if b is None else b.detach().requires_grad_()
    r = None if r is None else r.detach().requires_grad_()
    y = linear(x, w, b, activation=act, residual=r)
    leaves = [t for t in (x, w, b, r) if t is not None]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))


def _check(got, want, names=("y", "dx", "dw", "db", "dr")):
    for name, a, (v, e) in zip(names, got, want):
        assert a.shape == v.shape, name
        worst = ((a.double() - v).abs() - e).max().item()
        assert worst <= 1e-37, (name, worst, e.max().item())


def _make(M, K, N, dtype, whole, residual=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M * 7 + K * 3 + N)
    if whole:
        new = lambda *s: torch.randint(-1, 2, s, device="cuda", generator=g).to(dtype)          # noqa: E731
    else:
        new = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)                  # noqa: E731
    w = new(N, K) if whole else (new(N, K).float() / math.sqrt(K)).to(dtype)
    return new(M, K), w, new(N), new(M, N) if residual else None, new(M, N)


SIZES = [(1, 8, 8), (1, 1, 1), (3, 40, 17), (16, 512, 64), (17, 100, 130), (100, 81, 70), (130, 64, 1), (128, 128, 128), (257, 72, 300),
         (300, 200, 129), (1000, 264, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_forward_and_gradients(dtype, act, residual, M, K, N):
    x, w, b, r, dy = _make(M, K, N, dtype, act == "relu", residual)
    bf16 = dtype == torch.bfloat16
    _check(_run(x, w, b, r, dy, act), _formula(x, w, b, r, dy, act, bf16, bf16))


@pytest.mark.gpu
@pytest.mark.parametrize("act,residual", [("gelu", True), ("relu", False), (None, True)])
def test_the_large_tiles(act, residual):
    """Enough 256-tiles for the eight-wave form, with ragged last tiles; f32 at 128-tiles."""
    M, K, N = 4200, 264, 4100
    x, w, b, r, dy = _make(M, K, N, torch.bfloat16, act == "relu", residual)
    _check(_run(x, w, b, r, dy, act), _formula(x, w, b, r, dy, act, True, True))
    M, N = 3000, 3001
    x, w, b, r, dy = _make(M, 100, N, torch.float32, act == "relu", residual)
    _check(_run(x, w, b, r, dy, act), _formula(x, w, b, r, dy, act, False, False))


@pytest.mark.gpu
@pytest.mark.parametrize("act,residual,bias", [("gelu", True, True), ("relu", False, True), (None, False, False)])
@pytest.mark.parametrize("M,K,N", [(2300, 4099, 4100), (4097, 4168, 2056), (33000, 264, 264), (264, 8400, 4104)])
def test_every_product_on_the_256_tile(act, residual, bias, M, K, N):
    """More than 128 tiles of 256 in the forward pass, the input gradient or the weight gradient (all three in the first two), last
    tiles of a few rows or columns, depths that end inside a step of 64, rows of ``x`` further apart than its width."""
    x, w, b, r, dy = _make(M, K, N, torch.bfloat16, act == "relu", residual)
    if K % 8 == 0:
        wide = torch.full((M, K + 24), float("nan"), device="cuda", dtype=torch.bfloat16)
        wide[:, 8:8 + K] = x
        x = wide[:, 8:8 + K]
    b = b if bias else None
    want = _formula(x, w, b, r, dy, act, True, True)
    _check(_run(x, w, b, r, dy, act), want if bias else want[:3] + want[4:], ("y", "dx", "dw") + (("db",) if bias else ()) + ("dr",))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("M,K,N", [(50, 40, 33), (2000, 264, 520)])
def test_gradients_of_some_operands(dtype, act, M, K, N):
    """Whichever operands want one, each gradient is the same bit for bit."""
    from mitune.ops.linear import linear
    x, w, b, r, dy = _make(M, K, N, dtype, False)
    every = _run(x, w, b, r, dy, act)[1:]
    for wanted in range(1, 16):
        leaves = [t.detach().requires_grad_(bool(wanted >> i & 1)) for i, t in enumerate((x, w, b, r))]
        y = linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
        some = [t for t in leaves if t.requires_grad]
        for got, want in zip(torch.autograd.grad(y, some, dy), [g for g, t in zip(every, leaves) if t.requires_grad]):
            assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,M,K,N", [(torch.bfloat16, 4097, 4168, 2056), (torch.float32, 3001, 1000, 520)])
def test_results_repeat(dtype, M, K, N):
    """The same bits every time, and the same for a part of the rows on another tile: products are summed in one order."""
    x, w, b, r, dy = _make(M, K, N, dtype, False)
    first = _run(x, w, b, r, dy, "gelu")
    for _ in range(8):
        for u, v in zip(first, _run(x, w, b, r, dy, "gelu")):
            assert torch.equal(u, v)
    few = 900
    part = _run(x[:few], w, b, r[:few], dy[:few], "gelu")
    assert torch.equal(part[0], first[0][:few]) and torch.equal(part[1], first[1][:few])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act,residual", [("gelu", True), ("relu", True), (None, False)])
@pytest.mark.parametrize("M,K,N", [(40, 2200, 70), (130, 1025, 1100), (5, 1500, 2600)])
def test_long_contractions_over_few_tiles_are_split(dtype, act, residual, M, K, N):
    """Forward over K, input gradient over N: parts added in order, odd widths and last parts of another depth."""
    x, w, b, r, dy = _make(M, K, N, dtype, act == "relu", residual)
    bf16 = dtype == torch.bfloat16
    _check(_run(x, w, b, r, dy, act), _formula(x, w, b, r, dy, act, bf16, bf16))


@pytest.mark.gpu
def test_more_output_features_than_one_weight_gradient_launch_takes():
    M, K, N = 40, 16, 16400
    x, w, b, r, dy = _make(M, K, N, torch.float32, False, False)
    _check(_run(x, w, b, r, dy, "gelu"), _formula(x, w, b, r, dy, "gelu", False, False))
    N = 32700
    x, w, b, r, dy = _make(M, K, N, torch.bfloat16, False, False)
    _check(_run(x, w, b, r, dy, "gelu"), _formula(x, w, b, r, dy, "gelu", True, True))


@pytest.mark.gpu
def test_bias_types_and_no_bias():
    x, w, b, r, dy = _make(70, 48, 33, torch.bfloat16, False)
    got = _run(x, w, b.float(), r, dy, "gelu")
    want = _formula(x, w, b, r, dy, "gelu", True, True)
    exact_db = _formula(x, w, b, r, dy, "gelu", True, False)[3]
    assert got[3].dtype == torch.float32
    _check(got[:3] + [got[3]], want[:3] + [exact_db])
    none = _run(x, w, None, r, dy, "gelu")
    want = _formula(x, w, None, r, dy, "gelu", True, True)
    _check(none, want[:3] + want[4:], ("y", "dx", "dw", "dr"))


@pytest.mark.gpu
def test_bf16_parameters_without_an_epilogue():
    x, w, b, _, dy = _make(200, 72, 40, torch.bfloat16, False)
    got = _run(x, w, b, None, dy, None)
    assert [t.dtype for t in got] == [torch.bfloat16] * 4
    _check(got, _formula(x, w, b, None, dy, None, True, True))


@pytest.mark.gpu
def test_autocast_keeps_f32_masters():
    from mitune.ops.linear import linear
    x, w, b, r, dy = _make(96, 64, 80, torch.float32, False)
    half = [t.bfloat16() for t in (x, w, r, dy)]
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = linear(leaves[0], leaves[1], leaves[2], activation="gelu", residual=leaves[3])
    assert y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y, leaves, half[3])
    assert all(g.dtype == torch.float32 for g in grads)
    want = _formula(half[0], half[1], b, half[2], half[3], "gelu", True, False)
    _check([y.detach()] + list(grads), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_strides_and_an_expanded_gradient(dtype):
    from mitune.ops.linear import linear
    x, w, b, r, dy = _make(60, 32, 24, dtype, False)
    ref = _run(x, w, b, r, dy, "gelu")
    got = _run(x.view(3, 4, 5, 32), w, b, r.view(3, 4, 5, 24), dy.view(3, 4, 5, 24), "gelu")
    for a, e in zip(got, ref):
        assert torch.equal(a.reshape(e.shape), e)
    wide = torch.zeros(60, 75, device="cuda", dtype=dtype)
    for off in (0, 3, 16):
        wide[:, off:off + 32] = x
        tall = torch.zeros(40, 24, device="cuda", dtype=dtype).t()
        tall[:, :32] = w
        spread = torch.zeros(60, 50, device="cuda", dtype=dtype)
        spread[:, off:off + 24] = dy
        for a, e in zip(_run(wide[:, off:off + 32], tall[:, :32], b, r.t().contiguous().t(), spread[:, off:off + 24], "gelu"), ref):
            assert torch.equal(a, e)
    one = torch.ones((), device="cuda", dtype=dtype).expand(60, 24)
    for act in (None, "gelu"):
        for a, e in zip(_run(x, w, b, r, one, act), _run(x, w, b, r, one.contiguous(), act)):
            assert torch.equal(a, e)
    y = linear(x[0], w, b, activation="gelu", residual=r[0])
    assert y.shape == (24,) and torch.equal(y, linear(x[:1], w, b, activation="gelu", residual=r[:1])[0])
    assert linear(x[:0], w, b, activation="gelu").shape == (0, 24)


@pytest.mark.gpu
def test_relu_in_the_epilogue_equals_relu_behind_the_layer():
    """f32: the same sums, so the same bits, forward and backward."""
    from mitune.ops.linear import linear
    for M, K, N in ((300, 64, 128), (40, 20, 12), (70000, 16, 8)):
        x, w, b, _, dy = _make(M, K, N, torch.float32, False, False)
        got = _run(x, w, b, None, dy, "relu")
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = torch.relu(linear(*leaves))
        assert torch.equal(got[0], y.detach())
        assert torch.equal(got[1], torch.autograd.grad(y, leaves, dy)[0])


@pytest.mark.gpu
def test_not_a_number_stays_one():
    from mitune.ops.linear import linear
    x, w, b, _, dy = _make(20, 16, 8, torch.float32, False, False)
    x[3] = float("nan")
    for act in ("relu", "gelu"):
        y = linear(x, w, b, activation=act)
        assert y[3].isnan().all() and torch.isfinite(y[torch.arange(20) != 3]).all()
    got = _run(x, w, b, None, dy, "relu")
    assert got[1][torch.arange(20, device="cuda") != 3].isfinite().all() and got[2].isnan().any()


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the f32 forward pass, step 1e-2, entries of order one: curvature e^2 and rounding over e stay below
    2e-3 of the function's norm."""
    from mitune.ops.linear import linear
    x, w, b, r, dy = _make(30, 20, 12, torch.float32, False)
    grads = _run(x, w, b, r, dy, "gelu")[1:]
    g = torch.Generator(device="cuda").manual_seed(4)
    f = lambda a: (linear(a[0], a[1], a[2], activation="gelu", residual=a[3]).double() * dy.double()).sum().item()          # noqa: E731
    size = (linear(x, w, b, activation="gelu", residual=r).double() * dy.double()).norm().item()
    for i in range(4):
        step = torch.randn((x, w, b, r)[i].shape, device="cuda", generator=g)
        hi, lo = [x, w, b, r], [x, w, b, r]
        hi[i], lo[i] = hi[i] + 1e-2 * step, lo[i] - 1e-2 * step
        slope = (f(hi) - f(lo)) / 2e-2
        assert abs(slope - (grads[i].double() * step.double()).sum().item()) < 2e-3 * size * 20 ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_passes_replay_like_eager_ones(dtype):
    from mitune.ops.linear import linear
    x, w, b, r, dy = _make(300, 64, 40, dtype, False)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    call = lambda: linear(leaves[0], leaves[1], leaves[2], activation="gelu", residual=leaves[3])          # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(call(), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
        grads = torch.autograd.grad(y, leaves, dy)
        y = y.detach()
    for seed in range(3):
        new = _make(300, 64, 40, dtype, False, seed=seed + 1)
        for t, n in zip(leaves + [dy], new):
            t.data.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip([y] + list(grads), _run(*new, "gelu")):
            assert torch.equal(a, e)


@pytest.mark.gpu
def test_gpu_refusals():
    from mitune.ops.linear import linear
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    bad = [(x.half(), w.half(), None, None), (x.bfloat16(), w, None, None), (x, w, torch.zeros(6, device="cuda").bfloat16(), None),
           (x, w, None, torch.zeros(4, 6, device="cuda").bfloat16()), (x, w, torch.zeros(6), None)]
    for a, b, c, d in bad:
        with pytest.raises(TypeError):
            linear(a, b, c, activation="gelu", residual=d)
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(TypeError):
        linear(x, w, activation="relu")


def test_arguments_are_checked():
    from mitune.ops.linear import linear
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    wrong = [dict(activation="tanh"), dict(activation="relu", bias=torch.zeros(5)), dict(residual=torch.zeros(4, 5)),
             dict(residual=torch.zeros(6))]
    for kw in wrong:
        with pytest.raises(ValueError):
            linear(x, w, **kw)
    with pytest.raises(ValueError):
        linear(torch.zeros(4, 7), w, activation="relu")


def test_the_cpu_form():
    from mitune.ops.linear import linear
    g = torch.Generator().manual_seed(0)
    x, w, b, r = (torch.randn(*s, generator=g) for s in ((5, 8), (6, 8), (6,), (5, 6)))
    F = torch.nn.functional
    assert torch.equal(linear(x, w, b, activation="gelu", residual=r), F.gelu(F.linear(x, w, b)) + r)
    assert torch.equal(linear(x, w, b, activation="relu"), F.relu(F.linear(x, w, b)))
    assert torch.equal(linear(x, w, b, residual=r), F.linear(x, w, b) + r)
    assert torch.equal(linear(x, w), F.linear(x, w))
