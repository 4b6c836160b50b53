"""Calls of the long-sequence operators at the edge of what they take: refused on the host, or right on the GPU."""
import pytest
import torch


def test_weight_gradients_of_too_many_columns_are_refused_by_the_launchers():
    """A tile's column number is 16 bits: past 32767 tiles of 128 columns it would wrap around to addresses before the gradient."""
    from mitune.ops import lib as L
    so = L.load()
    for wide in (32767 * 128 + 8, 5_000_000):
        assert so.mt_linear_wgrad_launch(16, 16, 16, None, 8, 8, wide, 8, wide, 1, 1, None) == -2
        assert so.mt_wgrad_single_launch(16, 16, 16, None, 8, 8, wide, 1, 8 * wide + 8, None) == -2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layers_of_too_many_features_are_refused_before_they_run(dtype):
    from mitune.ops import linear as M
    from mitune.ops.linear import _fused_linear
    wide = M.MAX_FUSED_WIDTH + 8
    new = lambda *s: torch.empty(*s, device="meta", dtype=dtype)          # noqa: E731
    with pytest.raises(ValueError, match="features"):
        _fused_linear(new(4, 8), new(wide, 8), None, None, None)
    with pytest.raises(ValueError, match="features"):
        _fused_linear(new(4, wide).requires_grad_(), new(8, wide), None, "relu", None)
    if dtype == torch.bfloat16:
        wide = M.MAX_BF16_DW_WIDTH + 8
        with pytest.raises(ValueError, match="features"):
            _fused_linear(new(4, wide), new(8, wide).requires_grad_(), None, "relu", None)


def test_training_layers_of_too_many_rows_are_refused_before_they_run():
    from mitune.ops.linear import MAX_ROWS, _fused_linear
    x, w = torch.empty(MAX_ROWS + 1, 4, device="meta"), torch.empty(8, 4, device="meta")
    with pytest.raises(ValueError, match="rows"):
        _fused_linear(x, w.requires_grad_(), None, "relu", None)


def test_null_addresses_are_refused_by_the_launchers():
    """Tensors of a dispatch mode that hold no memory have address 0; each operand in turn."""
    from mitune.ops import lib as L
    so = L.load()
    gemm = lambda a, b, c, m: so.mt_linear_gemm_launch(0, a, b, None, None, c, None, None, m, 8, 8, 8, 8, 0, 0, 0, None)          # noqa: E731
    calls = [lambda *p: gemm(*p, 4), lambda *p: gemm(*p, 400),
             lambda *p: so.mt_linear_act_bwd_launch(*p, None, None, 8, 8, 8, 8, 1, 0, 0, None),
             lambda *p: so.mt_linear_wgrad_f32_parts_launch(*p, 8, 8, 8, 2, 128, 1, None),
             lambda *p: so.mt_linear_wgrad_launch(*p, None, 8, 8, 8, 8, 8, 0, 0, None)]
    for call in calls:
        for null in range(3):
            assert call(*(None if i == null else 16 for i in range(3))) == -2
    assert so.mt_norm_fwd_launch(None, None, None, 16, None, 8, 8, 8, 1e-5, 0, 0, None) == -2
    assert so.mt_norm_fwd_launch(16, None, None, None, None, 8, 8, 8, 1e-5, 0, 0, None) == -2
    for null in (0, 1, 3, 4):
        args = [16, 16, None, 16, 16]
        args[null] = None
        assert so.mt_norm_bwd_launch(*args, None, None, None, 8, 8, 8, 8, 0, 0, None) == -2
    for part, dw, db in ((16, None, None), (None, 16, None), (None, None, 16)):
        assert so.mt_norm_bwd_launch(16, 16, None, 16, 16, part, dw, db, 8, 8, 8, 8, 0, 0, None) == -2
    # q, k, v, out, dout, o, dq, dk, dv, low, lse, delta, halves and the lists of items: one uniform sequence of 8 rows
    used = {0: (0, 1, 2, 5), 1: (0, 1, 2, 3, 4, 6, 7, 8, 10, 11)}
    for backward, places in used.items():
        for null in places:
            at = [16 if i in places and i != null else 0 for i in range(15)]
            args = L.PACKED_ATTN_FORMAT.pack(*at, *[8] * 8, 8, 1, 1, 8, 1, 1, 1, 8, 8, 0, 1, 1, 0, 1.0)
            assert so.mt_packed_attn_launch(args, backward, 0, None) == -2


@pytest.mark.parametrize("heads,kv_heads,dtype,backward", [(16, 1, torch.float32, 0), (16, 16, torch.float32, 1), (8, 8, torch.bfloat16, 1),
                                                           (8, 4, torch.bfloat16, 1), (16, 8, torch.bfloat16, 0)])
def test_more_pieces_than_a_launch_has_threads_for(heads, kv_heads, dtype, backward):
    """Sequences of 33 rows, a workgroup per sequence and head (in the dk / dv kernel of bf16 one of twice as many threads): 2^32 threads and
    more are refused, before anything runs."""
    from mitune.ops import lib as L
    from mitune.ops.attention import SequencePack
    from mitune.ops.attention_hip import _packed_launch
    so, count, bf16 = L.load(), 1 << 20, dtype == torch.bfloat16
    form = 0 if bf16 else 2
    cut = count if bf16 and heads > kv_heads else 0
    args = L.PACKED_ATTN_FORMAT.pack(*[16] * 13, 0, 0, *[8] * 8, 33 * count, count, count, 33, count, heads, kv_heads, 8, 8, 0, form, form, cut,
                                     1.0)
    assert so.mt_packed_attn_launch(args, backward, int(bf16), None) == -2
    new = lambda h: torch.empty(33 * count, h, 8, device="meta", dtype=dtype)          # noqa: E731
    for keeps in (0, 16) if backward else (0,):          # a forward pass that keeps what the backward pass needs is refused as well
        with pytest.raises(ValueError, match="pieces"):
            _packed_launch(None, SequencePack.uniform(count, 33, device="cpu"), new(heads), new(kv_heads), new(kv_heads), False, 1.0,
                           int(not keeps and backward), lse=keeps)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 64, 64), (1, 520, 264), (2, 520, 264)])
def test_the_gradient_of_a_layer_joined_with_another_of_few_rows(dtype, residual, M, K, N):
    """``cat`` hands back slices of a wider gradient; a single row of one counts as contiguous whatever its row stride is.  Whole
    numbers, so that every product is exact."""
    from mitune.ops.linear import linear
    g = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *s: torch.randint(-2, 3, s, device="cuda", generator=g).to(dtype)          # noqa: E731
    leaves = [t.requires_grad_() for t in (new(M, K), new(N, K), new(N), new(M, N))]
    other, dy = new(M, 40), new(M, 40 + N + 40)
    used = leaves if residual else leaves[:3]
    y = linear(*leaves[:3], residual=leaves[3] if residual else None)
    got = torch.autograd.grad(torch.cat([other, y, other], dim=1), used, dy)
    d = dy[:, 40:40 + N].double()
    want = [d @ leaves[1].detach().double(), d.T @ leaves[0].detach().double(), d.sum(0), d]
    for a, b in zip(got, want):
        assert torch.equal(a, b.to(dtype))


def test_a_small_layers_backward_pass_is_spread_over_the_chip():
    """Captured training steps of small ReLU layers are no slower than the layer and the activation apart only while the pass that forms dz
    is not a few workgroups' long walk, and while one call does the rest."""
    from mitune.ops import lib as L
    from mitune.ops.linear import ACTIVATIONS, _bwd_plan, _early_sums
    so = L.load()
    for M, N in ((1600, 256), (3200, 1024), (1600, 64)):
        rows_at_once = 256 // min(64, N // 8)
        assert so.mt_linear_act_parts(M, N, 1) * 4 * rows_at_once >= M - 4 * rows_at_once
    assert _early_sums(True, ACTIVATIONS["gelu"]) and not _early_sums(True, ACTIVATIONS["relu"]) and not _early_sums(False, 2)
    assert _bwd_plan(1600, 256, 256, 64, 64, 1, False, True, True, True, True, 256)[3] == -1
    assert _bwd_plan(1600, 255, 256, 63, 64, 1, False, True, True, True, True, 256)[3] == -1


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1600, 64, 256), (50, 40, 33), (3200, 256, 1024)])
def test_the_bias_gradient_of_a_relu_layer_in_bf16(M, K, N):
    """Under ReLU a term of db is the upstream gradient or nothing: an f32 sum of M exact terms, rounded once.  ``z`` is whole numbers."""
    from mitune.ops.linear import linear
    g = torch.Generator(device="cuda").manual_seed(11)
    x, w, b = (torch.randint(-1, 2, s, device="cuda", generator=g).bfloat16().requires_grad_() for s in ((M, K), (N, K), (N,)))
    dy = torch.randn(M, N, device="cuda", generator=g).bfloat16()
    db, = torch.autograd.grad(linear(x, w, b, activation="relu"), b, dy)
    z = (x.double() @ w.double().T + b.double()).detach()
    terms = dy.double() * (z > 0)
    bound = (M + 130) * 2.0 ** -24 * terms.abs().sum(0) * (1 + 2.0 ** -8) + 2.0 ** -8 * terms.sum(0).abs()
    assert ((db.double() - terms.sum(0)).abs() <= bound).all()


def test_column_sums_of_few_rows_take_few_partial_rows():
    """The backward pass of a norm writes and reads an f32 partial row of dw and of db per workgroup: no more than a quarter of the rows,
    so that they stay below the bytes of x and dy."""
    from mitune.ops import lib as L
    so = L.load()
    for bf16 in (0, 1):
        for M, d in ((2048, 1024 // (2 - bf16)), (4095, 512), (200, 256), (64, 300), (1, 256)):
            assert so.mt_norm_bwd_parts(M, d, bf16) <= (M + 3) // 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", [(None, None), ("w", None), (None, "b")])
def test_a_residual_norm_without_parameters(dtype, which):
    """As plain torch takes it, and as these widths took it before they had kernels."""
    import torch.nn.functional as F

    from mitune.ops.layernorm import residual_layer_norm
    g = torch.Generator(device="cuda").manual_seed(13)
    x, r = (torch.randn(30, 81, device="cuda", generator=g).to(dtype) for _ in range(2))
    w, b = (None if n is None else torch.randn(81, device="cuda", generator=g).to(dtype) for n in which)
    y = residual_layer_norm(x, r, w, b)
    wide = [None if t is None else t.double() for t in (w, b)]
    want = F.layer_norm((x + r).double(), (81,), *wide)
    half = torch.finfo(dtype).eps / 2
    # f32 statistics of 81 terms, 100 u; the product with w and the sum with b, of order 10; one rounding of the output
    assert ((y.double() - want).abs() <= 200 * 2.0 ** -24 * (1 + want.abs()) * 4 + half * want.abs() * (1 + half)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[3, 40], [1, 300, 2], [129] + [500] * 60, [1, 256] * 70])
def test_rows_whose_scores_are_all_minus_infinity(dtype, lengths):
    """A softmax of nothing but -inf is 0 / 0: such rows are not numbers, as in the formula, and no other row is touched.  Long walks, walks
    that four waves share, and short sequences."""
    from mitune.ops.attention import SequencePack, packed_attention
    g = torch.Generator(device="cuda").manual_seed(14)
    rows = sum(lengths)
    q, k, v, do = (torch.rand(rows, 4, 16, device="cuda", generator=g).to(dtype) for _ in range(4))
    bad, at = torch.zeros(rows, dtype=torch.bool, device="cuda"), 0
    for n in lengths:          # causal: row 0 of a sequence sees itself alone; a second bad key leaves row 1 nothing either
        k[at:at + min(n, 2), 1] = float("-inf")
        bad[at:at + min(n, 2)] = True
        at += n
    v.requires_grad_()
    out = packed_attention(q, k, v, SequencePack(lengths), causal=True)
    want = torch.zeros(rows, 4, 16, dtype=torch.bool, device="cuda")
    want[bad, 1] = True
    assert torch.equal(out.isnan(), want)
    dv, = torch.autograd.grad(out, v, do)
    assert torch.equal(dv.isnan(), want)          # p of such a row is not a number for the keys it sees: itself, and the row before it


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [2, 16])
@pytest.mark.parametrize("lengths", [[1, 2, 3] * 30, [2, 4] * 40, [8, 16, 3] * 20])
def test_gradients_of_sequences_of_few_rows(lengths, heads, causal):
    """In bf16, as a share of a gradient's norm.  Rounding a number to bf16 is off by 0.425 * 2^-8 = 0.00166 of it in the mean of
    squares: the output's rounding.  With the roundings of p in the forward pass, which reach D and the log-sum, the same formulas in 64 bits
    give 0.0019 for two rows and less for more; with ds rounded once for its product, 0.0025."""
    from mitune.ops.attention import SequencePack, packed_attention, packed_attention_reference
    g = torch.Generator(device="cuda").manual_seed(15)
    pack, rows = SequencePack(lengths), sum(lengths)
    leaves = [torch.randn(rows, heads, 64, device="cuda", generator=g).bfloat16().requires_grad_() for _ in range(3)]
    do = torch.randn(rows, heads, 64, device="cuda", generator=g).bfloat16()
    got = torch.autograd.grad(packed_attention(*leaves, pack, causal=causal), leaves, do)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(packed_attention_reference(*wide, pack, causal), wide, do.double())
    for a, b in zip(got, want):
        assert ((a.double() - b).norm() / b.norm()).item() <= 0.0021


@pytest.mark.gpu
def test_the_query_gradient_of_a_causal_sequence_with_narrow_heads():
    """Its first rows, which see few keys, have the largest gradients.  The output's rounding and that of ds, 0.00166 of the norm each, are
    0.00235 together where both apply in full; with the errors of D and ds of the first rows it was 0.0025."""
    from mitune.ops.attention import SequencePack, packed_attention, packed_attention_reference
    g = torch.Generator(device="cuda").manual_seed(16)
    rows = 1797
    leaves = [torch.randn(rows, h, 16, device="cuda", generator=g).bfloat16().requires_grad_() for h in (64, 8, 8)]
    do = torch.randn(rows, 64, 16, device="cuda", generator=g).bfloat16()
    dq, = torch.autograd.grad(packed_attention(*leaves, SequencePack([rows]), causal=True), leaves[:1], do)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want, = torch.autograd.grad(packed_attention_reference(*wide, SequencePack([rows]), True), wide[:1], do.double())
    assert ((dq.double() - want).norm() / want.norm()).item() <= 0.00235
