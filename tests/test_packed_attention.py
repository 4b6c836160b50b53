"""Attention over packed sequences: the kernels against plain attention in 64 bits, element by element.

The tolerances are error bounds.  With ``u`` = 2^-24 (f32) and ``r`` = 2^-8 for bf16 operands, 0 for f32:
* a score is a sum of ``dk`` products: off by at most ``(dk + 2) u sum|q k| scale``; a probability therefore by the relative
  ``e_p``, twice that (its own score and the row's log-sum) plus a few ``u`` for exp2, log2 and their arguments' roundings;
* ``o``: ``r`` (p rounded for the product) + ``e_p`` + ``(n + 4) u`` of ``sum p |v|``, and ``r |o|`` (or ``u |o|``) at the end;
* ``D = do . o`` takes the rounded ``o``: off by ``sum |do| err(o)`` and ``(dv + 2) u sum |do o|``;
* ``ds = p (dp - D)``: ``e_p |ds| + p ((dv + 2) u sum |do v| + err(D))`` and ``r |ds|``;
* the gradients are sums of ``ds`` or ``p`` times an operand: the operand-weighted sums of those errors, ``(n + 4) u`` of the
  absolute sum, and the output's rounding.
"""
import math

import pytest
import torch

U = 2.0 ** -24


def _plain(q, k, v, lengths, causal, scale, do, bf16):
    """(values, bounds) of o, dq, dk, dv in f64, one head of one sequence at a time."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    h, hk, dk, dv = q.shape[1], k.shape[1], q.shape[2], v.shape[2]
    r = 2.0 ** -8 if bf16 else 0.0
    out_r = 2.0 ** -8 if bf16 else U
    val = [torch.zeros_like(t) for t in (do, q, k, v)]
    err = [torch.zeros_like(t) for t in (do, q, k, v)]
    at = 0
    for n in lengths:
        for i in range(h):
            j = i // (h // hk)
            rows = slice(at, at + n)
            Q, K, V, dO = q[rows, i], k[rows, j], v[rows, j], do[rows, i]
            if n == 0:
                continue
            s = Q @ K.T * scale
            sabs = (Q.abs() @ K.abs().T) * scale
            if causal:
                hide = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
                s = s.masked_fill(hide, float("-inf"))
                sabs = sabs.masked_fill(hide, 0.0)
            p = torch.softmax(s, -1)
            e_p = 2 * (dk + 4) * U * sabs.amax(-1, keepdim=True) + 16 * U
            o = p @ V
            pv = p @ V.abs()
            e_o = (r + e_p + (n + 4) * U) * pv + out_r * (o.abs() + (r + e_p) * pv)
            dp, dpabs = dO @ V.T, dO.abs() @ V.abs().T
            D = (dO * o).sum(-1, keepdim=True)
            e_D = (dO.abs() * e_o).sum(-1, keepdim=True) + (dv + 2) * U * (dO * o).abs().sum(-1, keepdim=True)
            ds = p * (dp - D)
            e_ds = e_p * ds.abs() + p * ((dv + 2) * U * dpabs + e_D + 2 * U * (dp.abs() + D.abs()))
            e_ds = e_ds + (r + 2 * U) * (ds.abs() + e_ds)
            sums = (n * (h // hk) + 4) * U
            val[0][rows, i], err[0][rows, i] = o, e_o
            val[1][rows, i] = ds @ K * scale
            err[1][rows, i] = scale * (e_ds @ K.abs() + sums * (ds.abs() @ K.abs()))
            val[2][rows, j] += ds.T @ Q * scale
            err[2][rows, j] += scale * (e_ds.T @ Q.abs() + sums * (ds.abs().T @ Q.abs()))
            val[3][rows, j] += p.T @ dO
            err[3][rows, j] += ((r + e_p + sums) * p).T @ dO.abs()
        at += n
    for x in (1, 2, 3):       # the outputs' own rounding, of the value as computed
        err[x] += out_r * (val[x].abs() + err[x])
    return val, err


def _check(got, val, err, slack=1e-30):
    for name, g, w, e in zip(("o", "dq", "dk", "dv"), got, val, err):
        assert g.shape == w.shape, (name, g.shape, w.shape)
        worst = ((g.double() - w).abs() - e).max().item() if w.numel() else 0.0
        assert torch.isfinite(g).all(), name
        assert worst <= slack, (name, worst, e.max().item())


def _inputs(lengths, rows, heads, kv_heads, dk, dv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows)
    make = lambda h, d: torch.randn(rows, h, d, device="cuda", generator=g).to(dtype)          # noqa: E731
    return make(heads, dk), make(kv_heads, dk), make(kv_heads, dv), make(heads, dv)


def _grads(q, k, v, pack, do, causal, scale=None):
    from mitune.ops.attention import packed_attention
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = packed_attention(q, k, v, pack, causal=causal, scale=scale)
    return (o.detach(),) + torch.autograd.grad(o, (q, k, v), do)


LENGTHS = [[1], [0, 5, 0], [128], [129, 127, 1, 64, 33], [300, 17, 2, 500], [31, 32, 63, 65, 96, 257]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("heads,kv_heads,dk,dv", [(2, 2, 64, 64), (4, 2, 32, 32), (3, 1, 128, 128), (2, 1, 20, 36), (2, 2, 96, 80),
                                                  (1, 1, 1, 3)])
def test_forward_and_gradients(dtype, causal, lengths, heads, kv_heads, dk, dv):
    from mitune.ops.attention import SequencePack
    rows = sum(lengths) + 7 * (len(lengths) % 2)
    q, k, v, do = _inputs(lengths, rows, heads, kv_heads, dk, dv, dtype)
    got = _grads(q, k, v, SequencePack(lengths, rows=rows), do, causal)
    val, err = _plain(q, k, v, lengths, causal, dk ** -0.5, do, dtype == torch.bfloat16)
    _check(got, val, err)
    for t in got:
        assert not t[sum(lengths):].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dk,dv", [(2, 2, 64, 64), (4, 2, 32, 32), (3, 1, 128, 128), (2, 1, 20, 36), (2, 2, 32, 64)])
def test_every_form(monkeypatch, dtype, form, causal, heads, kv_heads, dk, dv):
    """Waves that share a tile, that share a walk, and that walk alone over short sequences, whatever the launch's size would pick."""
    from mitune.ops import attention_hip
    from mitune.ops.attention import SequencePack
    monkeypatch.setattr(attention_hip, "FORM", form)
    lengths = [129, 5, 0, 300, 64, 33]
    rows = sum(lengths) + 150
    q, k, v, do = _inputs(lengths, rows, heads, kv_heads, dk, dv, dtype)
    got = _grads(q, k, v, SequencePack(lengths, rows=rows), do, causal)
    _check(got, *_plain(q, k, v, lengths, causal, dk ** -0.5, do, dtype == torch.bfloat16))
    for t in got:
        assert not t[sum(lengths):].any()
    for n in (90, 300):                                # uniform batches have no list
        q, k, v, do = _inputs([n] * 3, 3 * n, heads, kv_heads, dk, dv, dtype)
        want = _grads(q, k, v, SequencePack([n] * 3), do, causal)
        for a, b in zip(_grads(q, k, v, SequencePack.uniform(3, n), do, causal), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 1)])
def test_walks_cut_in_two(monkeypatch, causal, heads, kv_heads):
    """However many of the longest walks over the queries two workgroups share: none, some, all that have any."""
    from mitune.ops import attention_hip
    from mitune.ops.attention import SequencePack
    monkeypatch.setattr(attention_hip, "FORM", 0)
    lengths = [300, 130, 64]                          # 3 + 2 + 1 items of key rows
    q, k, v, do = _inputs(lengths, 500, heads, kv_heads, 64, 48, torch.bfloat16)
    want = _plain(q, k, v, lengths, causal, 0.125, do, True)
    order = 0 if causal else 1
    pack = SequencePack(lengths, rows=500)
    assert pack._cut(order, 256) == 0 and pack._cut(order, 1) == (5 if causal else 6)      # the two last keys of 130 walk over 2 rows of 712
    for cut in (0, 1, 4, 6):
        pack._cuts[order, kv_heads] = cut
        got = _grads(q, k, v, pack, do, causal)
        _check(got, *want)
        assert not any(t[sum(lengths):].any() for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_longer_sequence_with_a_scale_and_many_tiles(dtype):
    from mitune.ops.attention import SequencePack
    lengths = [1100, 2, 700]
    q, k, v, do = _inputs(lengths, sum(lengths), 4, 1, 64, 64, dtype)
    got = _grads(q, k, v, SequencePack(lengths), do, True, scale=0.3)
    _check(got, *_plain(q, k, v, lengths, True, 0.3, do, dtype == torch.bfloat16))


@pytest.mark.gpu
def test_scores_far_above_the_first_tiles_maximum():
    """The running maximum has to move again and again, by far more than the margin it is allowed to lag."""
    from mitune.ops.attention import SequencePack
    n = 600
    q, k, v, do = _inputs([n], n, 1, 1, 32, 32, torch.float32, seed=3)
    k = k * torch.linspace(0.1, 12.0, n, device="cuda")[:, None, None]
    got = _grads(q, k, v, SequencePack([n]), do, False)
    _check(got, *_plain(q, k, v, [n], False, 32 ** -0.5, do, False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_operands(dtype):
    """Slices of one fused projection are read in place; rows off the 16-byte grid, expanded and transposed operands give the
    same numbers as contiguous copies."""
    from mitune.ops.attention import SequencePack
    lengths, h, d = [150, 40], 4, 32
    rows = sum(lengths)
    pack = SequencePack(lengths)
    g = torch.Generator(device="cuda").manual_seed(5)
    do = torch.randn(rows, h, d, device="cuda", generator=g).to(dtype)
    for width in (3 * h * d, 3 * h * d + 1):
        qkv = torch.randn(rows, width, device="cuda", generator=g).to(dtype)
        q, k, v = (qkv[:, i * h * d:(i + 1) * h * d].unflatten(1, (h, d)) for i in range(3))
        a = _grads(q, k, v, pack, do, True)
        b = _grads(q.contiguous(), k.contiguous(), v.contiguous(), pack, do.transpose(0, 1).contiguous().transpose(0, 1), True)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    one = torch.randn(rows, 1, d, device="cuda", generator=g).to(dtype)
    a = _grads(q, one.expand(rows, h, d), v, pack, do, False)
    b = _grads(q, one.expand(rows, h, d).contiguous(), v, pack, do, False)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    flip = torch.randn(h, d, rows, device="cuda", generator=g).to(dtype).permute(2, 0, 1)      # rows innermost
    for x, y in zip(_grads(flip, k, v, pack, do, True), _grads(flip.contiguous(), k, v, pack, do, True)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_expanded_leaf_sums_its_gradient():
    from mitune.ops.attention import SequencePack, packed_attention
    g = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn(70, 4, 32, device="cuda", generator=g)
    one = torch.randn(70, 1, 32, device="cuda", generator=g, requires_grad=True)
    do = torch.randn(70, 4, 32, device="cuda", generator=g)
    pack = SequencePack([70])
    (a,) = torch.autograd.grad(packed_attention(q, one.expand(70, 4, 32), one.expand(70, 4, 32), pack), one, do)
    (b,) = torch.autograd.grad(packed_attention(q, one, one, pack), one, do)           # the same sharing, inside the kernel
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_outside_a_sequence_never_reach_it(dtype, causal):
    """NaN and infinities behind the last sequence and in a neighbouring one leave the others bit for bit as they were."""
    from mitune.ops.attention import SequencePack
    lengths, rows = [70, 45, 200], 340
    pack = SequencePack(lengths, rows=rows)
    q, k, v, do = _inputs(lengths, rows, 2, 1, 32, 32, dtype)
    want = _grads(q, k, v, pack, do, causal)
    for t, bad in zip((q, k, v, do), (float("nan"), float("inf"), float("-inf"), float("nan"))):
        t[70:115] = bad
        t[315:] = bad
    got = _grads(q, k, v, pack, do, causal)
    for a, b in zip(got, want):
        assert torch.equal(a[:70], b[:70]) and torch.equal(a[115:], b[115:])
        assert not b[315:].any()


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the f32 forward pass along random directions.  Step ``e`` with entries of order one: the
    difference's own error is e^2 (third derivative) + u |f| sqrt(terms) / e, here 1e-4 + 6e-8 * 40 / 1e-2: 1e-3 of |f| covers
    both."""
    from mitune.ops.attention import SequencePack, packed_attention
    lengths = [5, 130, 33]
    q, k, v, do = _inputs(lengths, sum(lengths), 4, 2, 32, 16, torch.float32)
    pack = SequencePack(lengths)
    grads = _grads(q, k, v, pack, do, True)[1:]
    g = torch.Generator(device="cuda").manual_seed(1)
    f = lambda *a: (packed_attention(*a, pack, causal=True).double() * do.double()).sum().item()          # noqa: E731
    size = (packed_attention(q, k, v, pack, causal=True).double() * do.double()).norm().item()
    for x in range(3):
        u = torch.randn((q, k, v)[x].shape, device="cuda", generator=g)
        e = 1e-2
        hi, lo = [q, k, v], [q, k, v]
        hi[x], lo[x] = hi[x] + e * u, lo[x] - e * u
        slope = (f(*hi) - f(*lo)) / (2 * e)
        want = (grads[x].double() * u.double()).sum().item()
        assert abs(slope - want) < 1e-3 * size * math.sqrt(32), (x, slope, want)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_uniform_packs_match_listed_ones_and_repeat_bit_for_bit(causal):
    from mitune.ops.attention import SequencePack
    q, k, v, do = _inputs([200] * 3, 600, 2, 2, 64, 64, torch.bfloat16)
    a = _grads(q, k, v, SequencePack.uniform(3, 200), do, causal)
    for _ in range(2):
        for x, y in zip(a, _grads(q, k, v, SequencePack([200, 200, 200]), do, causal)):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_captured_passes_replay_like_eager_ones():
    from mitune.ops.attention import SequencePack, packed_attention
    pack = SequencePack([100, 29], rows=140)
    q, k, v, do = _inputs([100, 29], 140, 2, 1, 64, 64, torch.bfloat16)
    q.requires_grad_(), k.requires_grad_(), v.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(packed_attention(q, k, v, pack, causal=True), (q, k, v), do)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = packed_attention(q, k, v, pack, causal=True)
        grads = torch.autograd.grad(o, (q, k, v), do)
        o = o.detach()
    for seed in range(3):
        for t, new in zip((q, k, v, do), _inputs([100, 29], 140, 2, 1, 64, 64, torch.bfloat16, seed=seed + 10)):
            t.data.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((o,) + grads, _grads(q, k, v, pack, do, True)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_another_stream_and_two_calls_at_once():
    from mitune.ops.attention import SequencePack
    pack = SequencePack([333, 12])
    sets = [_inputs([333, 12], 345, 2, 2, 32, 32, torch.float32, seed=s) for s in range(2)]
    want = [_grads(q, k, v, pack, do, True) for q, k, v, do in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for st, (q, k, v, do) in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(_grads(q, k, v, pack, do, True))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_empty_batches_and_gpu_refusals():
    from mitune.ops.attention import SequencePack, packed_attention
    e = torch.zeros(0, 2, 64, device="cuda", requires_grad=True)
    o = packed_attention(e, e, e, SequencePack([]))
    assert o.shape == (0, 2, 64)
    (g,) = torch.autograd.grad(o, e, torch.zeros_like(o))
    assert g.shape == e.shape
    none = torch.full((9, 2, 64), float("nan"), device="cuda")
    assert not packed_attention(none, none, none, SequencePack([0], rows=9)).any()
    q = torch.zeros(4, 1, 144, device="cuda")
    with pytest.raises(ValueError):
        packed_attention(q, q, q, SequencePack([4]))
    h = torch.zeros(4, 1, 64, device="cuda", dtype=torch.float16)
    with pytest.raises(TypeError):
        packed_attention(h, h, h, SequencePack([4]))
    f = torch.zeros(4, 1, 64, device="cuda")
    with pytest.raises(ValueError):
        packed_attention(f, f, f, SequencePack([4], device="cpu"))
    with pytest.raises(TypeError):
        SequencePack(torch.tensor([4], device="cuda"))


def test_packs_check_their_lengths():
    from mitune.ops.attention import SequencePack
    p = SequencePack([3, 0, 130, 5], rows=200, device="cpu")
    assert (p.total, p.rows, p.longest) == (138, 200, 130)
    assert SequencePack(torch.tensor([2, 2]), device="cpu").total == 4
    assert SequencePack.uniform(3, 7, device="cpu").rows == 21
    for bad in ([-1, 4], [2 ** 62, 2 ** 62, 2 ** 62, 2 ** 62]):
        with pytest.raises(ValueError):
            SequencePack(bad, device="cpu")
    with pytest.raises(ValueError):
        SequencePack([5, 5], rows=9, device="cpu")
    with pytest.raises(ValueError):
        SequencePack.uniform(2, -1, device="cpu")
    for bad in ([1.5, 2.0], [[1, 2], [3, 4]]):
        with pytest.raises(TypeError):
            SequencePack(bad, device="cpu")


def test_operands_are_checked():
    from mitune.ops.attention import SequencePack, packed_attention
    pack = SequencePack([3, 2], device="cpu")
    t = torch.zeros(5, 4, 8)
    assert packed_attention(t, t, t, pack).shape == (5, 4, 8)
    wrong = [(t[0], t, t), (t[:4], t, t), (t, t[:, :3], t[:, :3]), (t, t[..., :4], t), (t, t[:, :2], t), (t[..., :0], t[..., :0], t)]
    for q, k, v in wrong:
        with pytest.raises(ValueError):
            packed_attention(q, k, v, pack)
    with pytest.raises(TypeError):
        packed_attention(t, t.double(), t, pack)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            packed_attention(t, t, t, pack, scale=scale)


def test_the_cpu_form_is_attention_per_sequence():
    from mitune.ops.attention import SequencePack, attention_reference, packed_attention
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(12, h, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    o = packed_attention(q, k, v, SequencePack([5, 6], rows=12, device="cpu"))
    for a, b in ((0, 5), (5, 11)):
        for h in range(4):
            want = attention_reference(q[a:b, h], k[a:b, h // 2], v[a:b, h // 2])
            assert torch.allclose(o[a:b, h], want)
    c = packed_attention(q, k, v, SequencePack([5, 6], rows=12, device="cpu"), causal=True)
    assert torch.allclose(c[0], v[0].repeat_interleave(2, 0)) and torch.allclose(c[10], o[10]) and not c[11:].any()


def test_tile_lists_cover_every_row_once():
    """Every row in exactly one tile of each order, work not increasing, rows of no sequence as negative entries."""
    import numpy as np
    from mitune.ops import attention as A
    kept = []
    real = torch.from_numpy
    try:
        torch.from_numpy = lambda a: kept.append(a.copy()) or real(a)
        pack = A.SequencePack.__new__(A.SequencePack)
        pack._fix(530, 700, "cpu")
        pack.device = type("D", (), {"type": "cuda"})()
        pack.lengths = np.array([300, 0, 1, 129, 100])
        try:
            pack._lay_out()
        except Exception:
            pass                                   # the upload has no device to go to
    finally:
        torch.from_numpy = real
    at = 0
    for which, count in enumerate(pack._counts):
        for work in (lambda r, g: min(r[2] + g, r[1]), lambda r, g: r[1] - r[2], lambda r, g: r[1]):
            seen = np.zeros(700, dtype=int)
            last = None
            for r in kept[0][at:at + count].tolist():
                if r[1] < 0:
                    seen[r[0]:r[0] - r[1]] += 1
                    assert r[0] >= 530
                    continue
                grain = 128 if which == 0 or r[3] else 32
                assert r[3] == (which == 2 and r[1] <= A.SOLO_ROWS)
                lo, hi = r[0] + r[2], r[0] + min(r[1], r[2] + grain)
                seen[lo:hi] += 1
                cost = work(r, grain) / (1 if which == 0 or r[3] else 4)
                assert last is None or cost <= last
                last = cost
            assert (seen == 1).all()
            at += count
    assert at == len(kept[0])
