"""Autograd bindings of the attention kernels: short sequences (``csrc/attention.hip``) and packed sequences of any length
(``csrc/packed_attention.hip``)."""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F

from . import lib as L
from .attention import SOLO_ROWS

_KIND = {"softmax": 0, "relu": 1}


def available() -> bool:
    if not torch.cuda.is_available():
        return False
    L.load()          # raises if the library is missing on a GPU machine: no silent fallback
    return True


class FusedShortAttention(torch.autograd.Function):
    """q, k: [B, h, S, dk]; v: [B, h, S, dv]; keep: optional 0/1 mask [B, h, S, S]."""

    @staticmethod
    def forward(ctx, q, k, v, kind: str, keep: Optional[torch.Tensor], dropout_p: float):
        so = L.load()
        B, h, S, dk = q.shape
        dv = v.shape[-1]
        qb, kb, vb = (t.to(torch.bfloat16).contiguous() for t in (q, k, v))
        keep_u8 = keep.to(torch.uint8).contiguous() if keep is not None else None
        out = torch.empty(B, h, S, dv, device=q.device, dtype=torch.bfloat16)
        stat = torch.empty(B * h, S, device=q.device, dtype=torch.float32)
        scale = 1.0 / math.sqrt(dk)
        keep_scale = 1.0 / (1.0 - dropout_p) if keep is not None else 1.0
        L.check(so.mt_attn_fwd_launch(qb.data_ptr(), kb.data_ptr(), vb.data_ptr(),
                                      keep_u8.data_ptr() if keep_u8 is not None else None, out.data_ptr(),
                                      stat.data_ptr(), B * h, S, dk, dv, scale, keep_scale, _KIND[kind],
                                      L.raw_stream(q.device)), "mt_attn_fwd_launch")
        ctx.save_for_backward(qb, kb, vb, stat, keep_u8 if keep_u8 is not None else torch.empty(0, device=q.device))
        ctx.meta = (kind, scale, keep_scale, keep is not None, q.dtype, k.dtype, v.dtype)
        return out.to(q.dtype)

    @staticmethod
    def backward(ctx, grad_out):
        so = L.load()
        qb, kb, vb, stat, keep_u8 = ctx.saved_tensors
        kind, scale, keep_scale, has_keep, qd, kd, vd = ctx.meta
        B, h, S, dk = qb.shape
        dv = vb.shape[-1]
        do = grad_out.to(torch.bfloat16).contiguous()
        dq = torch.empty(B, h, S, dk, device=qb.device, dtype=torch.float32)
        dk_ = torch.empty_like(dq)
        dv_ = torch.empty(B, h, S, dv, device=qb.device, dtype=torch.float32)
        L.check(so.mt_attn_bwd_launch(qb.data_ptr(), kb.data_ptr(), vb.data_ptr(), do.data_ptr(),
                                      keep_u8.data_ptr() if has_keep else None, stat.data_ptr(), dq.data_ptr(),
                                      dk_.data_ptr(), dv_.data_ptr(), B * h, S, dk, dv, scale, keep_scale,
                                      _KIND[kind], L.raw_stream(qb.device)),
                "mt_attn_bwd_launch")
        return dq.to(qd), dk_.to(kd), dv_.to(vd), None, None, None


class FusedQKVAttention(torch.autograd.Function):
    """Attention on ONE fused projection output ``qkv`` [B, S, 2*h*dk + h*dv] (all queries, all keys, all values, each
    head-major) -> [B, S, h*dv].  The kernels read the three column blocks in place and the backward writes one
    gradient tensor of the same layout, so the projection is a single GEMM in each direction."""

    @staticmethod
    def forward(ctx, qkv, h: int, dk: int, kind: str, dropout_p: float, seed: Optional[torch.Tensor] = None):
        so = L.load()
        qkv = qkv.contiguous()
        B, S, W = qkv.shape
        dv = (W - 2 * h * dk) // h
        f32 = 1 if qkv.dtype == torch.float32 else 0
        es = qkv.element_size()
        out = torch.empty(B, S, h * dv, device=qkv.device, dtype=qkv.dtype)
        stat = torch.empty(B * h, S, device=qkv.device, dtype=torch.float32)
        scale = 1.0 / math.sqrt(dk)
        drops = seed is not None and dropout_p > 0.0
        keep_scale = 1.0 / (1.0 - dropout_p) if drops else 1.0
        seed = seed if drops else None
        base = qkv.data_ptr()
        L.check(so.mt_attn_fwd_strided_launch(base, base + h * dk * es, base + 2 * h * dk * es, None, out.data_ptr(),
                                              stat.data_ptr(), B * h, S, dk, dv, scale, keep_scale, _KIND[kind], h,
                                              W, W, h * dv, f32, seed.data_ptr() if seed is not None else None,
                                              float(dropout_p), L.raw_stream(qkv.device)),
                "mt_attn_fwd_strided_launch")
        ctx.save_for_backward(qkv, stat)
        ctx.meta = (h, dk, dv, kind, scale, keep_scale, f32)
        ctx.seed, ctx.p = seed, float(dropout_p)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        so = L.load()
        qkv, stat = ctx.saved_tensors
        h, dk, dv, kind, scale, keep_scale, f32 = ctx.meta
        B, S, W = qkv.shape
        es = qkv.element_size()
        do = grad_out.to(qkv.dtype).contiguous()
        # bf16 operands: the kernel rounds the gradient to bf16 itself (mode 2) -- no f32 tensor, no cast pass
        dqkv = torch.empty(B, S, W, device=qkv.device, dtype=qkv.dtype)
        base, g = qkv.data_ptr(), dqkv.data_ptr()
        L.check(so.mt_attn_bwd_strided_launch(base, base + h * dk * es, base + 2 * h * dk * es, do.data_ptr(), None,
                                              stat.data_ptr(), g, g + h * dk * es, g + 2 * h * dk * es, B * h, S, dk, dv,
                                              scale, keep_scale, _KIND[kind], h, W, W, h * dv, 1 if f32 else 2,
                                              ctx.seed.data_ptr() if ctx.seed is not None else None, ctx.p,
                                              L.raw_stream(qkv.device)), "mt_attn_bwd_strided_launch")
        return dqkv, None, None, None, None, None


class FusedSelfAttention(torch.autograd.Function):
    """Attention straight on projection outputs: ``qk`` [B, S, 2*h*dk] (queries then keys, head-major), ``v`` [B, S, h*dv]
    -> [B, S, h*dv].  f32 or bf16; no head split / merge copies, no dtype casts: the kernels read the strided operands
    in place and write the gradient of ``qk`` as one tensor."""

    @staticmethod
    def forward(ctx, qk, v, h: int, kind: str, keep: Optional[torch.Tensor], dropout_p: float,
                seed: Optional[torch.Tensor] = None):
        so = L.load()
        if v.dtype != qk.dtype:
            v = v.to(qk.dtype)
        qk, v = qk.contiguous(), v.contiguous()      # a column slice of a fused projection is copied here
        B, S, w2 = qk.shape
        dk, dv = w2 // (2 * h), v.shape[-1] // h
        f32 = 1 if qk.dtype == torch.float32 else 0
        es = qk.element_size()
        keep_u8 = keep.to(torch.uint8).contiguous() if keep is not None else None
        out = torch.empty(B, S, h * dv, device=qk.device, dtype=qk.dtype)
        stat = torch.empty(B * h, S, device=qk.device, dtype=torch.float32)
        scale = 1.0 / math.sqrt(dk)
        drops = keep is not None or (seed is not None and dropout_p > 0.0)
        keep_scale = 1.0 / (1.0 - dropout_p) if drops else 1.0
        seed = seed if (keep is None and drops) else None       # attention dropout drawn inside the kernel
        L.check(so.mt_attn_fwd_strided_launch(qk.data_ptr(), qk.data_ptr() + h * dk * es, v.data_ptr(),
                                              keep_u8.data_ptr() if keep_u8 is not None else None, out.data_ptr(),
                                              stat.data_ptr(), B * h, S, dk, dv, scale, keep_scale, _KIND[kind], h,
                                              2 * h * dk, h * dv, h * dv, f32,
                                              seed.data_ptr() if seed is not None else None, float(dropout_p),
                                              L.raw_stream(qk.device)), "mt_attn_fwd_strided_launch")
        ctx.save_for_backward(qk, v, stat, keep_u8 if keep_u8 is not None else torch.empty(0, device=qk.device))
        ctx.meta = (h, kind, scale, keep_scale, keep is not None, f32)
        ctx.seed, ctx.p = seed, float(dropout_p)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        so = L.load()
        qk, v, stat, keep_u8 = ctx.saved_tensors
        h, kind, scale, keep_scale, has_keep, f32 = ctx.meta
        B, S, w2 = qk.shape
        dk, dv = w2 // (2 * h), v.shape[-1] // h
        es = qk.element_size()
        do = grad_out.to(qk.dtype).contiguous()
        dqk = torch.empty(B, S, w2, device=qk.device, dtype=qk.dtype)
        dv_ = torch.empty(B, S, h * dv, device=qk.device, dtype=qk.dtype)
        L.check(so.mt_attn_bwd_strided_launch(qk.data_ptr(), qk.data_ptr() + h * dk * es, v.data_ptr(), do.data_ptr(),
                                              keep_u8.data_ptr() if has_keep else None, stat.data_ptr(), dqk.data_ptr(),
                                              dqk.data_ptr() + h * dk * es, dv_.data_ptr(), B * h, S, dk, dv, scale,
                                              keep_scale, _KIND[kind], h, 2 * h * dk, h * dv, h * dv, 1 if f32 else 2,
                                              ctx.seed.data_ptr() if ctx.seed is not None else None, ctx.p,
                                              L.raw_stream(qk.device)), "mt_attn_bwd_strided_launch")
        return dqk, dv_, None, None, None, None, None


def in_place(t: torch.Tensor) -> torch.Tensor:
    """``t`` [rows, heads, width] as the packed kernels can read it: 16-byte rows and heads, or else a copy padded with zero
    columns to that (zeros add nothing to a score; zero value columns give output columns that are cut off again)."""
    es = t.element_size()
    per = 16 // es
    if (t.stride(2) == 1 and t.shape[2] % per == 0 and t.stride(0) % per == 0 and t.stride(1) % per == 0
            and max(t.stride(0), t.stride(1)) * es <= 1 << 24 and t.data_ptr() % 16 == 0):
        return t
    pad = -t.shape[2] % per
    return F.pad(t, (0, pad)).contiguous() if pad else t.clone(memory_format=torch.contiguous_format)


FORM = None       # tests: the form of every launch


def packed_form(pack, lanes: int, bf16: bool) -> int:
    """How a launch over ``lanes`` heads divides its work: 0, workgroups own 128 rows and share the tiles they walk over (bf16); 1,
    they own 32 rows and their waves share the walk; 2, the same except that each wave of a short sequence's workgroup owns 32 rows.
    Measured, bf16, 0 / 1: one causal sequence of 2048, 8 heads of 128 (128 workgroups) forward 54 / 28 us; 8192, 2 heads (128)
    194 / 84, with its backward pass 1085 / 337; 4 x 2048, 16 heads (1024) 120 / 134.  Packs of sequences that 32 rows hold take the
    third form, 0 / 2 with their backward pass: 4000 of up to 8 rows, 16 heads of 64 1350 / 731 us, 64 of up to 4, 64 / 8 heads 61 / 51, 100 of
    up to 32, 16 heads of 128 98 / 97; 2000 of up to 128, 8 heads of 64 919 / 944."""
    if FORM is not None:
        return FORM if bf16 else max(1, FORM)
    if bf16 and pack._counts[0] * lanes >= 512 and pack.longest > L.PACKED_SPLIT_ROWS:
        return 0
    return 2 if pack._counts[0] * lanes >= 256 else 1


def _packed_launch(so, pack, q, k, v, causal: bool, scale: float, backward: int, out=0, dout=None, o=0, dq=0, dk=0, dv=0, low=0,
                   lse=0, delta=0) -> None:
    bf16 = q.dtype == torch.bfloat16
    form, kv_form = packed_form(pack, q.shape[1], bf16), packed_form(pack, k.shape[1], bf16)
    # A launch has fewer than 2^32 threads: 256 per piece and head; in the shared form's dk / dv 512, and shared heads' walks may be cut
    # in two.  A forward pass that keeps what the backward pass needs is refused where that would be.
    pieces = pack._counts[form] * q.shape[1]
    if backward or lse:
        pieces = max(pieces, pack._counts[kv_form] * k.shape[1] * (1 if kv_form else 2 if q.shape[1] == k.shape[1] else 4))
    if pieces >= 1 << 24:
        raise ValueError(f"{len(pack.lengths)} sequences of {pack.total} rows with {q.shape[1]} heads are more pieces than a launch takes")
    stream = L.raw_stream(q.device)
    items, n = pack._items(form, 0 if causal else 2, stream)
    kv_items, n_kv = pack._items(kv_form, 1 if causal else 2, stream)
    # a uniform batch has no list in which short sequences are marked: its sequences are short, or none is
    mark = lambda f: 1 if f == 2 and pack.longest > SOLO_ROWS else f          # noqa: E731
    cut, halves = 0, None
    if backward and kv_form == 0 and q.shape[1] > k.shape[1]:
        cut = pack._cut(0 if causal else 1, k.shape[1])
        if cut:
            widest = max(k.shape[2], v.shape[2])
            halves = torch.empty(cut * k.shape[1] * 4 * L.PACKED_OWN_ROWS * (32 if widest <= 32 else 64 if widest <= 64 else 128),
                                 device=q.device, dtype=torch.float32)
    qr, qh, _ = q.stride()
    kr, kh, _ = k.stride()
    vr, vh, _ = v.stride()
    dr, dh, _ = dout.stride() if dout is not None else (0, 0, 0)
    args = L.PACKED_ATTN_FORMAT.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out, dout.data_ptr() if dout is not None else 0, o, dq,
                                     dk, dv, low, lse, delta, halves.data_ptr() if cut else 0, items, kv_items, qr, qh, kr, kh, vr, vh, dr, dh, pack.rows, n, n_kv,
                                     pack.uniform_length, len(pack.lengths), q.shape[1], k.shape[1], q.shape[2], v.shape[2],
                                     int(causal), mark(form), mark(kv_form), cut, scale)
    with L.on(q.device):
        L.check(so.mt_packed_attn_launch(args, backward, int(bf16), stream), "mt_packed_attn_launch")


def packed_forward(q, k, v, pack, causal: bool, scale: float, keeps: bool):
    """(output, what a backward pass needs) of operands as ``in_place`` leaves them."""
    so = L.load()
    out = torch.empty(pack.rows, q.shape[1], v.shape[2], device=q.device, dtype=q.dtype)
    lse = torch.empty(q.shape[1], pack.rows, device=q.device, dtype=torch.float32) if keeps else None
    # what rounding took off the outputs of rows that see few keys, whose gradients would show it
    low = torch.empty_like(out) if keeps and q.dtype == torch.bfloat16 and (causal or pack.shortest <= L.PACKED_LOW_ROWS) else None
    _packed_launch(so, pack, q, k, v, causal, scale, 0, o=out.data_ptr(), low=low.data_ptr() if low is not None else 0,
                   lse=lse.data_ptr() if keeps else 0)
    return out, (q, k, v, out, low, lse)


class PackedAttention(torch.autograd.Function):
    """``ops.attention.packed_attention`` on a GPU; operands checked and laid out there."""

    @staticmethod
    def forward(ctx, q, k, v, pack, causal: bool, scale: float):
        ctx.pack, ctx.meta = pack, (causal, scale)
        out, saved = packed_forward(q, k, v, pack, causal, scale, True)
        ctx.save_for_backward(*saved)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        so = L.load()
        q, k, v, out, low, lse = ctx.saved_tensors
        pack, (causal, scale) = ctx.pack, ctx.meta
        if L.formula_backward(grad_out):
            from .attention import packed_attention_plain
            plain = lambda *t: packed_attention_plain(*t, pack, causal, scale)                                          # noqa: E731
            return (*L.grads_by_formula(plain, (q, k, v), grad_out), None, None, None)
        do = in_place(grad_out if grad_out.dtype == q.dtype else grad_out.to(q.dtype))
        delta = torch.empty_like(lse)
        grads = [torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v)]
        _packed_launch(so, pack, q, k, v, causal, scale, 1, out=out.data_ptr(), dout=do, dq=grads[0].data_ptr(),
                       dk=grads[1].data_ptr(), dv=grads[2].data_ptr(), low=low.data_ptr() if low is not None else 0,
                       lse=lse.data_ptr(), delta=delta.data_ptr())
        return (*grads, None, None, None)
