"""Dense layers on hand-written MFMA kernels -- forward, input gradient and weight gradient.

``linear(x, weight, bias)`` is ``torch.nn.functional.linear`` on the CPU (the oracle the GPU tests compare with).  On a
GPU no call reaches a BLAS-library GEMM:

* bf16 autocast: ``DenseBF16`` -- all three GEMMs on the 128x128 bf16 tile kernel of ``csrc/gemm.hip``;
* f32, small layers (at most ``SMALL_MAX_ROWS`` rows and ``in x out <= SMALL_MAX_WEIGHTS`` -- every projection of the
  sequence-regression Transformers at batch 32 x 50 tokens): ``SmallLinear`` -- forward on the exact-f32 64-tile kernel,
  and the backward's three products (input gradient, weight gradient, bias column sum) in ONE launch of
  ``mt_small_linear_bwd_tiled_launch`` (``csrc/small_linear.hip``: sixteen waves per 32x32 tile adding their
  accumulators through LDS in a fixed order; no workspace and no traffic between workgroups).  Measured per backward
  inside a replayed graph (three library launches / this one, us): 800x64x256 61.5 / 6.4, 1600x10x32 20.5 / 6.6,
  1600x64x256 29.9 / 6.9, 1600x128x384 27.5 / 13.0, 3200x64x256 43.7 / 18.3; past the bound larger LDS-staged tiles
  catch up (4800x256x768 77.1 / 74.4) and the layer goes to
* f32, everything else: ``DenseF32`` on the exact-f32 tile kernel of ``csrc/gemm_f32.hip``; the weight + bias gradient
  ``dW = dY^T X`` -- a long skinny contraction over the token rows -- is split over enough workgroups to fill the chip
  and the partial slabs are added in a fixed order by one small launch.

``linear(x, weight, bias, activation=..., residual=...)`` is the layer with its activation (``"relu"`` or ``"gelu"``, the erf
form) and the addition of a residual in the GEMM's epilogue, ``act(x W^T + b) + residual`` rounded once (``FusedLinear``,
``csrc/linear_ep.hip``); it also takes bf16 parameters with bf16 activations, outside autocast, and gives their gradients in
bf16.  Under bf16 autocast ``x`` and the residual are rounded to bf16 first, like ``x`` of a plain layer, and the output is bf16.
For bf16 ``act'`` is taken of ``z`` rounded to bf16 (where ReLU has no residual: of the output, whose sign is ``z``'s), and the
gradients of ``x`` and ``weight`` are products of ``dz`` rounded to bf16.

The tile kernels read rows in 16-byte pieces, so a dimension that is not a multiple of 4 (f32) or 8 (bf16) -- 81 input
features, a scalar output -- is padded with zero columns / zero rows up to the next multiple before the launch and the
result is sliced back; autograd carries the slice through, so gradients of the padding are dropped.  Operands these
kernels cannot take at all (f16 or f64 on a GPU) raise ``TypeError`` instead of taking a slower road silently; so do, with
autograd's own errors, forward-mode differentiation and ``torch.func`` transforms of a call on a GPU.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
import torch.nn.functional as F

from ..options import OPTIONS
from . import lib as L

SMALL_MAX_ROWS = 32768
SMALL_MAX_WEIGHTS = 65536     # in x out, e.g. 128 x 512
SMALL_MAX_MACS = 1 << 29      # rows x in x out; measured wins up to here: 6144x128x512 66.5 / 51.7 us, 12288x64x192
                              # 109.4 / 58.3, 24576x64x128 135.8 / 110.4 (library / fused)


def _shadow(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """bf16 copy of a parameter kept current by the flat optimiser (``FlatParams(bf16_shadow=True)``), if there is one."""
    return getattr(t, "_mt_bf16", None) if t is not None else None


def _bf16_autocast() -> bool:
    return torch.is_autocast_enabled() and torch.get_autocast_dtype("cuda") == torch.bfloat16


def _small(rows: int, in_f: int, out_f: int, training: bool) -> bool:
    if in_f * out_f > SMALL_MAX_WEIGHTS or rows <= 0:
        return False
    return rows <= SMALL_MAX_ROWS and rows * in_f * out_f <= SMALL_MAX_MACS if training else rows <= 4 * SMALL_MAX_ROWS


def _pad_operands(x, weight, bias, mult: int):
    """Zero columns on x and weight up to a multiple of ``mult`` input features, zero rows on weight (and zeros on the
    bias) up to a multiple of ``mult`` output features."""
    out_f, in_f = weight.shape
    pi, po = (-in_f) % mult, (-out_f) % mult
    if pi:
        x, weight = F.pad(x, (0, pi)), F.pad(weight, (0, pi))
    if po:
        weight = F.pad(weight, (0, 0, 0, po))
        bias = F.pad(bias, (0, po)) if bias is not None else None
    return x, weight, bias


ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2}
MAX_FUSED_WIDTH = 2_000_000           # output features, and input features where x has a gradient: tile numbers are 16 bits
MAX_ROWS = (1 << 31) - 257            # with gradients: a weight gradient's contraction is counted in 32 bits
MAX_BF16_DW_WIDTH = 32767 * 128       # input features of a bf16 weight gradient, for the same reason


def _check_fused(x, weight, bias, activation, residual) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    xs, ws, device = x.shape, weight.shape, x.device
    if len(ws) != 2 or len(xs) < 1 or xs[-1] != ws[1]:
        raise ValueError(f"x {tuple(xs)} does not fit weight {tuple(ws)}")
    if bias is not None and bias.shape != ws[:1]:
        raise ValueError(f"bias must be [{ws[0]}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != xs[:-1] + ws[:1]:
        raise ValueError(f"residual must have the output's shape {tuple(xs[:-1] + ws[:1])}, got {tuple(residual.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.device != device:
            raise TypeError(f"{name} is on {t.device}, x on {device}")


def _plain_fused(x, weight, bias, activation, residual) -> torch.Tensor:
    y = F.linear(x, weight, bias)
    y = F.relu(y) if activation == "relu" else F.gelu(y) if activation == "gelu" else y
    return y if residual is None else y + residual


def _fused_linear(x, weight, bias, activation, residual) -> torch.Tensor:
    """The layer through ``FusedLinear``, operands brought to the types it takes."""
    w16 = None
    if torch.is_autocast_enabled():
        if not _bf16_autocast() or weight.dtype != torch.float32:
            raise TypeError("mitune.ops.linear under autocast takes f32 master weights and bf16 compute only, got "
                            f"autocast {torch.get_autocast_dtype('cuda')} / weight {weight.dtype}")
        x, w16 = x.to(torch.bfloat16), _shadow(weight)
        residual = residual.to(torch.bfloat16) if residual is not None else None
    elif x.dtype not in (torch.float32, torch.bfloat16) or weight.dtype != x.dtype:
        raise TypeError(f"mitune.ops.linear on a GPU takes f32 or bf16 operands of one type (or bf16 autocast), got x {x.dtype} "
                        f"/ weight {weight.dtype}")
    if bias is not None and bias.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"bias must be {x.dtype} or f32, got {bias.dtype}")
    if residual is not None and residual.dtype != x.dtype:
        raise TypeError(f"residual must be {x.dtype}, got {residual.dtype}")
    wants = L.wants_grad(x, weight, bias, residual) or L.transformed(x, weight, bias, residual)
    out_f, in_f = weight.shape
    if max(out_f, in_f) > MAX_FUSED_WIDTH and (out_f > MAX_FUSED_WIDTH or (wants and (
            x.requires_grad or (x.dtype == torch.bfloat16 and in_f > MAX_BF16_DW_WIDTH)))):
        raise ValueError(f"a dense layer on a GPU has at most {MAX_FUSED_WIDTH} output features, as many input features for the "
                         f"gradient of x, and {MAX_BF16_DW_WIDTH} for that of a weight beside bf16, got weight {tuple(weight.shape)}")
    if wants and x.numel() > MAX_ROWS * in_f:
        raise ValueError(f"a dense layer with gradients takes at most {MAX_ROWS} rows on a GPU, got x {tuple(x.shape)}")
    if wants:
        return FusedLinear.apply(x, weight, bias, residual, ACTIVATIONS[activation], w16)
    return fused_forward(x, weight, bias, residual, ACTIVATIONS[activation], w16, False)[0]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``; on a GPU always on this package's own MFMA kernels (see the module text)."""
    fused = activation is not None or residual is not None
    if fused:
        _check_fused(x, weight, bias, activation, residual)
    if not x.is_cuda or x.numel() == 0 or weight.numel() == 0:
        return _plain_fused(x, weight, bias, activation, residual)
    if not fused and x.dtype == weight.dtype == torch.bfloat16 and not torch.is_autocast_enabled():
        _check_fused(x, weight, bias, activation, residual)
        fused = True
    if fused:
        return _fused_linear(x, weight, bias, activation, residual)
    out_f, in_f = weight.shape
    if torch.is_autocast_enabled():
        if not _bf16_autocast() or weight.dtype != torch.float32:
            raise TypeError("mitune.ops.linear under autocast takes f32 master weights and bf16 compute only, got "
                            f"autocast {torch.get_autocast_dtype('cuda')} / weight {weight.dtype}")
        if out_f == 1:
            # a scalar head: a row-wise dot product in f32 (one multiply + one row reduction), not a GEMV
            with torch.autocast("cuda", enabled=False):
                y = (x.float() * weight.float().reshape(-1)).sum(-1, keepdim=True)
                return y if bias is None else y + bias.float()
        xb = x if x.dtype == torch.bfloat16 else x.to(torch.bfloat16)
        if out_f % 8 == 0 and in_f % 8 == 0:
            return DenseBF16.apply(xb, weight, bias, _shadow(weight))
        xp, wp, bp = _pad_operands(xb, weight, bias, 8)
        y = DenseBF16.apply(xp, wp, bp, None)
        return y if wp.shape[0] == out_f else y[..., :out_f]
    if x.dtype != torch.float32 or weight.dtype != torch.float32 or (bias is not None and bias.dtype != torch.float32):
        raise TypeError(f"mitune.ops.linear on a GPU takes f32 operands (or bf16 autocast), got x {x.dtype} / weight "
                        f"{weight.dtype}" + (f" / bias {bias.dtype}" if bias is not None else ""))
    rows = x.numel() // max(in_f, 1)
    training = torch.is_grad_enabled() and (weight.requires_grad or x.requires_grad)
    fn = SmallLinear if _small(rows, in_f, out_f, training) else DenseF32
    if out_f % 4 == 0 and in_f % 4 == 0:
        return fn.apply(x, weight, bias)
    xp, wp, bp = _pad_operands(x, weight, bias, 4)
    y = fn.apply(xp, wp, bp)
    return y if wp.shape[0] == out_f else y[..., :out_f]


def _wgrad_splits(M: int, tiles: int, rows_per_split: int) -> int:
    return max(1, min(127, (M + rows_per_split - 1) // rows_per_split,               # 127: split index field
                      (OPTIONS.wgrad_workgroups + tiles - 1) // tiles))


def _wgrad_bf16(dyc: torch.Tensor, xc: torch.Tensor, out_f: int, in_f: int, has_bias: bool):
    """dW [out, in] and db [out] (f32) of a bf16 layer: split-K tiles over the rows, ordered slab sum."""
    so = L.load()
    M = xc.shape[0]
    ksplits = _wgrad_splits(M, ((out_f + 127) // 128) * ((in_f + 127) // 128), 64)
    slab = (out_f * in_f + out_f + 63) // 64 * 64
    arena = torch.empty(ksplits, slab, device=xc.device, dtype=torch.float32)
    db_ptr = arena.data_ptr() + out_f * in_f * 4 if has_bias else None
    L.check(so.mt_wgrad_single_launch(dyc.data_ptr(), xc.data_ptr(), arena.data_ptr(), db_ptr, M, out_f, in_f,
                                      ksplits, slab, L.raw_stream(xc.device)),
            "mt_wgrad_single_launch")
    return _slab_total(so, arena, ksplits, slab, out_f, in_f, has_bias, L.raw_stream(xc.device))


def _wgrad_f32(dyc: torch.Tensor, xc: torch.Tensor, out_f: int, in_f: int, has_bias: bool):
    """dW [out, in] and db [out] of an f32 layer: the contraction over the token rows is split so that the launch has
    about ``OPTIONS.wgrad_workgroups`` workgroups (a slice keeps at least 4 K-steps of 32 rows), slices summed in index
    order."""
    so = L.load()
    M = xc.shape[0]
    ksplits = _wgrad_splits(M, ((out_f + 63) // 64) * ((in_f + 63) // 64), 128)
    slab = (out_f * in_f + out_f + 63) // 64 * 64
    arena = torch.empty(ksplits, slab, device=xc.device, dtype=torch.float32)
    stream = L.raw_stream(xc.device)
    L.check(so.mt_wgrad_f32_single_launch(dyc.data_ptr(), xc.data_ptr(), arena.data_ptr(), M, out_f, in_f, ksplits, slab,
                                          1 if has_bias else 0, stream), "mt_wgrad_f32_single_launch")
    return _slab_total(so, arena, ksplits, slab, out_f, in_f, has_bias, stream)


def _slab_total(so, arena, ksplits, slab, out_f, in_f, has_bias, stream):
    if ksplits > 1:       # slices added in index order by one launch (weights and bias together)
        total = torch.empty(slab, device=arena.device, dtype=torch.float32)
        L.check(so.mt_slab_sum_launch(arena.data_ptr(), total.data_ptr(), out_f * in_f + (out_f if has_bias else 0), ksplits,
                                      slab, stream), "mt_slab_sum_launch")
    else:
        total = arena[0]
    dw = total[:out_f * in_f].view(out_f, in_f)
    db = total[out_f * in_f:out_f * in_f + out_f] if has_bias else None
    return dw, db


class DenseBF16(torch.autograd.Function):
    """A dense layer under bf16 autocast, all three GEMMs on the 128x128 bf16 MFMA tile kernel of ``csrc/gemm.hip``.

    ``x`` arrives in bf16; the weight operand is the bf16 shadow the flat optimiser keeps (``w16``) or a cast of the f32
    master; the bias is added in f32 from the master before the output is rounded to bf16."""

    @staticmethod
    def forward(ctx, x, weight, bias, w16=None):
        so = L.load()
        out_f, in_f = weight.shape
        with torch.autocast("cuda", enabled=False):
            wb = w16 if w16 is not None else weight.detach().to(torch.bfloat16)
            xc = x.reshape(-1, in_f)
            if not xc.is_contiguous():
                xc = xc.contiguous()
            if not wb.is_contiguous():
                wb = wb.contiguous()
            bf = None if bias is None else (bias.detach() if bias.dtype == torch.float32 else bias.detach().float())
            y = torch.empty(xc.shape[0], out_f, device=x.device, dtype=torch.bfloat16)
            L.check(so.mt_gemm_single_launch(0, xc.data_ptr(), wb.data_ptr(), y.data_ptr(),
                                             bf.data_ptr() if bf is not None else None, xc.shape[0], out_f, in_f,
                                             in_f, in_f, out_f, 0, 0, L.raw_stream(x.device)), "mt_gemm_single_launch")
        ctx.save_for_backward(xc, wb)
        ctx.has_bias = bias is not None
        ctx.x_shape = x.shape
        return y.view(x.shape[:-1] + (out_f,))

    @staticmethod
    def backward(ctx, dy):
        so = L.load()
        xc, wb = ctx.saved_tensors
        out_f, in_f = wb.shape
        with torch.autocast("cuda", enabled=False):
            dyc = dy.reshape(-1, out_f)
            if dyc.dtype != torch.bfloat16:
                dyc = dyc.to(torch.bfloat16)
            if not dyc.is_contiguous():
                dyc = dyc.contiguous()
            dx = None
            if ctx.needs_input_grad[0]:
                dx = torch.empty(xc.shape[0], in_f, device=dy.device, dtype=torch.bfloat16)
                L.check(so.mt_gemm_single_launch(1, dyc.data_ptr(), wb.data_ptr(), dx.data_ptr(), None, xc.shape[0], in_f,
                                                 out_f, out_f, in_f, in_f, 0, 0, L.raw_stream(dy.device)),
                        "mt_gemm_single_launch")
                dx = dx.view(ctx.x_shape)
            dw, db = _wgrad_bf16(dyc, xc, out_f, in_f, ctx.has_bias)
        return dx, dw, db, None


def _f32_forward(x, weight, bias):
    """y = x W^T + b on the exact-f32 tile kernel; returns (y, x as [rows, in], W contiguous)."""
    so = L.load()
    out_f, in_f = weight.shape
    xc = x.reshape(-1, in_f)
    if not xc.is_contiguous():
        xc = xc.contiguous()
    wc = weight.detach()
    if not wc.is_contiguous():
        wc = wc.contiguous()
    y = torch.empty(xc.shape[0], out_f, device=x.device, dtype=torch.float32)
    L.check(so.mt_gemm_f32_single_launch(0, xc.data_ptr(), wc.data_ptr(), y.data_ptr(),
                                         bias.data_ptr() if bias is not None else None, None, xc.shape[0], out_f, in_f,
                                         in_f, in_f, out_f, 0, L.raw_stream(x.device)), "mt_gemm_f32_single_launch")
    return y.view(x.shape[:-1] + (out_f,)), xc, wc


class DenseF32(torch.autograd.Function):
    """An f32 dense layer on the exact-f32 MFMA tile kernel of ``csrc/gemm_f32.hip`` (forward, input gradient, and weight
    + bias gradient in one launch each)."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        y, xc, wc = _f32_forward(x, weight, bias)
        ctx.save_for_backward(xc, wc)
        ctx.has_bias = bias is not None
        ctx.x_shape = x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        so = L.load()
        xc, wc = ctx.saved_tensors
        out_f, in_f = wc.shape
        dyc = dy.reshape(-1, out_f)
        if dyc.dtype != torch.float32:
            dyc = dyc.float()
        if not dyc.is_contiguous():
            dyc = dyc.contiguous()
        M, dev = xc.shape[0], dy.device
        dx = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty(M, in_f, device=dev, dtype=torch.float32)
            L.check(so.mt_gemm_f32_single_launch(1, dyc.data_ptr(), wc.data_ptr(), dx.data_ptr(), None, None, M, in_f, out_f,
                                                 out_f, in_f, in_f, 0, L.raw_stream(dev)), "mt_gemm_f32_single_launch")
            dx = dx.view(ctx.x_shape)
        dw, db = _wgrad_f32(dyc, xc, out_f, in_f, ctx.has_bias)
        return dx, dw, db


class SmallLinear(torch.autograd.Function):
    """A small f32 dense layer: forward on the exact-f32 64-tile kernel, the whole backward in one launch."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        y, xc, wc = _f32_forward(x, weight, bias)
        ctx.save_for_backward(xc, wc)
        ctx.has_bias = bias is not None
        ctx.x_shape = x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        so = L.load()
        xc, wc = ctx.saved_tensors
        out_f, in_f = wc.shape
        dyc = dy.reshape(-1, out_f)
        if not dyc.is_contiguous():
            dyc = dyc.contiguous()
        R, dev = xc.shape[0], xc.device
        dx = torch.empty(R, in_f, device=dev, dtype=torch.float32) if ctx.needs_input_grad[0] else None
        dw = torch.empty(out_f, in_f, device=dev, dtype=torch.float32)
        db = torch.empty(out_f, device=dev, dtype=torch.float32) if ctx.has_bias else None
        L.check(so.mt_small_linear_bwd_tiled_launch(xc.data_ptr(), wc.data_ptr(), dyc.data_ptr(),
                                                    dx.data_ptr() if dx is not None else None, dw.data_ptr(),
                                                    db.data_ptr() if db is not None else None, R, in_f, out_f,
                                                    OPTIONS.small_linear_tile, L.raw_stream(dev)),
                "mt_small_linear_bwd_tiled_launch")
        return (dx.view(ctx.x_shape) if dx is not None else None), dw, db


@functools.lru_cache(maxsize=1024)
def _gemm_parts(mode: int, M: int, N: int, depth: int, bf16: int) -> int:
    return L.load().mt_linear_parts(mode, M, N, depth, bf16)


@functools.lru_cache(maxsize=1024)
def _act_parts(M: int, columns: int, bf16: int) -> int:
    return L.load().mt_linear_act_parts(M, columns, bf16)


def _pieces(t: torch.Tensor) -> torch.Tensor:
    """``t`` [rows, columns] with rows of whole 16-byte pieces: itself when its rows start on such a boundary (less than 2^24 elements
    apart) and its width is a multiple of one, else a copy padded with zero columns."""
    per = 16 // t.element_size()
    width, (apart, step) = t.shape[1], t.stride()
    pad = -width % per
    if pad == 0 and step == 1 and apart % per == 0 and width <= apart < 1 << 24 and t.data_ptr() % 16 == 0:
        return t
    return F.pad(t, (0, pad)).contiguous() if pad else t.clone(memory_format=torch.contiguous_format)


def _rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    return t if t.dim() == 2 else t.reshape(-1, width)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _fused_gemm(so, mode: int, a, b, c, depth: int, stream, bias=None, residual=None, z=None, act: int = 0) -> None:
    """c = act(a b + bias) + residual: b is [columns, depth] in mode 0, [depth, columns] in mode 1."""
    M, N = c.shape
    bf16 = int(c.dtype == torch.bfloat16)
    n = _gemm_parts(mode, M, N, depth, bf16)
    part = torch.empty(n, M, N, device=c.device, dtype=torch.float32) if n > 1 else None
    L.check(so.mt_linear_gemm_launch(mode, a.data_ptr(), b.data_ptr(), _ptr(bias), _ptr(residual), c.data_ptr(), _ptr(z), _ptr(part),
                                     M, N, depth, a.stride(0), b.stride(0), act,
                                     int(bias is not None and bias.dtype == torch.bfloat16), bf16, stream), "mt_linear_gemm_launch")


def fused_forward(x, weight, bias, residual, act: int, w16, keep_z: bool):
    """(output, x's rows, the weight as multiplied, z or None)."""
    so = L.load()
    out_f, in_f = weight.shape
    dtype, dev = x.dtype, x.device
    xc = _pieces(_rows_of(x, in_f))
    wc = w16 if w16 is not None else weight if weight.dtype == dtype else weight.detach().to(dtype)
    wc = _pieces(wc)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    rc = _rows_of(residual, out_f).contiguous() if residual is not None else None
    y = torch.empty(xc.shape[0], out_f, device=dev, dtype=dtype)
    z = torch.empty_like(y) if keep_z else None
    with L.on(dev):
        _fused_gemm(so, 0, xc, wc, y, xc.shape[1], L.raw_stream(dev), bias, rc, z, act)
    return (y if x.dim() == 2 else y.view(x.shape[:-1] + (out_f,))), xc, wc, z


class FusedLinear(torch.autograd.Function):
    """``act(x W^T + b) + residual`` with x, W, residual and the output of one type, f32 or bf16 (under bf16 autocast W is the
    f32 master and its gradient f32); operands checked in ``linear``."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int, w16):
        backward = any(ctx.needs_input_grad[:3])
        # what act' is read from: y itself has z's sign under ReLU, unless a residual was added to it
        keep_z = backward and act != 0 and not (act == 1 and residual is None)
        y, xc, wc, z = fused_forward(x, weight, bias, residual, act, w16, keep_z)
        if backward:
            # x and the weight as multiplied, mostly they themselves; a second differentiation needs those it is asked for
            ctx.save_for_backward(xc, wc, z if keep_z else y if act else None, None if xc is x else x,
                                  None if wc is weight else weight, bias if act else None)
        ctx.meta = (act, x.shape, weight.shape[1], weight.dtype, bias.dtype if bias is not None else None,
                    residual.shape if residual is not None else None)
        return y

    @staticmethod
    def backward(ctx, dy):
        so = L.load()
        act, x_shape, in_f, w_dtype, b_dtype, r_shape = ctx.meta
        dx = dw = db = None
        if any(ctx.needs_input_grad[:3]):
            xc, wc, s, x, weight, bias = ctx.saved_tensors
            if L.formula_backward(dy):
                return _twice_differentiable(ctx, dy, xc if x is None else x, wc if weight is None else weight, bias)
            out_f = wc.shape[0]
            bf16, dev, M = xc.dtype == torch.bfloat16, xc.device, xc.shape[0]
            per = 8 if bf16 else 4
            stream = L.raw_stream(dev)
            with L.on(dev):
                g = _rows_of(dy if dy.dtype == xc.dtype else dy.to(xc.dtype), out_f)
                if act:
                    g = g if g.stride(1) == 1 else g.contiguous()
                    width = out_f + -out_f % per
                else:
                    g = _pieces(g)
                    # (a single row is contiguous to torch whatever its row stride is: clone, not contiguous)
                    g = g if g.stride(0) == g.shape[1] else g.clone(memory_format=torch.contiguous_format)
                    width = g.shape[1]
                need_x, need_w, need_b = ctx.needs_input_grad[:3]
                need_b = need_b and b_dtype is not None
                need_w = need_w or (need_b and not _early_sums(bf16, act))          # sums over dz's rows come with dW, or from act'
                plan = _bwd_plan(M, out_f, width, in_f, xc.shape[1], act, bf16, w_dtype == xc.dtype, need_x, need_w, need_b,
                                 OPTIONS.wgrad_workgroups)
                if plan is not None:
                    size, at, slab, splits = plan
                    n, k = out_f, in_f                # of the gradients as they are stored
                    if splits < 0:
                        need_w, n, k = True, width, xc.shape[1]
                        wc = F.pad(wc, (0, 0, 0, n - out_f)) if n != out_f else wc if wc.stride(0) == k else wc.contiguous()
                    xc = xc if xc.stride(0) == xc.shape[1] else xc.contiguous()
                    ws = torch.empty(size, device=dev, dtype=torch.uint8) if size else None
                    dx = torch.empty(x_shape if k == in_f else (M, k), device=dev, dtype=xc.dtype) if need_x else None
                    dw = torch.empty(n, k, device=dev, dtype=w_dtype) if need_w else None
                    db = torch.empty(n, device=dev, dtype=b_dtype) if need_b else None
                    args = L.LINEAR_BWD_FORMAT.pack(g.data_ptr(), s.data_ptr() if act else 0, xc.data_ptr(), wc.data_ptr(),
                                                    dx.data_ptr() if need_x else 0, dw.data_ptr() if need_w else 0,
                                                    db.data_ptr() if need_b else 0, ws.data_ptr() if size else 0, M, g.stride(0),
                                                    wc.stride(0), *at, slab, out_f, in_f, width, xc.shape[1], act, bf16,
                                                    w_dtype == torch.bfloat16, b_dtype == torch.bfloat16, splits,
                                                    OPTIONS.small_linear_tile)
                    L.check(so.mt_linear_bwd_launch(args, stream), "mt_linear_bwd_launch")
                    if n != out_f:
                        dw, db = dw[:out_f], db[:out_f] if need_b else None
                    if k != in_f:
                        dx, dw = dx[:, :in_f].reshape(x_shape) if need_x else None, dw[:, :in_f]
                    return dx, dw, db, (dy if r_shape is not None else None), None, None
                # more bf16 output features than one weight gradient launch takes
                if act:
                    dz = torch.empty(M, width, device=dev, dtype=xc.dtype)
                    part = None
                    if _early_sums(bf16, act) and b_dtype is not None and ctx.needs_input_grad[2]:
                        db = torch.empty(out_f, device=dev, dtype=b_dtype)
                        part = torch.empty(_act_parts(M, width, 1), out_f, device=dev, dtype=torch.float32)
                    L.check(so.mt_linear_act_bwd_launch(g.data_ptr(), s.data_ptr(), dz.data_ptr(),
                                                        part.data_ptr() if part is not None else None,
                                                        db.data_ptr() if part is not None else None, M, out_f, g.stride(0),
                                                        width, act, int(b_dtype == torch.bfloat16), 1, stream),
                            "mt_linear_act_bwd_launch")
                    b_dtype = None if part is not None else b_dtype
                else:
                    dz = g
                if ctx.needs_input_grad[0]:
                    dx = torch.empty(M, in_f, device=dev, dtype=xc.dtype)
                    _fused_gemm(so, 1, dz, wc, dx, out_f, stream)
                    dx = dx if len(x_shape) == 2 else dx.view(x_shape)
                if ctx.needs_input_grad[1] or (b_dtype is not None and ctx.needs_input_grad[2]):
                    dw, sums = _weight_grad(so, dz, xc, out_f, in_f, w_dtype, b_dtype, stream)
                    db = db if sums is None else sums
        return dx, dw, db, (dy if r_shape is not None else None), None, None


def _twice_differentiable(ctx, dy, x, weight, bias):
    act, _, _, _, b_dtype, r_shape = ctx.meta
    name = next(n for n, number in ACTIVATIONS.items() if number == act)
    if b_dtype is not None and bias is None:           # no activation: nothing depends on its value
        bias = torch.zeros(weight.shape[0], device=weight.device, dtype=b_dtype, requires_grad=ctx.needs_input_grad[2])
    cast = lambda t: None if t is None else t.float()                                                      # noqa: E731
    plain = lambda x, w, b: _plain_fused(x.float(), w.float(), cast(b), name, None).to(dy.dtype)           # noqa: E731
    return (*L.grads_by_formula(plain, (x, weight, bias), dy), dy if r_shape is not None else None, None, None)


def _early_sums(bf16: bool, act: int) -> bool:
    """Whether db is summed from dz before its rounding, by the pass that forms dz: where that rounds, which ReLU's does not."""
    return bf16 and act == ACTIVATIONS["gelu"]


@functools.lru_cache(maxsize=1024)
def _bwd_plan(M: int, out_f: int, rows: int, in_f: int, width: int, act: int, bf16: bool, same: bool, need_x: bool, need_w: bool,
              need_b: bool, workgroups: int):
    """How ``mt_linear_bwd_launch`` computes a layer's gradients: (bytes of workspace, where dz, the column sums, the parts of dx and
    those of dW lie in it (-1: not there), floats from part to part of dW, how many; 0: unsplit, -1: a small f32 layer,
    gradients with padded widths).  None: a layer whose weight gradient takes several launches.  Kept per shape; ``workgroups`` is
    the option that the split follows."""
    small = not bf16 and _small(M, width, rows, True)
    size, at = 0, []

    def take(wanted, count) -> None:
        nonlocal size
        at.append(size if wanted else -1)
        size += -(-count // 256) * 256 if wanted else 0

    early = _early_sums(bf16, act) and need_b
    take(act != 0, M * rows * (2 if bf16 else 4))
    take(early, _act_parts(M, rows, 1) * out_f * 4 if early else 0)
    if small:
        return size, (*at, -1, -1), 0, -1
    parts = _gemm_parts(1, M, in_f, out_f, int(bf16)) if need_x else 1
    take(parts > 1, parts * M * in_f * 4)
    tile = 128 if bf16 else 64
    most = 255 * tile if bf16 else rows
    splits = _fused_wgrad_splits(M, -(-min(rows, most) // tile) * -(-width // tile), bf16)
    if not need_w or (same and splits == 1):
        return size, (*at, -1), 0, 0
    if rows > most:
        return None
    slab = (rows * width + rows + 63) // 64 * 64
    take(True, splits * slab * 4)
    return size, tuple(at), slab, splits


def _fused_wgrad_splits(M: int, tiles: int, bf16: bool) -> int:
    """Row splits of a fused layer's weight gradient.  f32: four workgroups per CU (with the sum over them, 12800 x 512 x 2048 with
    its 256 tiles: 225 us in 2 splits, 206 in 4, 212 in 8; 25600 x 512 x 512 with 64: 112 us in 8, 110 in 16, 119 in 32); bf16:
    ``OPTIONS.wgrad_workgroups``."""
    return _wgrad_splits(M, tiles, 64) if bf16 else max(1, min(127, (M + 127) // 128, 1024 // tiles))


def _weight_grad(so, dz, xc, out_f: int, in_f: int, w_dtype, b_dtype, stream):
    """(dW [out_f, in_f], db [out_f] or None) of a bf16 layer of more output features than a launch takes (its tile rows are 8 bits):
    each part split over the rows, the slabs added in order and rounded once."""
    M, width, rows = dz.shape[0], xc.shape[1], dz.shape[1]
    xc = xc if xc.stride(0) == width else xc.contiguous()
    most = 255 * 128
    dw = torch.empty(out_f, in_f, device=dz.device, dtype=w_dtype)
    db = torch.empty(out_f, device=dz.device, dtype=b_dtype) if b_dtype is not None else None
    for r in range(0, rows, most):
        part = dz[:, r:r + most].contiguous()
        n = part.shape[1]
        real = min(n, out_f - r)
        splits = _fused_wgrad_splits(M, -(-n // 128) * -(-width // 128), True)
        slab = (n * width + n + 63) // 64 * 64
        arena = torch.empty(splits, slab, device=dz.device, dtype=torch.float32)
        L.check(so.mt_wgrad_single_launch(part.data_ptr(), xc.data_ptr(), arena.data_ptr(),
                                          arena.data_ptr() + n * width * 4 if db is not None else None, M, n, width, splits, slab,
                                          stream), "mt_wgrad_single_launch")
        L.check(so.mt_linear_wsum_launch(arena.data_ptr(), dw[r:].data_ptr(), db[r:].data_ptr() if db is not None else None, real, in_f,
                                         width, n * width, splits, slab, int(w_dtype == torch.bfloat16), int(b_dtype == torch.bfloat16),
                                         stream), "mt_linear_wsum_launch")
    return dw, db
