"""Fused dropout + residual add + LayerNorm: ``LN(residual + dropout(x))``.

This is the step that closes both halves of a post-norm encoder block
(/root/reference/ray-tune-hpo-regression.py:172,176).  As separate PyTorch ops it is three
memory-bound passes over [tokens, d]; fused it is one read of each input and one write.  On a GPU
``ops/csrc/layernorm.hip`` runs it with one wave per row (forward and backward); elsewhere the
reference below is used.

``layer_norm`` is the norm alone, over rows of any width in f32 or bf16 (``ops/csrc/norm.hip``).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

from .layernorm_hip import LayerNorm, norm_forward
from .lib import transformed, wants_grad


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, differentiable, in ``x``'s type; statistics and
    column sums in f32.  ``weight`` and ``bias`` ([d], either may be missing) have ``x``'s type, or f32 beside a bf16 ``x``.  On a
    GPU ``x`` is f32 or bf16, rows of any width; rows may lie apart (a column slice of a wider tensor is read in place).  Second
    derivatives, forward-mode differentiation, ``torch.func`` transforms and tracing go through plain torch."""
    shape, device = x.shape, x.device
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"layer_norm needs rows of at least one column, got {tuple(shape)}")
    d = shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (d,):
            raise ValueError(f"{name} must be [{d}], got {tuple(t.shape)}")
        if t.device != device:
            raise TypeError(f"{name} is on {t.device}, x on {device}")
        if t.dtype != x.dtype and not (x.dtype == torch.bfloat16 and t.dtype == torch.float32):
            raise TypeError(f"{name} must be {x.dtype} (or f32 beside a bf16 x), got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must share a type, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if x.is_cuda and x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"layer_norm on a GPU takes f32 or bf16 rows, got {x.dtype}")
    if not x.is_cuda or transformed(x, weight, bias):
        wide = torch.promote_types(x.dtype, weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype)
        cast = lambda t: None if t is None else t.to(wide)          # noqa: E731
        return F.layer_norm(x.to(wide), (d,), cast(weight), cast(bias), eps).to(x.dtype)
    if d > 1 << 29:
        raise ValueError(f"layer_norm on a GPU takes rows of at most {1 << 29} columns, got {d}")
    if wants_grad(x, weight, bias):
        return LayerNorm.apply(x, weight, bias, float(eps))
    return norm_forward(x, weight, bias, float(eps), False)[0]


def residual_layer_norm_reference(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                                  bias: torch.Tensor, eps: float = 1e-5,
                                  keep_mask: Optional[torch.Tensor] = None, dropout_p: float = 0.0) -> torch.Tensor:
    if keep_mask is not None:
        x = x * keep_mask.to(x.dtype) * (1.0 / (1.0 - dropout_p))
    return F.layer_norm(residual + x, (x.shape[-1],), weight, bias, eps)


def residual_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                        eps: float = 1e-5, dropout_p: float = 0.0) -> torch.Tensor:
    fused = x.is_cuda and x.dtype == torch.float32 and x.shape[-1] <= 2048 and x.shape[-1] % 4 == 0
    if fused:
        from .layernorm_hip import FusedResidualLayerNorm, available
        if available():
            seed = None
            if dropout_p > 0.0:           # the mask is drawn inside the kernel from a device-resident seed
                from .rng import next_seed
                seed = next_seed(x.device)
            return FusedResidualLayerNorm.apply(x, residual, weight, bias, eps, None, dropout_p, seed)
    keep = None
    if dropout_p > 0.0:
        from .elementwise import keep_mask
        keep = keep_mask(x.shape, dropout_p, x.device)
    if (x.is_cuda and not torch.compiler.is_compiling() and x.dtype in (torch.float32, torch.bfloat16)
            and all(t is None or t.dtype == x.dtype for t in (residual, weight, bias)) and x.shape == residual.shape
            and not torch.is_autocast_enabled() and not transformed(x, residual, weight, bias)):
        if keep is not None:                # rows the fused kernels do not take: the norm alone on its own kernels
            x = x * keep.to(x.dtype) * (1.0 / (1.0 - dropout_p))
        return layer_norm(residual + x, weight, bias, eps)
    return residual_layer_norm_reference(x, residual, weight, bias, eps, keep, dropout_p)


def residual_layer_norm_mixed(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                              eps: float = 1e-5, dropout_p: float = 0.0, want_bf16: bool = True):
    """``(y, y16)``: ``y = LayerNorm(residual + dropout(x))`` in f32 (the residual stream) and its bf16 copy for the next
    GEMM (``None`` when ``want_bf16`` is false).  ``x`` may be the bf16 output of an autocast GEMM: on a GPU with rows of at
    most 256 columns one kernel per direction does all of it (``csrc/layernorm.hip``, mixed forms); elsewhere the f32 path
    plus explicit casts."""
    d = x.shape[-1]
    if (x.is_cuda and d <= 256 and d % 4 == 0 and x.dtype in (torch.float32, torch.bfloat16)
            and residual.dtype == torch.float32):
        from .layernorm_hip import MixedResidualLayerNorm, available
        if available():
            seed = None
            if dropout_p > 0.0:
                from .rng import next_seed
                seed = next_seed(x.device)
            out = MixedResidualLayerNorm.apply(x, residual, weight, bias, eps, dropout_p, seed, bool(want_bf16))
            return out if want_bf16 else (out, None)
    y = residual_layer_norm(x.float(), residual.float(), weight, bias, eps, dropout_p)
    return y, (y.to(torch.bfloat16) if want_bf16 else None)
