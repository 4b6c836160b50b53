"""Attention: fused HIP kernels on a GPU, plain PyTorch elsewhere.

**Packed sequences of any length** (``packed_attention``): rows of sequences of different lengths one after the other, causal
or not, query heads in groups that share a key / value head, forward and backward (``ops/csrc/packed_attention.hip``).
``self_attention`` and ``self_attention_qkv`` use it past the short kernels' 128 tokens for softmax scores without dropout (evaluation,
and training with an attention dropout of 0); with dropout they run ``attention_reference`` there, scores and mask in memory.

**Short sequences**: one fused kernel per direction.

The reference's sequences are 50 or 96 tokens long
(/root/reference/ray-tune-hpo-regression-sample.py:28, /root/reference/ray-tune-hpo-regression.py:446), so a
whole (batch, head) problem -- Q, K, V and the S x S score tile -- fits in one workgroup's LDS and
registers: no flash-style streaming or online softmax is needed.  Two score functions share the
kernels:

* ``"softmax"``: ``P = softmax(Q K^T / sqrt(dk))``                      (``nn.MultiheadAttention`` semantics)
* ``"relu"``   : ``A = relu(Q K^T / sqrt(dk)); P = A / (rowsum(A) + eps)``  (the reference's softmax-free
  "LinearAttention", :113-117, with a row normalisation so the output scale does not grow with S).

``short_attention`` is differentiable.  On a GPU, shapes inside the kernel envelope (S <= 128, head
dims <= 64 and multiples of 8) run ``ops/csrc/attention.hip`` (bf16 MFMA, f32 softmax and
accumulation); anything else, and every CPU call, runs ``attention_reference``.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import numpy as np
import torch

from .lib import PACKED_ITEM_BYTES, PACKED_OWN_ROWS, PACKED_SPLIT_ROWS, transformed

RELU_EPS = 1e-6
MAX_SEQ = 128
MAX_HEAD_DIM = 64


def attention_reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kind: str = "softmax",
                        keep_mask: Optional[torch.Tensor] = None, dropout_p: float = 0.0) -> torch.Tensor:
    """q, k: [..., S, dk]; v: [..., S, dv]; ``keep_mask`` ([..., S, S], 0/1) applies attention dropout."""
    s = (q @ k.transpose(-2, -1)) * (1.0 / math.sqrt(q.shape[-1]))
    if kind == "softmax":
        p = torch.softmax(s, dim=-1)
    elif kind == "relu":
        a = torch.relu(s)
        p = a / (a.sum(-1, keepdim=True) + RELU_EPS)
    else:
        raise ValueError(f"kind must be 'softmax' or 'relu', got {kind!r}")
    if keep_mask is not None:
        p = p * keep_mask.to(p.dtype) * (1.0 / (1.0 - dropout_p))
    return p @ v


def _hip_ok(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> bool:
    if not q.is_cuda or q.dim() != 4:
        return False
    s, dk, dv = q.shape[-2], q.shape[-1], v.shape[-1]
    return (s <= MAX_SEQ and dk <= MAX_HEAD_DIM and dv <= MAX_HEAD_DIM and dk % 8 == 0 and dv % 8 == 0
            and k.shape[-2] == s and v.shape[-2] == s)


def short_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kind: str = "softmax",
                    dropout_p: float = 0.0) -> torch.Tensor:
    """Self-attention over short sequences, [B, h, S, d] in and out."""
    keep = None
    if dropout_p > 0.0:
        shape = q.shape[:-1] + (k.shape[-2],)
        from .elementwise import keep_mask
        keep = keep_mask(shape, dropout_p, q.device)
    if _hip_ok(q, k, v):
        from .attention_hip import FusedShortAttention, available
        if available():
            return FusedShortAttention.apply(q, k, v, kind, keep, dropout_p)
    return attention_reference(q, k, v, kind, keep, dropout_p)


WIDE_HEAD_DIM = 128      # heads of 65..128 elements fit the kernels' LDS budget for sequences of at most WIDE_MAX_SEQ tokens
WIDE_MAX_SEQ = 96


def _kernel_envelope(t: torch.Tensor, S: int, dk: int, dv: int) -> bool:
    """Strided (projection-output) operands: any head width from 1 to 64 -- widths that are not multiples of 8 are staged
    element by element -- and up to 128 for short sequences."""
    if not (t.is_cuda and t.dtype in (torch.float32, torch.bfloat16) and S <= MAX_SEQ and dk > 0 and dv > 0):
        return False
    widest = max(dk, dv)
    return widest <= MAX_HEAD_DIM or (widest <= WIDE_HEAD_DIM and S <= WIDE_MAX_SEQ)


def _packed_envelope(t: torch.Tensor, dk: int, dv: int, kind: str, dropout_p: float, *more: torch.Tensor) -> bool:
    """What the kernels for sequences of any length take of the calls below: softmax scores without dropout, outside of transforms and
    of compiled code, which plain torch leaves in one graph."""
    return (t.is_cuda and not torch.compiler.is_compiling() and t.dtype in (torch.float32, torch.bfloat16) and t.numel() > 0
            and kind == "softmax" and dropout_p == 0.0 and 0 < dk <= PACKED_MAX_HEAD_DIM and 0 < dv <= PACKED_MAX_HEAD_DIM
            and not transformed(t, *more))


def _packed_self_attention(qkv, B: int, S: int, h: int, dk: int, dv: int) -> torch.Tensor:
    """[B, S, h*dv] of queries, keys and values [B*S, h, width] each, on the packed kernels."""
    q, k, v = (t.unflatten(1, (h, d)) for t, d in zip(qkv, (dk, dk, dv)))
    return packed_attention(q, k, v, SequencePack.uniform(B, S, device=q.device)).reshape(B, S, h * dv)


def self_attention_qkv(qkv: torch.Tensor, num_heads: int, dk: int, kind: str = "softmax",
                       dropout_p: float = 0.0) -> torch.Tensor:
    """Multi-head self-attention on ONE fused projection output ``qkv`` [B, S, 2*h*dk + h*dv]: all queries, all keys,
    all values, each block head-major.  On a GPU the kernels read the three blocks in place and return one gradient
    tensor for the projection (sequences past the short kernels' envelope, softmax without dropout: the packed kernels read
    them in place too); elsewhere the blocks are split and ``self_attention`` runs."""
    B, S, W = qkv.shape
    h = num_heads
    dv = (W - 2 * h * dk) // h
    if _kernel_envelope(qkv, S, dk, dv):
        from .attention_hip import FusedQKVAttention, available
        if available():
            seed = None
            if dropout_p > 0.0:
                from .rng import next_seed
                seed = next_seed(qkv.device)
            return FusedQKVAttention.apply(qkv, h, dk, kind, dropout_p, seed)
    if _packed_envelope(qkv, dk, dv, kind, dropout_p):
        return _packed_self_attention(qkv.reshape(B * S, W).split([h * dk, h * dk, h * dv], dim=1), B, S, h, dk, dv)
    qk, v = qkv.split([2 * h * dk, h * dv], dim=-1)
    return self_attention(qk, v, h, kind, dropout_p)


def self_attention(qk: torch.Tensor, v: torch.Tensor, num_heads: int, kind: str = "softmax",
                   dropout_p: float = 0.0) -> torch.Tensor:
    """Multi-head self-attention on projection outputs: ``qk`` [B, S, 2*h*dk] (all queries, then all keys, head-major),
    ``v`` [B, S, h*dv]; returns [B, S, h*dv].  On a GPU the fused kernels read these tensors in place (no head
    split/merge copies, no casts), past their envelope the packed kernels (softmax, no dropout); elsewhere the heads are split
    and ``attention_reference`` runs."""
    B, S, w2 = qk.shape
    h = num_heads
    dk, dv = w2 // (2 * h), v.shape[-1] // h
    if _kernel_envelope(qk, S, dk, dv):
        from .attention_hip import FusedSelfAttention, available
        if available():
            seed = None
            if dropout_p > 0.0:           # no [B, h, S, S] mask tensor: the kernels hash (seed, element index)
                from .rng import next_seed
                seed = next_seed(qk.device)
            return FusedSelfAttention.apply(qk, v, h, kind, None, dropout_p, seed)
    if _packed_envelope(qk, dk, dv, kind, dropout_p, v) and v.dtype == qk.dtype:
        return _packed_self_attention(qk.reshape(B * S, w2).chunk(2, dim=1) + (v.reshape(B * S, h * dv),), B, S, h, dk, dv)
    keep = None
    if dropout_p > 0.0:
        from .elementwise import keep_mask
        keep = keep_mask((B, h, S, S), dropout_p, qk.device)
    q, k = qk.chunk(2, dim=-1)
    split = lambda t, d: t.reshape(B, S, h, d).transpose(1, 2)          # noqa: E731
    o = attention_reference(split(q, dk), split(k, dk), split(v, dv), kind, keep, dropout_p)
    return o.transpose(1, 2).reshape(B, S, h * dv)


# ---- packed sequences -----------------------------------------------------------------------------------------------------
PACKED_MAX_HEAD_DIM = 128
SOLO_ROWS = 256          # packs' short sequences: see attention_hip.packed_form


class SequencePack:
    """Where the sequences of a packed batch lie: sequence ``i`` takes the ``lengths[i]`` rows after those before it, and
    ``rows`` (default: their sum) is the number of rows of the tensors; rows behind the last sequence belong to none.

    Made once per batch and used by every layer and both passes: the lengths are checked on the host, and the list of
    pieces the kernels work through, longest first, is laid out on ``device`` (default: the current GPU if there is
    one); a captured graph reads that list, so the pack has to live as long as the graph.
    ``SequencePack.uniform(count, length)`` is ``count`` sequences of one length; it needs no list."""

    def __init__(self, lengths: Union[Sequence[int], np.ndarray, torch.Tensor], rows: Optional[int] = None, device=None):
        if isinstance(lengths, torch.Tensor):
            if lengths.is_cuda:
                raise TypeError("SequencePack takes the lengths on the host (a list, an array or a CPU tensor)")
            lengths = lengths.numpy()
        n = np.asarray(lengths)
        if n.size == 0:
            n = n.reshape(-1).astype(np.int64)
        if n.ndim != 1 or n.dtype.kind not in "iu":
            raise TypeError("lengths must be a flat list of whole numbers")
        if (n < 0).any():
            raise ValueError("a sequence's length cannot be negative")
        # summed as Python integers: an int64 sum of absurd lengths could wrap around the check below
        total = sum(int(v) for v in n)
        self._fix(total, total if rows is None else rows, device)
        self.lengths = n.astype(np.int64)
        self.longest = int(self.lengths.max(initial=0))
        self.shortest = int(self.lengths.min(initial=1 << 31, where=self.lengths > 0))
        self.uniform_length = 0
        self._lay_out()

    @classmethod
    def uniform(cls, count: int, length: int, device=None) -> "SequencePack":
        if count < 0 or length < 0:
            raise ValueError("a pack has no negative counts or lengths")
        self = cls.__new__(cls)
        self._fix(int(count) * int(length), int(count) * int(length), device)
        self.lengths = np.full(int(count), int(length), dtype=np.int64)
        self.longest = self.shortest = int(length) if count else 0
        self.uniform_length = int(length) if count else 0
        own, fine = (-(-int(length) // r) * int(count) for r in (PACKED_OWN_ROWS, PACKED_SPLIT_ROWS))
        self._counts, self._lists, self._stream = (own, fine, own if length <= SOLO_ROWS else fine), None, 0
        self._cuts = {}
        return self

    def _fix(self, total: int, rows: int, device) -> None:
        rows = int(rows)
        if rows < total:
            raise ValueError(f"sequences of {total} rows do not fit {rows} rows")
        if rows > 0x7FFFFFFF - PACKED_OWN_ROWS:
            raise ValueError(f"a pack holds at most {0x7FFFFFFF - PACKED_OWN_ROWS} rows, got {rows}")
        device = torch.device(device if device is not None else ("cuda" if torch.cuda.is_available() else "cpu"))
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.total, self.rows, self.device = total, rows, device

    def _lay_out(self) -> None:
        """Three lists of items (``{first row of the sequence, its length, item's first row in it, solo}``): 128 rows each; 32 rows
        each; and 128 rows walked alone by four waves for sequences of at most ``SOLO_ROWS`` rows, else 32.  Each in three orders,
        most work first: by keys up to the item's end (causal queries), by queries from its start (causal keys), by length (all
        see all).  Rows of no sequence follow as entries of negative length, which the kernels fill with zeros."""
        n = self.lengths
        starts = np.concatenate([[0], np.cumsum(n)])[:-1]
        at = np.arange(self.total, self.rows, PACKED_OWN_ROWS)
        tail = np.zeros((len(at), 4), dtype=np.int32)
        tail[:, 0], tail[:, 1] = at, -np.minimum(PACKED_OWN_ROWS, self.rows - at)
        short = n <= SOLO_ROWS
        lists, counts = [], []
        for solo in (np.zeros_like(short), np.zeros_like(short), short):
            grain = np.where(solo, PACKED_OWN_ROWS, PACKED_SPLIT_ROWS) if len(lists) else np.full(len(n), PACKED_OWN_ROWS)
            parts = -(-n // grain)
            seq = np.repeat(np.arange(len(n)), parts)
            first = (np.arange(len(seq)) - np.repeat(np.cumsum(parts) - parts, parts)) * grain[seq]
            items = np.stack([starts[seq], n[seq], first, solo[seq]], axis=1).astype(np.int32)
            walkers = np.where(solo[seq] | (len(lists) == 0), 1, 4)          # waves that share an item's walk
            orders = [np.argsort(-(work / walkers), kind="stable")
                      for work in (np.minimum(first + grain[seq], n[seq]), n[seq] - first, n[seq])]
            lists += [np.concatenate([items[o], tail]) for o in orders]
            counts.append(len(items) + len(tail))
        self._counts = tuple(counts)
        self._lists, self._stream, self._cuts = None, 0, {}
        if self.device.type == "cuda":
            from .lib import raw_stream
            # a blocking copy: the list is there for whichever stream uses it first
            self._lists = torch.from_numpy(np.concatenate(lists)).to(self.device)
            self._stream = raw_stream(self.device)

    def _cut(self, order: int, lanes: int) -> int:
        """How many of the 128-row key items, longest walk first (``order`` 0 causal, 1 no mask), are worth two workgroups: those that
        alone walk further than a CU's share of all walks over ``lanes`` heads, which the launch would end up waiting for."""
        if (order, lanes) not in self._cuts:
            n = self.lengths[self.lengths > 0]
            parts = -(-n // PACKED_OWN_ROWS)
            seq = np.repeat(np.arange(len(n)), parts)
            first = (np.arange(len(seq)) - np.repeat(np.cumsum(parts) - parts, parts)) * PACKED_OWN_ROWS
            walks = n[seq] - (first if order == 0 else 0)
            self._cuts[order, lanes] = int((walks > walks.sum() * lanes / 256).sum())
        return self._cuts[order, lanes]

    def _items(self, which: int, order: int, stream: int):
        """(address, number) of a list for a launch on ``stream``: ``which`` 0 / 1 / 2 as laid out above, ``order`` 0 causal queries,
        1 causal keys, 2 no mask.  Uniform batches have no list (address 0)."""
        if self._lists is None:
            return 0, self._counts[which]
        if stream != self._stream:       # keeps the allocator from handing the list's memory on too early
            self._lists.record_stream(torch.cuda.current_stream(self.device))
        at = 3 * sum(self._counts[:which]) + order * self._counts[which]
        return self._lists.data_ptr() + at * PACKED_ITEM_BYTES, self._counts[which]


def packed_attention_reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pack: SequencePack, causal: bool = False,
                               scale: Optional[float] = None) -> torch.Tensor:
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    group = int(q.shape[1]) // int(k.shape[1])          # numbers under a tracer too
    out, at = [], 0
    for n in pack.lengths.tolist():
        qs, ks, vs = (t[at:at + n].transpose(0, 1) for t in (q, k, v))
        ks, vs = ks.repeat_interleave(group, 0), vs.repeat_interleave(group, 0)
        s = (qs @ ks.transpose(1, 2)) * scale
        if causal:
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
        out.append((torch.softmax(s, dim=-1) @ vs).transpose(0, 1))
        at += n
    out.append(q.new_zeros(pack.rows - at, q.shape[1], v.shape[-1]))
    return torch.cat(out)


def packed_attention_plain(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pack: SequencePack, causal: bool,
                           scale: float) -> torch.Tensor:
    """The formula in f32, also under autocast, rounded once, for what the kernels do not serve."""
    with torch.autocast(q.device.type, enabled=False):
        return packed_attention_reference(q.float(), k.float(), v.float(), pack, causal, scale).to(q.dtype)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pack: SequencePack, causal: bool = False,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Softmax attention within every sequence of ``pack``: ``q`` [rows, heads, dk], ``k`` [rows, kv_heads, dk], ``v``
    [rows, kv_heads, dv] -> [rows, heads, dv], all f32 or all bf16, differentiable.  Query head ``i`` reads key / value head
    ``i // (heads // kv_heads)``; with ``causal`` a row sees its sequence's rows up to itself.  ``scale`` defaults to
    ``1 / sqrt(dk)``.  Second derivatives, forward-mode differentiation, ``torch.func`` transforms and tracing go through plain
    torch, which holds a sequence's scores in memory.  Rows behind the last sequence give zeros, and nothing of what they hold is used.

    On a GPU: heads of at most 128 elements.  Operands may be strided (a slice of a fused projection is read in place when its
    rows lie on 16-byte boundaries and is copied otherwise).  f32 operands are multiplied exactly; for bf16 the probabilities
    are rounded to bf16 for the second product.  A value that is not finite reaches every row of its own sequence that lies
    within 128 rows of one that may see it, and no other sequence; a row whose scores are all -inf is not a number, as the softmax of
    such a row is."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"{name} must be [rows, heads, width], got {tuple(t.shape)}")
        if t.shape[0] != pack.rows:
            raise ValueError(f"{name} has {t.shape[0]} rows, the pack {pack.rows}")
        if t.dtype != q.dtype or t.device != q.device:
            raise TypeError(f"q, k and v must share one type and device, got {q.dtype} on {q.device} and {t.dtype} on {t.device}")
    heads, kv_heads, dk, dv = q.shape[1], k.shape[1], q.shape[2], v.shape[2]
    if k.shape[2] != dk or v.shape[1] != kv_heads:
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)} and v {tuple(v.shape)}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key / value heads")
    if dk < 1 or dv < 1:
        raise ValueError("heads must have at least one element")
    scale = 1.0 / math.sqrt(dk) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if not q.is_cuda:
        return packed_attention_reference(q, k, v, pack, causal, scale)
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"packed_attention on a GPU takes f32 or bf16 operands, got {q.dtype}")
    if max(dk, dv) > PACKED_MAX_HEAD_DIM:
        raise ValueError(f"packed_attention on a GPU takes heads of at most {PACKED_MAX_HEAD_DIM} elements, got {max(dk, dv)}")
    if pack.device != q.device:
        raise ValueError(f"the pack lies on {pack.device}, the operands on {q.device}")
    if transformed(q, k, v):
        return packed_attention_plain(q, k, v, pack, causal, scale)
    from .attention_hip import PackedAttention, in_place, packed_forward
    from .lib import wants_grad
    q, k, v = in_place(q), in_place(k), in_place(v)
    if wants_grad(q, k, v):
        out = PackedAttention.apply(q, k, v, pack, bool(causal), scale)
    else:
        out = packed_forward(q, k, v, pack, bool(causal), scale, False)[0]
    return out if v.shape[2] == dv else out[..., :dv].contiguous()
