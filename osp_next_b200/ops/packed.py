"""Attention over packed sequences (kernels: ``ops/csrc/packed_attn_fwd.cu``, ``packed_attn_bwd.cu``).

A language model's batch is sequences of different lengths.  :class:`SequencePack` says which rows
belong to which sequence; it is made once for a batch and serves every layer, forward and backward.
:func:`packed_attention` is the forward, ``models.functional.packed_attention`` the form under
autograd.

CPU tensors run the PyTorch reference (:mod:`.reference`); CUDA tensors run the kernels.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import numpy as np
import torch

from . import reference as ref
from ._ext import ext

TILE = 128             # rows of a tensor-core tile: group heads x positions, or keys
_LONG_STEPS = 6        # mean key tiles of an item from which a forward CTA takes two row tiles
_MIN_FWD_STEPS = 4     # key tiles below which splitting an item further costs more than it gives
_MIN_KEY_STEPS = 8     # the same for the row tiles of a key tile's gradient
_SHORT = 32            # longest sequence of a pack whose gradients' kernels multiply dS as two bf16 numbers


def _whole(v, what: str) -> np.ndarray:
    if isinstance(v, torch.Tensor):
        if v.dtype.is_floating_point or v.dtype == torch.bool or v.dim() != 1:
            raise TypeError(f"SequencePack: {what} as whole numbers in one dimension")
        v = v.tolist()
    out = np.asarray(list(v), dtype=object)
    if out.ndim != 1 or any(isinstance(x, (bool, np.bool_)) or not isinstance(x, (int, np.integer)) for x in out):
        raise TypeError(f"SequencePack: {what} as whole numbers in one dimension")
    if any(x < 0 or x >= 1 << 31 for x in out):
        raise ValueError(f"SequencePack: {what} from 0 to 2^31 - 1")
    return out.astype(np.int64)


class SequencePack:
    """Where the sequences of a batch lie in the rows of q [Nq, heads, D] and of k, v [Nk, ...].

    ``lengths``: queries of each sequence (whole numbers; 0 is a sequence without rows).
    ``key_lengths``: its keys, where they are not as many; its queries are then its last tokens.
    ``starts`` / ``key_starts``: first row of each sequence; without them one lies behind another.
    Sequences must not overlap.  Rows of no sequence are zeros in results.

    Work lists for the kernels are laid out on the device at the first call with each kind (forward,
    backward, number of heads), which waits for their upload, and kept here: make that call before
    capturing a graph, and keep the pack as long as the graph."""

    def __init__(self, lengths: Sequence[int], key_lengths: Optional[Sequence[int]] = None,
                 starts: Optional[Sequence[int]] = None, key_starts: Optional[Sequence[int]] = None, device="cuda"):
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.lengths = _whole(lengths, "lengths")
        self.starts, self.rows, self.dense = self._place(self.lengths, starts, "starts")
        if key_lengths is None:
            if key_starts is not None:
                raise ValueError("SequencePack: key_starts without key_lengths")
            self.key_lengths, self.key_starts, self.key_rows, self.key_dense = (
                self.lengths, self.starts, self.rows, self.dense)
        else:
            self.key_lengths = _whole(key_lengths, "key_lengths")
            if len(self.key_lengths) != len(self.lengths):
                raise ValueError(f"SequencePack: {len(self.lengths)} lengths, {len(self.key_lengths)} key_lengths")
            self.key_starts, self.key_rows, self.key_dense = self._place(self.key_lengths, key_starts, "key_starts")
        self.longest = int(max(self.lengths.max(initial=0), self.key_lengths.max(initial=0)))
        self._lists = {}

    @classmethod
    def padded(cls, lengths: Sequence[int], row_length: int, device="cuda") -> "SequencePack":
        """Sequences at the start of each row of a padded batch [len(lengths), row_length]."""
        n = _whole(lengths, "lengths")
        if len(n) and n.max() > row_length:
            raise ValueError(f"SequencePack: a length of {n.max()} in rows of {row_length}")
        return cls(n, starts=np.arange(len(n)) * row_length, device=device)

    @staticmethod
    def _place(lengths, starts, what):
        """(first rows, rows needed, whether every one of them belongs to a sequence)."""
        if starts is None:
            ends = np.cumsum(lengths)
            starts, rows, dense = ends - lengths, int(ends[-1]) if len(ends) else 0, True
        else:
            starts = _whole(starts, what)
            if len(starts) != len(lengths):
                raise ValueError(f"SequencePack: {len(lengths)} lengths, {len(starts)} {what}")
            used = lengths > 0
            order = np.argsort(starts[used], kind="stable")
            s, n = starts[used][order], lengths[used][order]
            if np.any(s[1:] < s[:-1] + n[:-1]):
                raise ValueError("SequencePack: sequences overlap")
            rows = int((s + n).max(initial=0))
            dense = rows == int(n.sum())
        if rows >= 1 << 31:
            raise ValueError("SequencePack: more than 2^31 - 1 rows")
        return starts, rows, dense

    def __len__(self):
        return len(self.lengths)

    def __repr__(self):
        return (f"SequencePack({len(self)} sequences, {int(self.lengths.sum())} queries, "
                f"{int(self.key_lengths.sum())} keys, {self.device})")

    # ------------------------------------------------------------------ work lists

    def _upload(self, *arrays):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("SequencePack: its first call of a kind lays out work lists; make it before capturing")
        with torch.cuda.device(self.device):
            out = [torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(self.device) for a in arrays]
            torch.cuda.current_stream().synchronize()      # seen by every stream from here on
        return out

    def _sms(self):
        return torch.cuda.get_device_properties(self.device).multi_processor_count

    def forward_lists(self, group: int, heads: int, causal: bool):
        """(items, joins, slots, positions per row tile, row tiles per CTA, heads run together) of the
        forward kernel for ``heads`` groups of ``group`` query heads; lists on the device."""
        key = ("fwd", group, heads, causal)
        hit = self._lists.get(key)
        if hit is None:
            tiles = row_tiles(self, group, causal)
            (items, joins), slots = forward_items(self, group, heads, causal, self._sms(), tiles)
            together = heads_together(items[:, 6] - items[:, 5], heads, self._sms() * (2 if tiles == 1 else 1))
            hit = self._lists[key] = (*self._upload(items, joins), slots, positions(self, group), tiles, together)
        return hit

    def backward_lists(self, group: int, kv_heads: int, causal: bool):
        """(rows, keys, joins, slots, heads run together in dQ, and in dK, dV) of the backward kernels;
        lists on the device."""
        key = ("bwd", group, kv_heads, causal)
        hit = self._lists.get(key)
        if hit is None:
            keys, joins, slots = key_items(self, group, kv_heads, causal, self._sms())
            rows = row_items(self, group, causal)
            hit = self._lists[key] = (*self._upload(rows, keys, joins), slots,
                                      heads_together(rows[:, 6], kv_heads, self._sms()),
                                      heads_together(-(-keys[:, 4] // (TILE // group)), kv_heads, self._sms()))
        return hit


def _tiles(n):
    return -(-n // TILE)


def positions(pack, group):
    """Positions of a forward row tile: as many as its 128 rows take, no more than any sequence has."""
    return max(1, min(TILE // group, int(pack.lengths.max(initial=0))))


def row_tiles(pack, group, causal):
    """Row tiles of a forward CTA: two share the key tiles that they read, one leaves room for a second
    CTA on the SM, which covers the latency of short passes and of tiles of few rows (one token each over
    up to 8192 keys: 127 us in ones, 155 in twos; 8 prompts of 512 tokens 46 and 48; one of 8192: 555
    and 474).  Sequences that fit one tile have no use for two."""
    per = positions(pack, group)
    if pack.lengths.max(initial=0) <= per:
        return 1
    _, steps = _row_items(pack, group, causal, 2 * per)
    return 1 if steps.mean() < _LONG_STEPS else 2


def _row_items(pack, group, causal, per):
    """Items of ``per`` queries each, without splits: int64 [n, 8] and their key tiles."""
    count = -(-pack.lengths // per)
    seq = np.repeat(np.arange(len(pack)), count)
    first = (np.arange(len(seq)) - np.repeat(np.cumsum(count) - count, count)) * per
    lq, lk = pack.lengths[seq], pack.key_lengths[seq]
    n_q = np.minimum(per, lq - first)
    limit = first + 1 + lk - lq
    seen = np.clip(np.minimum(lk, limit + n_q - 1), 0, None) if causal else lk
    steps = _tiles(seen)
    items = np.stack([pack.starts[seq] + first, n_q, limit, pack.key_starts[seq], lk, np.zeros_like(lk), steps,
                      np.full_like(lk, -1)], 1).reshape(-1, 8)
    return items, steps


def _longest_first(items, steps):
    return items[np.argsort(-steps, kind="stable")]


def row_items(pack, group, causal):
    """Items of the dQ kernel: one row tile each, over the keys that its last query sees."""
    return _longest_first(*_row_items(pack, group, causal, TILE // group))


def _split(steps, kv_heads, sms, least):
    """Parts of each item: an item longer than an even share of all work per SM is split, into parts
    of no fewer than ``least`` steps."""
    share = max(least, -(-int(steps.sum()) * kv_heads // sms))
    return np.maximum(1, -(-steps // share))


def heads_together(steps, heads, slots):
    """Heads whose items run side by side, longest first: as few as fill the ``slots`` CTAs that run at
    a time, so that these share keys in L2 (gradients over 16 heads of 8192 keys: dK and dV 904 us six
    at a time, 943 all together), but enough for the last ones to take twice their longest item."""
    total = int(steps.sum())
    if not total:
        return heads
    least = max(-(-slots // len(steps)), -(-2 * int(steps.max()) * slots // total))
    return -(-heads // max(1, heads // least))


def forward_items(pack, group, kv_heads, causal, sms, tiles):
    """((items, joins), slots) of the forward kernel: ``tiles`` row tiles each, longest first; items
    with many keys are split, and joined in the order of their parts."""
    items, steps = _row_items(pack, group, causal, tiles * positions(pack, group))
    parts = _split(steps, kv_heads, sms * (2 if tiles == 1 else 1), _MIN_FWD_STEPS)
    size = -(-steps // parts)
    parts = np.maximum(1, -(-steps // np.maximum(size, 1)))         # no empty part
    cut = parts > 1
    slot0 = np.cumsum(np.where(cut, parts, 0)) - np.where(cut, parts, 0)
    joins = np.stack([items[cut, 0], items[cut, 1], slot0[cut], parts[cut]], 1).reshape(-1, 4)
    at = np.repeat(np.arange(len(items)), parts)
    part = np.arange(len(at)) - np.repeat(np.cumsum(parts) - parts, parts)
    out = items[at]
    out[:, 5] = part * size[at]
    out[:, 6] = np.minimum(steps[at], (part + 1) * size[at])
    out[:, 7] = np.where(cut[at], slot0[at] + part, -1)
    return (_longest_first(out, out[:, 6] - out[:, 5]), joins), int(parts[cut].sum())


def key_items(pack, group, kv_heads, causal, sms):
    """(items, joins, slots) of the dK, dV kernel: one tile of 128 keys each, over the row tiles from
    the first query that sees it on."""
    per = TILE // group
    count = _tiles(pack.key_lengths)
    seq = np.repeat(np.arange(len(pack)), count)
    key0 = (np.arange(len(seq)) - np.repeat(np.cumsum(count) - count, count)) * TILE
    lq, lk = pack.lengths[seq], pack.key_lengths[seq]
    sees = key0 - (lk - lq)                                         # position of the query that stands at key0
    first = np.clip(sees, 0, lq) if causal else np.zeros_like(lq)
    steps = -(-(lq - first) // per)
    parts = _split(steps, kv_heads, sms, _MIN_KEY_STEPS)
    size = -(-steps // parts)
    parts = np.maximum(1, -(-steps // np.maximum(size, 1)))
    cut = parts > 1
    slot0 = np.cumsum(np.where(cut, parts, 0)) - np.where(cut, parts, 0)
    k_row, n_k = pack.key_starts[seq] + key0, np.minimum(TILE, lk - key0)
    joins = np.stack([k_row[cut], n_k[cut], slot0[cut], parts[cut]], 1).reshape(-1, 4)
    at = np.repeat(np.arange(len(seq)), parts)
    part = np.arange(len(at)) - np.repeat(np.cumsum(parts) - parts, parts)
    begin = first[at] + part * size[at] * per
    n_q = np.where(cut[at], np.minimum(lq[at] - begin, size[at] * per), lq[at] - begin)
    out = np.stack([k_row[at], n_k[at], begin, pack.starts[seq][at] + begin, n_q, sees[at] - begin,
                    np.where(cut[at], slot0[at] + part, -1), lk[at]], 1).reshape(-1, 8)
    return _longest_first(out, -(-n_q // per)), joins, int(parts[cut].sum())


# ---------------------------------------------------------------------------- calls

def check_packed(q, k, v, pack, rel_bias=None, what="packed_attention", scale=None):
    """Raise for operands that do not fit each other or the pack."""
    if scale is not None and not abs(float(scale)) < 1e38:         # in fp32, times log2 e
        raise ValueError(f"{what}: a finite scale, got {scale}")
    if not isinstance(pack, SequencePack):
        raise TypeError(f"{what}: pack has to be a SequencePack")
    for n, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"{what}: {n} [tokens, heads, head_dim], got {tuple(t.shape)}")
        if t.device != q.device or t.dtype != q.dtype:
            raise TypeError(f"{what}: q, k and v of one type on one device")
    if q.device.type != pack.device.type or (q.is_cuda and q.device != pack.device):
        raise ValueError(f"{what}: tensors on {q.device}, pack on {pack.device}")
    if not q.dtype.is_floating_point:
        raise TypeError(f"{what}: floating-point q, k and v, got {q.dtype}")
    Hq, D = q.shape[1:]
    if k.shape != v.shape or k.shape[2] != D:
        raise ValueError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} against q {tuple(q.shape)}")
    Hkv = k.shape[1]
    if Hkv == 0 or Hq % Hkv or not 1 <= Hq // Hkv <= TILE:
        raise ValueError(f"{what}: {Hq} query heads against {Hkv} key heads (a multiple of them, at most {TILE} to one)")
    if D == 0 or D % 8 or D > 128:
        raise ValueError(f"{what}: head_dim a multiple of 8 up to 128, got {D}")
    if q.shape[0] < pack.rows or k.shape[0] < pack.key_rows:
        raise ValueError(f"{what}: the pack needs {pack.rows} query and {pack.key_rows} key rows, "
                         f"got {q.shape[0]} and {k.shape[0]}")
    if rel_bias is not None:
        if rel_bias.dim() != 2 or rel_bias.shape[0] != Hq or rel_bias.shape[1] % 2 == 0:
            raise ValueError(f"{what}: rel_bias [{Hq}, 2 M - 1], got {tuple(rel_bias.shape)}")
        if rel_bias.shape[1] < 2 * pack.longest - 1:
            raise ValueError(f"{what}: rel_bias reaches {(rel_bias.shape[1] + 1) // 2} positions, the longest "
                             f"sequence has {pack.longest}")
        if rel_bias.device != q.device:
            raise TypeError(f"{what}: rel_bias on {rel_bias.device}, q on {q.device}")


def packed_attention(q, k, v, pack: SequencePack, causal: bool = True, scale: Optional[float] = None, rel_bias=None,
                     return_lse: bool = False):
    """softmax(scale q k^T + bias) v inside each sequence of ``pack``: o [Nq, heads, D] like q
    (+ log-sum-exp [Nq, heads] fp32, natural log).

    q [Nq, heads, D], k and v [Nk, key heads, D] (bf16 on the GPU; rows of any stride, views of a
    fused projection among them).  Heads h G .. (h + 1) G - 1 of q read key head h, G = heads / key
    heads.  D: multiples of 8 up to 128.  ``scale``: any finite number (1 / sqrt(D) without one).  Query i of
    a sequence with lq queries and lk keys stands at position i + lk - lq; ``causal`` queries see the keys up
    to their position.  ``rel_bias`` fp32
    [heads, 2 M - 1] adds ``rel_bias[h, key position - query position + M - 1]``, finite values; on the GPU
    those beyond +-6.9e37 count as that, so that the type's lowest value hides a key.
    A query that sees no key gives zeros and a log-sum-exp of -inf; so do rows of no sequence.
    Values of other sequences never reach a sequence's rows; a NaN or infinity in v reaches every
    query of its own sequence whose tile of keys it lies in, those that a causal mask hides it from
    among them.

    It records no graph: ``models.functional.packed_attention`` is the form under autograd."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (rel_bias is not None and rel_bias.requires_grad)):
        check_packed(q, k, v, pack, rel_bias, scale=scale)
        raise RuntimeError("packed_attention has no gradient: use models.functional.packed_attention, or "
                           "torch.no_grad()")
    if not q.is_cuda:
        check_packed(q, k, v, pack, rel_bias, scale=scale)
        scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
        o, lse = ref.packed_attention(q, k, v, pack, causal, scale, rel_bias)
        return (o, lse) if return_lse else o
    o, lse, _ = _forward(q, k, v, pack, causal, scale, rel_bias, bool(return_lse), False)
    return (o, lse) if return_lse else o


def _forward(q, k, v, pack, causal, scale, rel_bias, want_lse, want_low):
    """(o, log-sum-exp, what o's rounding left) on the GPU; the last two None where not asked for."""
    try:
        # the kernel's own checks come first: a call of a few microseconds has no time for both
        Hkv = k.shape[1]
        group = 1 if rel_bias is not None else q.shape[1] // Hkv  # heads of a row tile (one with a bias)
        items, joins, slots, per, tiles, together = pack.forward_lists(group, q.shape[1] // group, bool(causal))
        return ext().packed_attn_fwd(q, k, v, items, joins, slots, per, tiles, together, bool(causal),
                                     -1.0 if scale is None else float(scale), scale is None, rel_bias, want_lse,
                                     want_low, pack.rows, pack.key_rows, pack.longest, pack.dense)
    except (AttributeError, IndexError, RuntimeError, TypeError, ValueError, ZeroDivisionError):
        check_packed(q, k, v, pack, rel_bias, scale=scale)
        if q.dtype != torch.bfloat16:
            raise TypeError(f"packed_attention: bf16 on the GPU, got {q.dtype}") from None
        raise


def packed_attention_for_grad(q, k, v, pack: SequencePack, causal: bool = True, scale: Optional[float] = None):
    """(o, log-sum-exp, remainder) for :func:`packed_attention_bwd` on the GPU: the remainder, a byte per
    value, is what the rounding of o to bf16 left."""
    return _forward(q, k, v, pack, causal, scale, None, True, True)


def packed_attention_bwd(q, k, v, o, dout, lse, pack: SequencePack, causal: bool = True, scale: Optional[float] = None,
                         remainder=None):
    """Gradients (dq, dk, dv) of :func:`packed_attention` without a bias, from its output and
    log-sum-exp (and the remainder of :func:`packed_attention_for_grad`); rows of no sequence get zeros."""
    if not q.is_cuda:
        check_packed(q, k, v, pack, what="packed_attention_bwd", scale=scale)
        return ref.packed_attention_bwd(q, k, v, dout, pack, causal,
                                        1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale))
    try:
        Hkv = k.shape[1]
        rows, keys, joins, slots, row_heads, key_heads = pack.backward_lists(q.shape[1] // Hkv, Hkv, bool(causal))
        fill = not (pack.dense and pack.key_dense and q.shape[0] == pack.rows and k.shape[0] == pack.key_rows)
        if q.shape[0] < pack.rows or k.shape[0] < pack.key_rows:
            raise ValueError("packed_attention_bwd: fewer rows than the pack's")
        return ext().packed_attn_bwd(q, k, v, o, dout, lse, remainder, rows, keys, joins, slots, row_heads, key_heads,
                                     bool(causal), 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale), fill,
                                     pack.longest <= _SHORT)
    except (AttributeError, IndexError, RuntimeError, TypeError, ValueError, ZeroDivisionError):
        check_packed(q, k, v, pack, what="packed_attention_bwd", scale=scale)
        if q.dtype != torch.bfloat16:
            raise TypeError(f"packed_attention_bwd: bf16 on the GPU, got {q.dtype}") from None
        raise
