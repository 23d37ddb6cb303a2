"""Paged KV cache: rotary positions with the append to pages, attention of one new token per sequence
over pages, and eviction of the rows that gathered the least attention.

The reference keeps one contiguous cache per request (agent-test/v2/engine.py:33-55) and rotates one
way only (kernels.py:136-143); here a sequence is a list of pages, so it grows page by page, shrinks,
and may share pages with others, and the rotation, the value type, the head size and the number of
query heads per KV head are the caller's.

  pages  [num_pages, 2, nkv, page_rows, head_dim] BF16 or FP16 (K, then V); any strides that are
         multiples of 8 values with the last dimension contiguous, e.g. one layer of a pool
         [num_pages, layers, 2, nkv, page_rows, head_dim], in any order in memory.  head_dim is a
         multiple of 16 from 32 to 256 for the append, 64 or 128 for attention and eviction
  table  [sequences, width] int32: the pages of each sequence in order (row r in page
         table[s, r // page_rows]); entries behind a sequence's rows are never read

  Rotary(head_dim, base, ...)                       a rotation: layout, part of the head, scaling
  rotary(x, pos, rot)                               rotate heads, without a cache
  paged_append(q, k, v, pos, row, pages, table, rot)    rotate q and k, write k and v to their rows
  paged_decode_attention(q, pages, table, lens, scale)  one new token per sequence
  paged_evict(pages, table, lens, scores, keep, new_table)   keep the best rows, in new pages

Every call runs on torch's current stream of the tensors' device, takes scratch from torch's allocator
for the call alone, never synchronises, and can be captured in a CUDA graph.  What only the device can
see (a length or row beyond the table, a page number outside the pool) is never read or written
through and is reported by _lib.take_device_status().
"""
from __future__ import annotations

import math

import torch

from . import _lib


# ----------------------------------------------------------------- rotary positions
def rotary_frequencies(rotary_dim: int, base: float, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, fast_turns: float = 32.0, slow_turns: float = 1.0):
    """(radians per position of each of the rotary_dim / 2 pairs as a list of floats, gain).

    Pair i turns by base^(-2 i / rotary_dim) a position.  For contexts `factor` times the trained
    original_length:
      "linear"  every pair `factor` times slower
      "ntk"     base times factor^(r / (r - 2)): the slowest pair is `factor` times slower, the
                fastest as before
      "yarn"    pairs that turn less than slow_turns times over original_length are `factor` times
                slower, those that turn more than fast_turns times as before, a ramp between; cosines
                and sines times 1 + ln(factor) / 10"""
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if not math.isfinite(base) or base <= 1.0:
        raise ValueError("base must be finite and greater than 1")
    if not math.isfinite(factor) or factor < 1.0 or (scaling is None and factor != 1.0):
        raise ValueError("factor must be finite and at least 1, and 1 without scaling")
    r = rotary_dim
    if scaling == "ntk":
        base = base * factor ** (r / (r - 2))
    freq = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    if scaling != "yarn":
        return freq, 1.0
    if not original_length or original_length < 1 or not 0 < slow_turns < fast_turns:
        raise ValueError("yarn needs original_length >= 1 and 0 < slow_turns < fast_turns")
    # the pair that turns t times over original_length
    pair = [r * math.log(original_length / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast_turns, slow_turns)]
    low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), r - 1)
    # (high <= 0: even pair 0 turns less than slow_turns times)
    ramp = [1.0 if high <= 0 else min(1.0, max(0.0, (i - low) / max(high - low, 1e-3))) for i in range(r // 2)]
    return [f * (1 - s) + f / factor * s for f, s in zip(freq, ramp)], 1.0 + 0.1 * math.log(factor)


class Rotary:
    """A rotation of heads by position, made once and used by every call.

    head_dim: a multiple of 16, 32 to 256.  rotary_dim: how much of a head turns (a multiple of 16;
    the whole head by default); the rest passes unchanged.  interleaved: pairs are dims (2i, 2i + 1)
    instead of (i, i + rotary_dim / 2).  scaling, factor, original_length, fast_turns, slow_turns: as
    rotary_frequencies.  The per-pair speeds live on `device` in FP64, so angles of far positions keep
    their precision."""

    def __init__(self, head_dim: int, base: float = 1e6, *, rotary_dim: int | None = None, interleaved: bool = False,
                 scaling: str | None = None, factor: float = 1.0, original_length: int | None = None,
                 fast_turns: float = 32.0, slow_turns: float = 1.0, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim % 16 or not 32 <= head_dim <= 256:
            raise ValueError("head_dim must be a multiple of 16 from 32 to 256")
        if rotary_dim % 16 or not 16 <= rotary_dim <= head_dim:
            raise ValueError("rotary_dim must be a multiple of 16 from 16 to head_dim")
        freq, self.gain = rotary_frequencies(rotary_dim, float(base), scaling, float(factor), original_length,
                                             fast_turns, slow_turns)
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, bool(interleaved)
        self.frequencies = freq
        self.turns = torch.tensor([f / (2 * math.pi) for f in freq], dtype=torch.float64).to(device)
        self.device = self.turns.device
        self._handle = (self.turns, head_dim, rotary_dim // 2, int(self.interleaved), self.gain)


def _handle(rot):
    if not isinstance(rot, Rotary):
        raise ValueError("rot must be a Rotary")
    return rot._handle


def rotary(x, pos, rot: Rotary, *, out=None):
    """x [tokens, heads, head_dim] rotated, token t to position pos[t] (int32 CUDA [tokens]).

    BF16 or FP16, any strides that are multiples of 8; computed in FP32 and rounded once.  out may be
    x itself."""
    return _lib.binding().rotary(x, pos, _handle(rot), out)


def paged_append(q, k, v, pos, row, pages, table, rot: Rotary, *, seq=None, qw=None, kw=None, eps: float = 1e-6,
                 out=None):
    """Rotates q and k to their positions and writes k and v to their rows of the cache; returns q.

    q [T, nq, D], k and v [T, nkv, D] (e.g. views of one projection's output); pos, row, seq int32
    CUDA [T]: token t turns to position pos[t] and goes to row row[t] of sequence seq[t] (sequence t
    without seq: one token per sequence).  A row is not a position: after an eviction they differ.
    qw, kw [D]: RMS-normalise each q and k head first (both or neither).  A negative row marks a
    padding token: q is rotated, the cache is left alone.  The (seq, row) pairs of a call must differ.
    out may be q itself."""
    return _lib.binding().paged_append(q, k, v, pos, row, pages, table, _handle(rot), seq, qw, kw, eps, out)


# ----------------------------------------------------------------- attention
def paged_decode_attention(q, pages, table, lens, scale: float, *, max_len: int | None = None, scores=None,
                           scores_out=None, out=None):
    """Attention of one new token per sequence over its lens[b] rows; returns [B, nq, D].

    q [B, nq, D]; nq any multiple of nkv; D 64 or 128; page_rows a multiple of 16; lens int32 CUDA [B]
    (0: the output row is zeros, as where every score is -infinity).  max_len: host bound on lens (what
    the table holds by default); a longer length is cut to it and reported.  It sizes the launch and, with
    scores, the scratch (4 B * nq * max_len bytes), and with it at most 256 rows are attended in one launch
    instead of two: worth giving for short sequences in a wide table.  The order of the sums, and so the
    last bits, may differ with it.  scores [B, nkv, >= max_len] FP32: the softmax weight of
    each row, summed over the query heads of its KV head, is added to it, in place or into scores_out
    (scores itself, or a buffer that does not overlap it); entries behind lens[b] stay as they are.
    Infinite V values give infinities, NaN where both signs meet, NaN gives NaN: every row's weight counts
    as positive, however small.
    Scores, weights and all sums are FP32; a weight enters its product with V in two parts of the pages'
    type (16 bits for BF16, 22 for FP16), and the result is rounded once."""
    return _lib.binding().paged_decode_attention(q, pages, table, lens, scale, max_len, scores, scores_out, out)


# ----------------------------------------------------------------- eviction
def paged_evict(pages, table, lens, scores, keep: int, new_table, *, sinks: int = 0, recent: int = 0,
                max_len: int | None = None, new_scores=None):
    """Shortens every sequence to at most `keep` rows; returns (rows, new_lens).

    Each KV head of a sequence longer than `keep` keeps its first `sinks` rows, its last `recent` rows
    and, of those between, the rows with the highest scores [B, nkv, >= max_len] (FP32; equal scores:
    the lower row; NaN lowest).  The kept rows of K and V move, in order, to rows 0, 1, ... of
    new_table's pages: pages of the same tensor that no sequence of `table` uses.  The old pages are
    left as they were.  rows [B, nkv, keep] int32: the old row of each new one, -1 behind the last;
    new_lens [B] int32.  new_scores [B, nkv, >= keep]: receives the kept rows' scores and zeros behind
    them.  Heads of one sequence keep different rows, so positions must be those the keys were rotated
    with: a row number is not one any more.  keep may exceed what any sequence has, up to 0x7f000000."""
    return _lib.binding().paged_evict(pages, table, lens, scores, keep, new_table, sinks, recent, max_len, new_scores)
