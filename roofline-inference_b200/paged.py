"""Paged KV cache: rotary positions with the append to pages, attention of one new token per sequence
over pages, and eviction of the rows that gathered the least attention.

The reference keeps one contiguous cache per request (agent-test/v2/engine.py:33-55) and rotates one
way only (kernels.py:136-143); here a sequence is a list of pages, so it grows page by page, shrinks,
and may share pages with others, and the rotation, the value type, the head size and the number of
query heads per KV head are the caller's.

  pages  [num_pages, 2, nkv, page_rows, head_dim] BF16 or FP16 (K, then V); any strides that are
         multiples of 8 values with the last dimension contiguous, e.g. one layer of a pool
         [num_pages, layers, 2, nkv, page_rows, head_dim]
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

import contextlib
import ctypes
import math

import torch

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # RIB_DTYPE_BF16, RIB_DTYPE_F16
_EPS = 1e-6


class _Cache(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("table", ctypes.c_void_p), ("table_stride", ctypes.c_longlong),
                ("stride_page", ctypes.c_longlong), ("stride_half", ctypes.c_longlong),
                ("stride_head", ctypes.c_longlong), ("stride_row", ctypes.c_longlong)] + \
               [(n, ctypes.c_int) for n in ("dtype", "num_pages", "nkv", "page_rows", "head_dim", "seqs", "width")]


class _Rotary(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("pairs", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("gain", ctypes.c_float)]


# ----------------------------------------------------------------- argument checks
def _require(name, t, device, dtype, dim):
    """A CUDA tensor on `device` of the given dtype and number of dimensions, last one contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"tensors on different devices: {device} vs {t.device}")
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")


def _vector(name, t, device, n):
    _require(name, t, device, torch.int32, 1)
    if t.shape[0] != n:
        raise ValueError(f"{name} must hold {n} numbers, got {t.shape[0]}")
    return t.data_ptr()


def _table_struct(pages, table) -> _Cache:
    if not isinstance(pages, torch.Tensor) or pages.dtype not in _DTYPES:
        raise ValueError("pages must be a bfloat16 or float16 tensor")
    _require("pages", pages, None, pages.dtype, 5)
    shape, stride = pages.shape, pages.stride()
    if shape[1] != 2 or not all(shape):
        raise ValueError(f"pages must be [num_pages, 2, nkv, page_rows, head_dim], got {tuple(shape)}")
    _require("table", table, pages.device, torch.int32, 2)
    return _Cache(pages.data_ptr(), table.data_ptr(), table.stride(0), stride[0], stride[1], stride[2], stride[3],
                  _DTYPES[pages.dtype], shape[0], shape[2], shape[3], shape[4], table.shape[0], table.shape[1])


def _on(device):
    """Makes `device` current for the call where it is not (launches and scratch go there)."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _output(out, shape, like, name="out"):
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _require(name, out, like.device, like.dtype, len(shape))
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(out.shape)}")
    return out


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
    ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 1e-3))) for i in range(r // 2)]
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
        self._struct = _Rotary(self.turns.data_ptr(), rotary_dim // 2, int(self.interleaved), self.gain)

    def _for(self, dim: int, device):
        if dim != self.head_dim:
            raise ValueError(f"heads have {dim} dims, the rotation {self.head_dim}")
        if self.device != device:
            raise ValueError(f"tensors on different devices: {device} vs {self.device}")
        return ctypes.byref(self._struct)


def _heads(name, t, like, tokens=None, heads=None):
    _require(name, t, like.device, like.dtype, 3)
    if (tokens is not None and t.shape[0] != tokens) or (heads is not None and t.shape[1] != heads) \
            or t.shape[2] != like.shape[-1]:
        raise ValueError(f"{name} must be [{tokens}, {heads or 'heads'}, {like.shape[-1]}], got {tuple(t.shape)}")
    return t.data_ptr(), t.stride(0), t.stride(1)


def rotary(x, pos, rot: Rotary, *, out=None):
    """x [tokens, heads, head_dim] rotated, token t to position pos[t] (int32 CUDA [tokens]).

    BF16 or FP16, any strides that are multiples of 8; computed in FP32 and rounded once.  out may be
    x itself."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES:
        raise ValueError("x must be a bfloat16 or float16 tensor")
    _require("x", x, None, x.dtype, 3)
    tokens, heads, dim = x.shape
    dev = x.device
    r = rot._for(dim, dev)
    out = _output(out, x.shape, x)
    p = _vector("pos", pos, dev, tokens)
    if tokens == 0 or heads == 0:
        return out
    with _on(dev):
        st = _lib.load().rib_rotary_apply(r, x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0),
                                          out.stride(1), p, tokens, heads, dim, _DTYPES[x.dtype], _stream(dev))
    _lib.check(st, "rotary")
    return out


def paged_append(q, k, v, pos, row, pages, table, rot: Rotary, *, seq=None, qw=None, kw=None, eps: float = _EPS,
                 out=None):
    """Rotates q and k to their positions and writes k and v to their rows of the cache; returns q.

    q [T, nq, D], k and v [T, nkv, D] (e.g. views of one projection's output); pos, row, seq int32
    CUDA [T]: token t turns to position pos[t] and goes to row row[t] of sequence seq[t] (sequence t
    without seq: one token per sequence).  A row is not a position: after an eviction they differ.
    qw, kw [D]: RMS-normalise each q and k head first (both or neither).  A negative row marks a
    padding token: q is rotated, the cache is left alone.  The (seq, row) pairs of a call must differ.
    out may be q itself."""
    cache = _table_struct(pages, table)
    D, dev = cache.head_dim, pages.device
    like = pages
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [tokens, nq, head_dim]")
    T, nq = q.shape[0], q.shape[1]
    qp, kp, vp = _heads("q", q, like, T, nq), _heads("k", k, like, T, cache.nkv), _heads("v", v, like, T, cache.nkv)
    r = rot._for(D, dev)
    if (qw is None) != (kw is None):
        raise ValueError("qw and kw come together")
    if qw is not None:
        for name, w in (("qw", qw), ("kw", kw)):
            _require(name, w, dev, like.dtype, 1)
            if w.shape[0] != D:
                raise ValueError(f"{name} must hold {D} values")
    if seq is None and T > cache.seqs:
        raise ValueError(f"{T} tokens for {cache.seqs} sequences: seq says where each belongs")
    out = _output(out, q.shape, q)
    pos_p, row_p = _vector("pos", pos, dev, T), _vector("row", row, dev, T)
    seq_p = None if seq is None else _vector("seq", seq, dev, T)
    if T == 0:
        return out
    with _on(dev):
        st = _lib.load().rib_paged_append(
            ctypes.byref(cache), r, *qp, *kp, *vp, out.data_ptr(), out.stride(0), out.stride(1), pos_p, row_p, seq_p,
            T, nq, None if qw is None else qw.data_ptr(), None if kw is None else kw.data_ptr(), eps, _stream(dev))
    _lib.check(st, "paged_append")
    return out


# ----------------------------------------------------------------- attention
def _scores(name, t, device, batch, nkv, least):
    _require(name, t, device, torch.float32, 3)
    if t.shape[0] != batch or t.shape[1] != nkv or t.shape[2] < least:
        raise ValueError(f"{name} must be [{batch}, {nkv}, >= {least}], got {tuple(t.shape)}")


def paged_decode_attention(q, pages, table, lens, scale: float, *, max_len: int | None = None, scores=None,
                           scores_out=None, out=None):
    """Attention of one new token per sequence over its lens[b] rows; returns [B, nq, D].

    q [B, nq, D]; nq any multiple of nkv; D 64 or 128; page_rows a multiple of 16; lens int32 CUDA [B]
    (0: the output row is zeros).  max_len: host bound on lens (what the table holds by default); it
    sizes nothing but the scores' scratch.  scores [B, nkv, >= max_len] FP32: the softmax weight of
    each row, summed over the query heads of its KV head, is added to it, in place or into scores_out;
    entries behind lens[b] stay as they are.  Weights and sums are FP32; the result is rounded once."""
    cache = _table_struct(pages, table)
    dev = pages.device
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [B, nq, head_dim]")
    B, nq = q.shape[0], q.shape[1]
    qp, qs, qh = _heads("q", q, pages, B, nq)
    if cache.head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {cache.head_dim}")
    if cache.page_rows % 16:
        raise ValueError(f"page_rows must be a multiple of 16, got {cache.page_rows}")
    if not 0 < B <= cache.seqs:
        raise ValueError(f"{B} queries for {cache.seqs} sequences")
    if nq % cache.nkv or not nq:
        raise ValueError(f"nq ({nq}) must be a multiple of nkv ({cache.nkv})")
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    room = cache.width * cache.page_rows
    max_len = room if max_len is None else int(max_len)
    if not 1 <= max_len <= room:
        raise ValueError("KV capacity exceeded")
    lens_p = _vector("lens", lens, dev, B)
    sp, ss, sh, op, os_, oh = None, 0, 0, None, 0, 0
    if scores is not None:
        _scores("scores", scores, dev, B, cache.nkv, max_len)
        scores_out = scores if scores_out is None else scores_out
        _scores("scores_out", scores_out, dev, B, cache.nkv, max_len)
        sp, ss, sh = scores.data_ptr(), scores.stride(0), scores.stride(1)
        op, os_, oh = scores_out.data_ptr(), scores_out.stride(0), scores_out.stride(1)
    elif scores_out is not None:
        raise ValueError("scores_out needs scores")
    out = _output(out, q.shape, q)
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    L = _lib.load()
    with _on(dev):
        nbytes = L.rib_paged_decode_workspace_bytes(B, max_len, nq, cache.head_dim, int(sp is not None))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        st = L.rib_paged_decode_attention(ctypes.byref(cache), qp, qs, qh, lens_p, B, nq, max_len, scale,
                                          out.data_ptr(), sp, ss, sh, op, os_, oh, ws.data_ptr(), nbytes, _stream(dev))
    _lib.check(st, "paged_decode_attention")
    return out


# ----------------------------------------------------------------- eviction
def _overlap(a, b) -> bool:
    """Whether the address ranges that two tensors span meet."""
    def span(t):
        lo = t.data_ptr()
        return lo, lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


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
    with: a row number is not one any more."""
    cache = _table_struct(pages, table)
    dev = pages.device
    if cache.head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {cache.head_dim}")
    if not isinstance(lens, torch.Tensor) or lens.dim() != 1:
        raise ValueError("lens must be [B]")
    B = lens.shape[0]
    if not 0 < B <= cache.seqs:
        raise ValueError(f"{B} lengths for {cache.seqs} sequences")
    lens_p = _vector("lens", lens, dev, B)
    room = cache.width * cache.page_rows
    max_len = room if max_len is None else int(max_len)
    if not 1 <= max_len <= room:
        raise ValueError("KV capacity exceeded")
    _scores("scores", scores, dev, B, cache.nkv, max_len)
    _require("new_table", new_table, dev, torch.int32, 2)
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError("need keep >= 1, sinks >= 0, recent >= 0 and sinks + recent <= keep")
    if new_table.shape[0] < B or new_table.shape[1] * cache.page_rows < keep:
        raise ValueError(f"new_table must name pages for {keep} rows of {B} sequences, got {tuple(new_table.shape)}")
    np_, ns, nh, nw = None, 0, 0, 0
    if new_scores is not None:
        _scores("new_scores", new_scores, dev, B, cache.nkv, keep)
        if _overlap(scores, new_scores):
            raise ValueError("new_scores must not overlap scores")
        np_, ns, nh, nw = new_scores.data_ptr(), new_scores.stride(0), new_scores.stride(1), new_scores.shape[2]
    rows = torch.empty((B, cache.nkv, keep), dtype=torch.int32, device=dev)
    new_lens = torch.empty(B, dtype=torch.int32, device=dev)
    with _on(dev):
        st = _lib.load().rib_paged_evict(ctypes.byref(cache), new_table.data_ptr(), new_table.stride(0),
                                         new_table.shape[1], lens_p, B, max_len, scores.data_ptr(), scores.stride(0),
                                         scores.stride(1), keep, sinks, recent, rows.data_ptr(), new_lens.data_ptr(),
                                         np_, ns, nh, nw, _stream(dev))
    _lib.check(st, "paged_evict")
    return rows, new_lens
