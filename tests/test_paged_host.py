"""CPU: what the paged-cache operators refuse on the host (C ABI and Python binding, before any launch),
the rotary frequencies, and the page pool.  No call here reaches a kernel launch."""
from __future__ import annotations

import ctypes
import importlib
import math

import pytest
import torch

from conftest import ROOT  # noqa: F401  (puts the repository on sys.path)

FAKE, MISALIGNED = 0x10000, 0x10008  # never dereferenced
OK, EINVAL, ECAPACITY, EALIGN = 0, 1, 2, 3
paged = importlib.import_module("roofline-inference_b200.paged")


class CacheStruct(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("table", ctypes.c_void_p), ("table_stride", ctypes.c_longlong),
                ("stride_page", ctypes.c_longlong), ("stride_half", ctypes.c_longlong),
                ("stride_head", ctypes.c_longlong), ("stride_row", ctypes.c_longlong)] + \
               [(n, ctypes.c_int) for n in ("dtype", "num_pages", "nkv", "page_rows", "head_dim", "seqs", "width")]


class RotaryStruct(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("pairs", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("gain", ctypes.c_float)]


def cache(**kw):
    c = CacheStruct(FAKE, FAKE, 4, 2 * 2 * 16 * 64, 2 * 16 * 64, 16 * 64, 64, 0, 10, 2, 16, 64, 3, 4)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def rot(**kw):
    r = RotaryStruct(FAKE, 32, 0, 1.0)
    for k, v in kw.items():
        setattr(r, k, v)
    return ctypes.byref(r)


BAD_CACHES = [(dict(pages=None), EINVAL), (dict(table=None), EINVAL), (dict(dtype=2), EINVAL), (dict(num_pages=0), EINVAL),
              (dict(nkv=0), EINVAL), (dict(page_rows=0), EINVAL), (dict(head_dim=24), EINVAL), (dict(head_dim=72), EINVAL),
              (dict(head_dim=272), EINVAL), (dict(seqs=0), EINVAL), (dict(width=0), EINVAL), (dict(stride_row=32), EINVAL),
              (dict(stride_page=-8), EINVAL), (dict(width=0x7f0001, page_rows=256), EINVAL), (dict(pages=MISALIGNED), EALIGN),
              (dict(table=FAKE + 2), EALIGN), (dict(stride_row=68), EALIGN), (dict(stride_head=1028), EALIGN)]


def test_rotary_apply_refuses(rib):
    L = rib.load_library()

    def call(r=None, x=FAKE, xs=(256, 64), out=FAKE, os_=(256, 64), pos=FAKE, tokens=2, heads=4, dim=64, dtype=0):
        return L.rib_rotary_apply(rot() if r is None else r, x, *xs, out, *os_, pos, tokens, heads, dim, dtype, None)
    for kw in (dict(x=None), dict(out=None), dict(pos=None), dict(tokens=-1), dict(heads=0), dict(dim=16), dict(dim=72),
               dict(dim=272), dict(dtype=2), dict(r=rot(turns=None)), dict(r=rot(pairs=0)), dict(r=rot(pairs=12)),
               dict(r=rot(pairs=40)), dict(r=rot(gain=0.0)), dict(r=rot(gain=math.nan))):
        assert call(**kw) == EINVAL, kw
    for kw in (dict(x=MISALIGNED), dict(out=MISALIGNED), dict(pos=FAKE + 1), dict(xs=(256, 60)), dict(os_=(4, 64)),
               dict(r=rot(turns=FAKE + 4))):
        assert call(**kw) == EALIGN, kw
    assert call(tokens=0) == OK  # nothing to do


def test_append_refuses(rib):
    L = rib.load_library()

    def call(c=None, r=None, q=FAKE, k=FAKE, v=FAKE, out=FAKE, pos=FAKE, row=FAKE, seq=None, tokens=3, nq=4, qw=None,
             kw=None, eps=1e-6, strides=(512, 64)):
        return L.rib_paged_append(cache() if c is None else c, rot() if r is None else r, q, *strides, k, 512, 64, v,
                                  512, 64, out, 256, 64, pos, row, seq, tokens, nq, qw, kw, eps, None)
    for kw, status in BAD_CACHES:
        assert call(c=cache(**kw)) == status, kw
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(pos=None), dict(row=None), dict(tokens=-1),
               dict(nq=0), dict(qw=FAKE), dict(kw=FAKE), dict(qw=FAKE, kw=FAKE, eps=-1.0),
               dict(qw=FAKE, kw=FAKE, eps=math.nan), dict(tokens=4), dict(r=rot(pairs=36))):
        assert call(**kw) == EINVAL, kw
    for kw in (dict(q=MISALIGNED), dict(v=MISALIGNED), dict(qw=MISALIGNED, kw=FAKE), dict(seq=FAKE + 1),
               dict(strides=(510, 64))):
        assert call(**kw) == EALIGN, kw
    assert call(tokens=0) == OK


def test_attention_refuses(rib):
    L = rib.load_library()
    ws = L.rib_paged_decode_workspace_bytes(3, 64, 4, 64, 1)
    plain = L.rib_paged_decode_workspace_bytes(3, 64, 4, 64, 0)
    assert 0 < plain < ws
    for bad in [(0, 64, 4, 64, 0), (3, 0, 4, 64, 0), (3, 64, 0, 64, 0), (3, 64, 4, 96, 0)]:
        assert L.rib_paged_decode_workspace_bytes(*bad) == 0

    def call(c=None, q=FAKE, qs=(256, 64), lens=FAKE, batch=3, nq=4, max_len=64, scale=0.125, out=FAKE, scores=FAKE,
             scores_out=FAKE, wsp=FAKE, nbytes=ws):
        return L.rib_paged_decode_attention(cache() if c is None else c, q, *qs, lens, batch, nq, max_len, scale, out,
                                            scores, 128, 64, scores_out, 128, 64, wsp, nbytes, None)
    for kw, status in BAD_CACHES:
        assert call(c=cache(**kw)) == status, kw
    for kw in (dict(q=None), dict(lens=None), dict(out=None), dict(batch=0), dict(batch=4), dict(nq=3), dict(nq=0),
               dict(max_len=0), dict(max_len=65), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf),
               dict(scale=math.nan), dict(scores=None), dict(scores_out=None), dict(wsp=None), dict(nbytes=ws - 1),
               dict(c=cache(head_dim=32, stride_row=32)), dict(c=cache(page_rows=8)), dict(c=cache(page_rows=24))):
        assert call(**kw) == EINVAL, kw
    for kw in (dict(q=MISALIGNED), dict(out=MISALIGNED), dict(wsp=MISALIGNED), dict(lens=FAKE + 2), dict(scores=FAKE + 2),
               dict(qs=(256, 60))):
        assert call(**kw) == EALIGN, kw


def test_evict_refuses(rib):
    L = rib.load_library()

    def call(c=None, table=FAKE, stride=2, width=2, lens=FAKE, batch=3, max_len=64, scores=FAKE, keep=32, sinks=4,
             recent=8, rows=FAKE, new_lens=FAKE, new=FAKE, new_rows=32):
        return L.rib_paged_evict(cache() if c is None else c, table, stride, width, lens, batch, max_len, scores, 128, 64,
                                 keep, sinks, recent, rows, new_lens, new, 64, 32, new_rows, None)
    for kw, status in BAD_CACHES:
        assert call(c=cache(**kw)) == status, kw
    for kw in (dict(table=None), dict(lens=None), dict(scores=None), dict(rows=None), dict(new_lens=None), dict(batch=0),
               dict(batch=4), dict(max_len=0), dict(max_len=65), dict(keep=0), dict(keep=33, new_rows=33), dict(sinks=-1),
               dict(recent=-1), dict(sinks=16, recent=17), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), dict(new_rows=31),
               dict(width=0), dict(stride=-1), dict(c=cache(head_dim=96, stride_row=96))):
        assert call(**kw) == EINVAL, kw
    for kw in (dict(table=FAKE + 2), dict(scores=FAKE + 1), dict(rows=FAKE + 2), dict(new=FAKE + 3)):
        assert call(**kw) == EALIGN, kw


def test_python_entry_points_refuse_host_tensors_and_wrong_handles(rib):
    r = rib.Rotary(64, device="cpu")
    bf = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    pages = torch.zeros((4, 2, 2, 16, 64), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros((2, 2), dtype=torch.int32)
    s = torch.zeros((2, 2, 32))
    with pytest.raises(ValueError, match="CUDA"):
        rib.rotary(bf, i, r)
    with pytest.raises(ValueError, match="CUDA"):
        rib.paged_append(bf, bf, bf, i, i, pages, t, r)
    with pytest.raises(ValueError, match="CUDA"):
        rib.paged_decode_attention(bf, pages, t, i, 0.125)
    with pytest.raises(ValueError, match="CUDA"):
        rib.paged_evict(pages, t, i, s, 8, t)
    with pytest.raises(ValueError, match="Rotary"):
        rib.rotary(bf, i, None)
    with pytest.raises(ValueError, match="torch.Tensor"):
        rib.rotary([1.0], i, r)


# ------------------------------------------------------------------ frequencies
def test_plain_and_linear_frequencies():
    f, gain = paged.rotary_frequencies(128, 1e6)
    assert gain == 1.0 and len(f) == 64
    for i in (0, 1, 17, 63):
        assert f[i] == pytest.approx(math.exp(-2 * i / 128 * math.log(1e6)), rel=1e-14)
    g, gain = paged.rotary_frequencies(128, 1e6, "linear", 4.0)
    assert gain == 1.0 and all(a == b / 4 for a, b in zip(g, f))


def test_ntk_frequencies_keep_the_fastest_and_stretch_the_slowest():
    f, _ = paged.rotary_frequencies(64, 1e4)
    g, gain = paged.rotary_frequencies(64, 1e4, "ntk", 8.0)
    assert gain == 1.0 and g[0] == f[0] == 1.0
    assert g[-1] == pytest.approx(f[-1] / 8, rel=1e-12)
    assert all(a <= b for a, b in zip(g, f))


def test_yarn_frequencies_by_turns():
    """Pairs that turn more than 32 times over the original length are as before, those that turn less
    than once are stretched, between them a ramp."""
    n, factor = 4096, 4.0
    f, _ = paged.rotary_frequencies(128, 1e4)
    g, gain = paged.rotary_frequencies(128, 1e4, "yarn", factor, n)
    assert gain == pytest.approx(1 + 0.1 * math.log(factor), rel=1e-15)
    ratios = [a / b for a, b in zip(g, f)]
    turns = [n * x / (2 * math.pi) for x in f]
    step = turns[0] / turns[1]  # the edges lie on whole pairs: one pair of slack
    assert all(r == pytest.approx(1.0) for r, t in zip(ratios, turns) if t > 32 * step)
    assert all(r == pytest.approx(1 / factor) for r, t in zip(ratios, turns) if t < 1 / step)
    assert all(a >= b - 1e-12 for a, b in zip(ratios, ratios[1:]))
    assert any(0.3 < r < 0.95 for r in ratios)


@pytest.mark.parametrize("kw", [dict(head_dim=24), dict(head_dim=16), dict(head_dim=272), dict(rotary_dim=8),
                                dict(rotary_dim=24), dict(rotary_dim=144), dict(base=1.0), dict(base=math.inf),
                                dict(scaling="dynamic"), dict(factor=2.0), dict(scaling="linear", factor=0.5),
                                dict(scaling="yarn", factor=2.0),
                                dict(scaling="yarn", factor=2.0, original_length=4096, fast_turns=1.0, slow_turns=2.0)])
def test_rotary_refuses(rib, kw):
    with pytest.raises(ValueError):
        rib.Rotary(**{"head_dim": 128, "device": "cpu", **kw})


# ------------------------------------------------------------------ pages
def test_page_pool(rib):
    p = rib.PagePool(2, 1, 5, page_rows=16, head_dim=8, device="cpu")
    assert tuple(p.storage.shape) == (2, 5, 2, 1, 16, 8) and p.layer(1).data_ptr() == p.storage[1].data_ptr()
    assert [p.pages_for(n) for n in (0, 1, 16, 17)] == [0, 1, 1, 2]
    a, b = p.take(2), p.take(2)
    assert not set(a) & set(b) and p.free_pages == 1
    with pytest.raises(rib.PoolFull):
        p.take(2)
    assert p.free_pages == 1
    p.give(a)
    with pytest.raises(ValueError):
        p.give(a)                   # twice
    with pytest.raises(ValueError):
        p.give([b[0], b[0]])
    with pytest.raises(ValueError):
        p.give([99])
    p.give(b)
    assert sorted(p.take(5)) == [0, 1, 2, 3, 4]
    for bad in (dict(pages=0), dict(page_rows=48), dict(n_kv=0)):
        with pytest.raises(ValueError):
            rib.PagePool(**{"n_layers": 1, "n_kv": 1, "pages": 4, "page_rows": 16, "device": "cpu", **bad})
