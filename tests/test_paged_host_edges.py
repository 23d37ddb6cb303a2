"""CPU: paged-cache calls at the edges of what they take, and the page accounting of PagedDecoder.  No call here
reaches a kernel launch."""
from __future__ import annotations

import importlib
import math
from types import SimpleNamespace

import pytest
import torch

from test_paged_host import EINVAL, FAKE, cache

MOST = 0x7f000000


@pytest.mark.parametrize("keep,new_rows", [(MOST + 1, MOST + 1), (2 ** 31 - 1, 2 ** 31 - 1), (32, MOST + 1),
                                           (32, 2 ** 31 - 1)])
def test_evict_refuses_more_rows_than_its_loops_count(rib, keep, new_rows):
    """A thread of the selection writes every 512th to 8192nd of `keep` rows (and of the score rows behind them),
    counting in 32 bits: for a keep within that many of 2^31 the count would wrap and the thread write far below its
    buffer.  Refused before anything is launched."""
    L = rib.load_library()
    status = L.rib_paged_evict(cache(), FAKE, 2, 2, FAKE, 3, 32, FAKE, 128, 64, keep, 4, 8, FAKE, FAKE, FAKE, 64, 32,
                               new_rows, None)
    assert status == EINVAL


def test_attention_refuses_more_tiles_than_a_run_counts(rib):
    """A CTA counts the tiles of its run in 32 bits. Sequences that share their pages (a table stride of 0) can add up
    to more than the 148 x 2 or x 3 CTAs count: the run's length would wrap, and the join would read records that
    nothing wrote."""
    L = rib.load_library()
    many = cache(seqs=1 << 20, nkv=1 << 10, width=MOST // 256, page_rows=256, table_stride=0)
    status = L.rib_paged_decode_attention(many, FAKE, 1 << 16, 64, FAKE, 1 << 20, 1 << 10, MOST, 0.125, FAKE, None, 0, 0,
                                          None, 0, 0, FAKE, 1 << 40, None)
    assert status == EINVAL


def test_attention_refuses_a_scale_beyond_fp32_in_log2_units(rib):
    """scale * log2 e has to be finite in FP32: beyond it a score of 0 would be 0 times infinity."""
    L = rib.load_library()
    ws = L.rib_paged_decode_workspace_bytes(3, 64, 4, 64, 0)
    for scale in (2.4e38, 3.4e38):
        assert L.rib_paged_decode_attention(cache(), FAKE, 256, 64, FAKE, 3, 4, 64, scale, FAKE, None, 0, 0, None, 0, 0,
                                            FAKE, ws, None) == EINVAL


# ------------------------------------------------------------------ PagedDecoder's pages
def decoder(rib, rows, *, pages, max_rows, keep=None, layers=2, page_rows=16):
    """A decoder with one sequence of rows[i] rows in slot i, whose device work is stubbed out by the caller."""
    engine = SimpleNamespace(world=1, cfg=SimpleNamespace(num_layers=layers), device=torch.device("cpu"), n_kv=1,
                             nq_local=2, base=1e6, layers=[{}] * layers)
    pool = rib.PagePool(layers, 1, pages, page_rows, device="cpu")
    d = rib.PagedDecoder(engine, pool, len(rows), max_rows, keep=keep, sinks=0, recent=0)
    for i, n in enumerate(rows):
        ids = pool.take(pool.pages_for(n))
        d.pages[i] = ids
        d.table[i, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        d._set_rows(i, n)
    return d, pool


def pages_of(d):
    return (list(d.rows), [list(p) for p in d.pages], d.row.tolist(), d.lens.tolist(), d.table.tolist(),
            d.pool.free_pages)


@pytest.fixture
def no_eviction(monkeypatch):
    """paged_evict without its device work."""
    module = importlib.import_module("roofline-inference_b200.paged_batch")
    calls = []
    monkeypatch.setattr(module, "paged_evict", lambda *a, **kw: calls.append(a))
    return calls


@pytest.mark.parametrize("rows,pages,max_rows,keep,after", [
    ([64, 16], 6, 64, 16, [2, 2]),           # 1 free: the eviction gives 4 back, then both grow
    ([64, 64, 16], 10, 64, 16, [2, 2, 2]),   # 1 free: the second eviction lives on the first one's pages
    ([64, 48], 9, 64, 20, [2, 4]),           # 2 free, both for the eviction, which leaves room for the other
    ([17, 16], 4, 17, 16, [2, 2]),           # every page in use afterwards
])
def test_eviction_frees_the_pages_that_others_grow_into(rib, no_eviction, rows, pages, max_rows, keep, after):
    d, pool = decoder(rib, rows, pages=pages, max_rows=max_rows, keep=keep)
    d._make_room()
    assert [len(p) for p in d.pages] == after
    assert d.rows == [keep if n == max_rows else n for n in rows]
    used = [p for ids in d.pages for p in ids]
    assert len(set(used)) == len(used) and pool.free_pages == len(pool.layer(0)) - len(used)
    for i, ids in enumerate(d.pages):
        assert d.table[i].tolist() == ids + [-1] * (d.table.shape[1] - len(ids))


@pytest.mark.parametrize("rows,pages,max_rows,keep", [
    ([64, 16], 6, 64, 32),            # an eviction to 2 pages with 1 free
    ([64], 4, 64, 16),                # ... to 1 page with none
    ([17, 16, 16], 5, 17, 16),        # the eviction fits, the three that grow afterwards do not
])
def test_room_that_is_not_there_changes_nothing(rib, no_eviction, rows, pages, max_rows, keep):
    d, _ = decoder(rib, rows, pages=pages, max_rows=max_rows, keep=keep)
    before = pages_of(d)
    with pytest.raises(rib.PoolFull):
        d._make_room()
    assert pages_of(d) == before and not no_eviction


def test_eviction_that_fails_leaves_the_sequence_as_it_was(rib, monkeypatch):
    """A layer's eviction that raises (memory for its outputs, say): pages, rows and all layers' scores stay."""
    module = importlib.import_module("roofline-inference_b200.paged_batch")
    d, pool = decoder(rib, [64], pages=6, max_rows=64, keep=16, layers=3)
    d.scores.copy_(torch.rand(d.scores.shape))
    before, scores = pages_of(d), d.scores.clone()

    def fails_in_layer_1(pages, *a, new_scores, **kw):
        if pages.data_ptr() == pool.layer(1).data_ptr():
            raise RuntimeError("out of memory")
        new_scores.fill_(7.0)
    monkeypatch.setattr(module, "paged_evict", fails_in_layer_1)
    with pytest.raises(RuntimeError, match="out of memory"):
        d._make_room()
    assert pages_of(d) == before and torch.equal(d.scores, scores)


def test_add_that_fails_gives_its_pages_back(rib, monkeypatch):
    module = importlib.import_module("roofline-inference_b200.paged_batch")
    d, pool = decoder(rib, [16], pages=6, max_rows=64)
    d.remove(0)
    d.e.cfg.vocab_size = 10
    monkeypatch.setattr(rib.PagedDecoder, "_prefill", lambda self, tokens, ids: None)

    def fails(logits):
        raise RuntimeError("out of memory")
    monkeypatch.setattr(module, "argmax", fails)
    with pytest.raises(RuntimeError, match="out of memory"):
        d.add([1, 2, 3])
    assert pool.free_pages == 6 and d.free_slots() == [0]


# ------------------------------------------------------------------ building
def test_library_loads_without_a_host_compiler(rib, monkeypatch):
    """A library that is up to date loads whatever became of the binding (another torch, no g++); only the calls
    that need the binding ask for it, and fail loudly."""
    L = importlib.import_module("roofline-inference_b200._lib")
    L.load()

    def no_compiler(*a):
        raise RuntimeError("no compiler")
    monkeypatch.setattr(L, "_lib", None)
    monkeypatch.setattr(L, "_binding_module", None)
    monkeypatch.setattr(L, "binding_is_current", lambda: False)
    monkeypatch.setattr(L, "_run", no_compiler)
    monkeypatch.setattr(L, "_nvcc", no_compiler)
    assert L.load().rib_version() > 0
    with pytest.raises(RuntimeError, match="no compiler"):
        L.binding()


def test_step_returns_a_tensor_of_the_callers_own(rib, monkeypatch):
    """What a step returned stays what it was when later steps run, eager or replayed."""
    d, _ = decoder(rib, [3], pages=6, max_rows=64)
    monkeypatch.setattr(rib.PagedDecoder, "_forward", lambda self: None)
    monkeypatch.setattr(rib.PagedDecoder, "_argmax", lambda self, logits: self.next.copy_(self.tok + 1))
    d.tok.fill_(5)
    first = d.step()
    second = d.step()
    assert (first.tolist(), second.tolist(), d.tok.tolist()) == ([6], [7], [7])
    d.graph = SimpleNamespace(replay=lambda: (d.next.fill_(40), d.tok.copy_(d.next)))
    third = d.step()
    d.graph = SimpleNamespace(replay=lambda: (d.next.fill_(41), d.tok.copy_(d.next)))
    d.step()
    assert (first.tolist(), second.tolist(), third.tolist()) == ([6], [7], [40])


# ------------------------------------------------------------------ frequencies
@pytest.mark.parametrize("length,slow", [(1, 1.0), (3, 1.0), (6, 1.0), (100, 20.0)])
def test_yarn_stretches_every_pair_of_a_short_original_length(rib, length, slow):
    """Pairs that turn less than slow_turns times over original_length are `factor` times slower: all of them where
    even the fastest (one radian a position) does."""
    paged = importlib.import_module("roofline-inference_b200.paged")
    f, _ = paged.rotary_frequencies(64, 1e4)
    g, _ = paged.rotary_frequencies(64, 1e4, "yarn", 4.0, length, slow_turns=slow)
    assert length < 2 * math.pi * slow
    assert g == [x / 4 for x in f]


@pytest.mark.parametrize("what", ["pool", "rotary device", "rotary dims"])
def test_decoder_refuses_what_its_calls_could_not_use(rib, what):
    """A pool or a rotation on another device, or a rotation of other heads, is refused when the decoder is made."""
    d, pool = decoder(rib, [3], pages=6, max_rows=64)
    rotary = None
    if what == "pool":
        pool = rib.PagePool(2, 1, 6, 16, device="meta")
    else:
        rotary = rib.Rotary(128, device="meta") if what == "rotary device" else rib.Rotary(64, device="cpu")
    with pytest.raises(ValueError):
        rib.PagedDecoder(d.e, pool, 1, 64, rotary=rotary)
