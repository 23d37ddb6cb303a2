"""GPU: PagedDecoder where test_gpu_paged_batch.py does not reach."""
from __future__ import annotations

import pytest
import torch

from test_gpu_paged_batch import small_engine

pytestmark = pytest.mark.gpu


def test_prefill_scratch_does_not_grow_with_the_layers(rib):
    """A prompt's rows pass through one layer's scratch: 24 layers take no more memory beside the pool than 2 do.
    A cache of all layers would be 2 x 2 heads x 4096 rows x 128 dims x 2 bytes = 4 MB a layer more."""
    grown = []
    for layers in (2, 24):
        e = small_engine(rib, layers=layers)
        pool = rib.PagePool.for_engine(e, pages=80, page_rows=64)
        d = rib.PagedDecoder(e, pool, slots=1, max_rows=5000)
        d.remove(d.add([1] * 4096))  # first-call set-up
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        d.add(list(range(900)) + [7] * 3196)
        torch.cuda.synchronize()
        grown.append(torch.cuda.max_memory_allocated() - before)
        del d, pool, e
    assert grown[1] <= grown[0] + (4 << 20), grown


def contiguous(rib, e, prompts, room):
    caches = []
    for p in prompts:
        c = e.new_cache(len(p) + room)
        e.prefill(torch.tensor(p, dtype=torch.int32, device="cuda"), c, last=True)
        caches.append(c)
    return rib.BatchDecoder(e, caches)


def test_more_slots_than_the_library_products_take(rib):
    """Above 64 slots the projections run on the tiled GEMM: eager and captured steps agree bit for bit, idle slots
    between busy ones, and with the contiguous decoder within the bound of the other model tests."""
    e = small_engine(rib, layers=2)
    prompts = [[(7 * i + j) % 1000 for j in range(1 + 3 * i % 40)] for i in range(70)]
    outs = []
    for use_graph in (False, True):
        pool = rib.PagePool.for_engine(e, pages=400, page_rows=16)
        d = rib.PagedDecoder(e, pool, slots=80, max_rows=64)
        if use_graph:
            d.capture()
        slots = [d.add(p) for p in prompts]
        for i in slots[::9]:
            d.remove(i)
        busy = [i for i in slots if d.pages[i] is not None]
        log = []
        for step in range(6):
            d.tok.copy_(torch.arange(80, dtype=torch.int32) * 3 + step)
            log.append(d.step()[busy])
        outs.append(log)
        assert 400 - pool.free_pages == sum(len(p) for p in d.pages if p is not None)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    d.tok.copy_(torch.arange(80, dtype=torch.int32) * 3)
    got = d.logits()[busy]
    batch = contiguous(rib, e, [prompts[i] for i in busy], 16)
    for step in range(6):
        batch.logits(torch.tensor([3 * i + step for i in busy], dtype=torch.int32, device="cuda"))
    want = batch.logits(torch.tensor([3 * i for i in busy], dtype=torch.int32, device="cuda"))
    assert (got - want).abs().max() <= 2e-2 * want.abs().max()
    assert rib._lib.take_device_status() == 0


def test_two_decoders_share_a_pool(rib):
    """Decoders that take pages from one pool in turn give the logits that each gives with a pool of its own, bit for
    bit, eager and captured, through several evictions."""
    e = small_engine(rib)
    prompts = [[5, 6, 7] * 9, list(range(100, 131))]

    def run(pools, use_graph):
        ds = [rib.PagedDecoder(e, pool, slots=2, max_rows=40, keep=18, sinks=1, recent=5) for pool in pools]
        log = []
        for d, p in zip(ds, prompts):
            if use_graph:
                d.capture()
            d.add(p)
        for step in range(50):
            for k, d in enumerate(ds):
                d.tok.fill_((37 * step + 11 * k) % 1000)
                if use_graph:
                    d.step()
                log.append(d.graph_logits[0].clone() if use_graph else d.logits()[0])
        used = [p for d in ds for ids in d.pages if ids for p in ids]
        if pools[0] is pools[1]:
            assert len(set(used)) == len(used) and pools[0].free_pages == 10 - len(used)
        return log

    def pool():
        return rib.PagePool.for_engine(e, pages=10, page_rows=16)
    shared = pool()
    want = run([pool(), pool()], False)
    assert all(torch.equal(x, y) for x, y in zip(run([shared, shared], False), want))
    shared = pool()
    assert all(torch.equal(x, y) for x, y in zip(run([shared, shared], True), want))
    assert rib._lib.take_device_status() == 0


def test_steps_on_a_stream_of_its_own(rib):
    """A decoder made, filled, captured and stepped under another current stream."""
    e = small_engine(rib)
    logs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            pool = rib.PagePool.for_engine(e, pages=8, page_rows=16)
            d = rib.PagedDecoder(e, pool, slots=1, max_rows=33, keep=16, sinks=0, recent=4).capture()
            d.add(list(range(30)))
            outs = []
            for step in range(40):
                d.tok.fill_(37 * step % 1000)
                d.step()
                outs.append(d.graph_logits.clone())
        stream.synchronize()
        logs.append(outs)
    assert all(torch.equal(x, y) for x, y in zip(*logs))
    assert not torch.equal(logs[0][0], logs[0][-1])
    assert rib._lib.take_device_status() == 0
