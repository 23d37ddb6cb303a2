"""GPU: batched decode over paged caches (PagedDecoder) against a plain FP64 forward of the same weights.

Logits are compared within 2e-2 of the largest, the bound that the framework's other model tests put on
BF16 activations against a forward without their roundings (a few hundred roundings of 2^-9 on the way)."""
from __future__ import annotations

import importlib

import pytest
import torch

from paged_ref import kept_rows, rotate64

pytestmark = pytest.mark.gpu
TOL = 2e-2


def small_engine(rib, layers=2, heads=4, seed=5):
    cfg = rib.Qwen3Config(num_layers=layers, hidden_size=256, num_heads=heads, num_kv_heads=heads // 2,
                          intermediate_size=512, vocab_size=1000)
    return rib.Engine(rib.random_weights(cfg, seed=seed).to("cuda"))


def norm(x, w):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()


def mlp(h, w):
    x = norm(h, w["post_norm"])
    g, u = (x @ w["gu"].double().T).chunk(2, -1)
    return h + (torch.nn.functional.silu(g) * u) @ w["down"].double().T


def project(e, h, w, pos, rot):
    nq, nkv = e.nq_local, e.n_kv
    qkv = (norm(h, w["in_norm"]) @ w["qkv"].double().T).view(h.shape[0], nq + 2 * nkv, 128)
    args = (pos, rot.frequencies, rot.gain, rot.rotary_dim, rot.interleaved)
    q, _ = rotate64(qkv[:, :nq], *args, w=w["q_norm"])
    k, _ = rotate64(qkv[:, nq:nq + nkv], *args, w=w["k_norm"])
    return q, k, qkv[:, nq + nkv:]


def plain_logits(e, tokens, rot):
    """Logits of the last of `tokens`, every one attending to all before it."""
    h = e.embed.double()[tokens]
    n = h.shape[0]
    pos = torch.arange(n, device="cuda")
    mask = torch.ones(n, n, device="cuda").tril().bool()
    for w in e.layers:
        q, k, v = project(e, h, w, pos, rot)
        k, v = (t.repeat_interleave(2, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * e.scale
        p = torch.softmax(s.masked_fill(~mask, -torch.inf), -1)
        o = torch.einsum("hqk,khd->qhd", p, v).reshape(n, -1)
        h = mlp(h + o @ w["o"].double().T, w)
    return norm(h[-1], e.final_norm) @ e.embed.double().T


def near(got, want):
    d = (got.double() - want).abs().max() / want.abs().max()
    assert d <= TOL, float(d)


@pytest.mark.parametrize("page_rows", [16, 64])
@pytest.mark.parametrize("scaling", [None, "yarn"])
def test_prefill_and_steps(rib, page_rows, scaling):
    """Prompts of one token, of one that ends a page and of several pages; a step at a page's border."""
    e = small_engine(rib)
    kw = dict(scaling=scaling, factor=4.0, original_length=64) if scaling else {}
    rot = rib.Rotary(128, e.base, interleaved=False, **kw)
    pool = rib.PagePool.for_engine(e, pages=40, page_rows=page_rows)
    d = rib.PagedDecoder(e, pool, slots=4, max_rows=200, rotary=rot)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (1, page_rows, 130)]
    slots = [d.add(p) for p in prompts]
    assert slots == [0, 1, 2] and d.free_slots() == [3]
    seqs = [list(p) for p in prompts]
    for s, p in zip(slots, prompts):
        want = plain_logits(e, p, rot)
        assert (want.max() - want[int(d.tok[s])]) <= TOL * want.abs().max()  # the greedy token, or one as good
    for step in range(3):
        for s, q in zip(slots, seqs):
            q.append(int(d.tok[s]))
        lg = d.logits()
        for s, q in zip(slots, seqs):
            near(lg[s], plain_logits(e, q, rot))
        d.tok.copy_(torch.randint(0, 1000, (4,), generator=g).int())
    assert d.rows[:3] == [n + 3 for n in (1, page_rows, 130)]
    used = 40 - pool.free_pages
    assert used == sum(pool.pages_for(r) for r in d.rows[:3])
    for s in slots:
        d.remove(s)
    assert pool.free_pages == 40
    assert rib._lib.take_device_status() == 0


def test_graph_equals_eager_with_membership_and_eviction(rib):
    """The captured step gives the eager step's tokens bit for bit while sequences join, leave, grow and
    are evicted between replays."""
    e = small_engine(rib, layers=3)
    outs = []
    for use_graph in (False, True):
        pool = rib.PagePool.for_engine(e, pages=24, page_rows=16)
        d = rib.PagedDecoder(e, pool, slots=3, max_rows=48, keep=20, sinks=2, recent=6)
        if use_graph:
            d.capture()
        d.tok.zero_()
        log = []
        a = d.add([5, 6, 7])
        for step in range(120):
            if step == 10:
                b = d.add(list(range(1, 41)))
            if step == 60:
                d.remove(a)
            if step == 70:
                a = d.add([9] * 48)   # full at once: cut before its first step
            live = [i for i in range(3) if d.pages[i] is not None]
            t = d.step().cpu()
            log.append([(i, int(t[i])) for i in live])
            assert all(d.rows[i] <= 48 for i in live)
            assert 24 - pool.free_pages == sum(len(p) for p in d.pages if p is not None)
        assert d.positions[b] == 40 + 110 and d.rows[b] <= 48
        outs.append(log)
        for i in (a, b):
            d.remove(i)
        assert pool.free_pages == 24
    assert outs[0] == outs[1]
    assert rib._lib.take_device_status() == 0


def test_step_after_eviction_attends_to_the_kept_rows(rib):
    """An eviction keeps the rows that each head's scores rank highest, and the next step's logits are
    those of attention over what the pages then hold."""
    e = small_engine(rib)
    rot = rib.Rotary(128, e.base)
    pool = rib.PagePool.for_engine(e, pages=12, page_rows=16)
    d = rib.PagedDecoder(e, pool, slots=1, max_rows=40, keep=24, sinks=2, recent=5)
    d.add(list(range(3, 33)))
    while d.rows[0] < 40:
        d.step()
    before = [s[0].clone() for s in d.scores]
    old = [pool.layer(l)[torch.tensor(d.pages[0])].clone() for l in range(2)]
    token, pos = int(d.tok[0]), d.positions[0]
    lg = d.logits()
    assert d.rows[0] == 25 and len(d.pages[0]) == 2
    h = e.embed.double()[[token]]
    for l, w in enumerate(e.layers):
        q, k, v = project(e, h, w, torch.tensor([pos], device="cuda"), rot)
        o = []
        for head in range(e.n_kv):
            at = torch.tensor(kept_rows(before[l][head].cpu(), 40, 24, 2, 5), device="cuda")
            K, V = (old[l][at // 16, i, head, at % 16].double() for i in (0, 1))
            K, V = torch.cat([K, k[:, head]]), torch.cat([V, v[:, head]])
            p = torch.softmax(q[0, 2 * head:2 * head + 2] @ K.T * e.scale, -1)
            o.append(p @ V)
        h = mlp(h + torch.cat(o).reshape(1, -1) @ w["o"].double().T, w)
    near(lg[0], (norm(h[0], e.final_norm) @ e.embed.double().T))


def test_agrees_with_the_contiguous_decoder(rib):
    e = small_engine(rib, layers=3, heads=8)
    prompts = [[1, 2, 3, 4, 5], list(range(100, 180))]
    caches = []
    for p in prompts:
        c = e.new_cache(len(p) + 8)
        e.prefill(torch.tensor(p, dtype=torch.int32, device="cuda"), c, last=True)
        caches.append(c)
    batch = rib.BatchDecoder(e, caches)
    pool = rib.PagePool.for_engine(e, pages=16, page_rows=16)
    d = rib.PagedDecoder(e, pool, slots=2, max_rows=128)
    for p in prompts:
        d.add(p)
    for step in range(4):
        toks = torch.tensor([7 + step, 900 - step], dtype=torch.int32, device="cuda")
        d.tok.copy_(toks)
        want, got = batch.logits(toks), d.logits()
        assert (got - want).abs().max() <= TOL * want.abs().max()


def test_refusals(rib):
    e = small_engine(rib)
    pool = rib.PagePool.for_engine(e, pages=4, page_rows=16)
    for kw in (dict(slots=0), dict(max_rows=0), dict(keep=0), dict(keep=64), dict(keep=8, sinks=5, recent=4)):
        with pytest.raises(ValueError):
            rib.PagedDecoder(e, pool, **{"slots": 2, "max_rows": 64, **kw})
    with pytest.raises(ValueError):
        rib.PagedDecoder(e, rib.PagePool(3, e.n_kv, 4, device="cuda"), 2, 64)
    d = rib.PagedDecoder(e, pool, slots=2, max_rows=32)
    for bad in ([], [1000], [-1], [1] * 33):
        with pytest.raises(ValueError):
            d.add(bad)
    assert pool.free_pages == 4
    with pytest.raises(ValueError):
        d.remove(0)
    d.add([1] * 31)
    with pytest.raises(ValueError):
        d.capture()
    d.step()
    with pytest.raises(ValueError, match="capacity"):
        d.step()                       # 32 rows, no eviction
    d.add([2] * 31)
    d.remove(0)
    held = pool.take(2)
    assert pool.free_pages == 0
    d2 = rib.PagedDecoder(e, pool, slots=1, max_rows=32)
    with pytest.raises(rib.PoolFull):
        d2.add([1])
    pool.give(held)


def test_full_pool_changes_nothing(rib):
    e = small_engine(rib)
    pool = rib.PagePool.for_engine(e, pages=2, page_rows=16)
    d = rib.PagedDecoder(e, pool, slots=2, max_rows=64)
    d.add([1] * 16)
    d.add([2] * 16)
    state = (list(d.rows), [list(p) for p in d.pages], d.row.tolist(), d.lens.tolist(), d.table.tolist())
    with pytest.raises(rib.PoolFull):
        d.step()
    assert state == (list(d.rows), [list(p) for p in d.pages], d.row.tolist(), d.lens.tolist(), d.table.tolist())
    d.remove(1)
    d.step()
    assert d.rows[0] == 17
