"""GPU: the paged-cache operators where the other tests do not reach.  Tolerances as in test_gpu_paged.py, or
derived where they are used."""
from __future__ import annotations

import importlib
import math

import pytest
import torch

from paged_ref import attend64, half_step, make_cache, smallest_half
from test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def lib():
    L = importlib.import_module("roofline-inference_b200._lib")
    L.take_device_status()
    return L


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ long sums
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,D", [(2, 64), (2, 128), (16, 64), (16, 128)])
def test_attention_long_sums_are_not_truncated(rib, lib, nq, D, dtype):
    """2^20 rows in few CTAs: every warp adds up 16384 tiles.  V is 1 in the first half of the rows and -1 in the
    second, which has the first half's keys in another order, so the output is 0 whatever the error of a single
    weight.  What is left is the error of adding m = 16384 tiles to a sum of at most half of all weights, m
    roundings to nearest of 2^-24 of it each: with independent roundings beyond 8 sqrt(m) of them once in 10^13
    (8 standard deviations).  The join's few additions are within the same.  Sums that round toward 0 lose half a
    step every time, 8 times as much."""
    n, P, B = 1 << 20, 256, 450
    g = gen(1)
    k = (torch.randint(-64, 65, (n // 2,), generator=g) / 64).to(dtype)
    pages = torch.zeros((n // P, 2, 1, P, D), dtype=dtype, device="cuda")
    pages[:, 0, 0, :, 0] = torch.cat([k, k[torch.randperm(n // 2, generator=g)]]).view(-1, P).cuda()
    pages[:n // P // 2, 1] = 1
    pages[n // P // 2:, 1] = -1
    table = torch.arange(n // P, dtype=torch.int32, device="cuda").expand(B, -1)  # every sequence has the same pages
    q = torch.zeros((B, nq, D), dtype=dtype, device="cuda")
    q[:, :, 0] = 8.0
    got = rib.paged_decode_attention(q, pages, table, i32([n] * B), 0.125)
    assert lib.take_device_status() == 0
    worst = float(got.double().abs().max())
    assert worst <= 0.5 * 8 * math.sqrt(16384) * 2.0 ** -24, worst


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,D", [(1, 1, 64), (4, 2, 128), (8, 1, 64), (16, 1, 128), (20, 1, 64), (40, 2, 128)])
@pytest.mark.parametrize("n", [5, 250, 6000])
@pytest.mark.parametrize("low", ["one row", "half of the rows"])
def test_attention_infinite_and_nan_values(rib, lib, low, n, nq, nkv, D, dtype):
    """Infinities in V that are attended to give infinities, NaN where both signs meet; NaN gives NaN; the other
    dims are as without them.  The first row's weight is about 2^-45 of the largest, or that of the first half of
    the rows 2^-290: no weight is so small that an infinity would not show."""
    g = gen(n)
    pages, table = make_cache([n], nkv, D, 16, dtype, g)
    at = lambda r: (int(table[0, r // 16]), r % 16)  # noqa: E731
    q = torch.randn((1, nq, D), generator=g).to(dtype).cuda()
    q[..., 0] = 16.0
    K = pages[:, 0, :, :, 0]
    K[...] = torch.where(K.isnan(), K, 0)  # dim 0 of the keys sets some rows far below the others
    for r in range(1 if low == "one row" else n // 2):
        page, slot = at(r)
        pages[page, 0, :, slot, 0] = -(31 if low == "one row" else 200) * math.sqrt(D) / 16
    for r, d, x in [(0, 1, math.inf), (n // 2, 2, -math.inf), (n - 1, 3, math.inf), (n // 3, 4, math.nan),
                    (1, 5, math.inf), (n - 2, 5, -math.inf), (0, D - 1, -math.inf)]:
        page, slot = at(r)
        pages[page, 1, :, slot, d] = x
    clean = pages.clone()
    page, slot = torch.tensor([at(r) for r in range(n)], device="cuda").T
    V = clean[page, 1, :, slot]
    clean[page, 1, :, slot] = torch.where(V.isfinite(), V, 0)
    lens, scale = [n], D ** -0.5
    want, _, bound, _ = attend64(q, clean, table, lens, scale)
    got = rib.paged_decode_attention(q, pages, table, i32(lens), scale)
    assert lib.take_device_status() == 0
    for d, x in [(1, math.inf), (2, -math.inf), (3, math.inf), (D - 1, -math.inf)]:
        assert (got[..., d] == x).all(), (d, got[..., d])
    for d in (4, 5):
        assert got[..., d].isnan().all()
    rest = torch.tensor([d for d in range(D) if d not in (1, 2, 3, 4, 5, D - 1)], device="cuda")
    a, w, b = got[..., rest].double(), want[..., rest], bound[..., rest]
    assert ((a - w).abs() <= w.abs() * half_step(dtype) + smallest_half(dtype) + b).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,D", [(4, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("n", [1, 250, 6000])
def test_attention_scores_of_minus_infinity(rib, lib, n, nq, nkv, D, dtype):
    """Rows whose keys make their scores -infinity get no weight; where all do, the output is zeros and no row's
    score changes."""
    g = gen(n)
    pages, table = make_cache([n, n], nkv, D, 16, dtype, g)
    clean = pages.clone()
    at = torch.arange(n, device="cuda")
    pages[table[0, at // 16].long(), 0, :, at % 16, 0] = -math.inf        # sequence 0: every row
    some = at[(at % 3 > 0) | (at < n // 2)] if n > 1 else at[:0]            # sequence 1: most rows
    pages[table[1, some // 16].long(), 0, :, some % 16, 0] = -math.inf
    q = torch.randn((2, nq, D), generator=g).to(dtype).cuda()
    q[..., 0] = 1.0
    old = torch.rand((2, nkv, table.shape[1] * 16), generator=g).cuda()
    scores = old.clone()
    got = rib.paged_decode_attention(q, pages, table, i32([n, n]), D ** -0.5, scores=scores)
    assert lib.take_device_status() == 0
    assert (got[0] == 0).all() and torch.equal(scores[0], old[0])
    # sequence 1: attention over the rows that are left, gathered into pages of their own
    left = at[~torch.isin(at, some)]
    m = left.numel()
    short, one = make_cache([m], nkv, D, 16, dtype, g)
    to = torch.arange(m, device="cuda")
    short[one[0, to // 16].long(), :, :, to % 16] = clean[table[1, left // 16].long(), :, :, left % 16]
    want, weights, bound, rel = attend64(q[1:], short, one, [m], D ** -0.5)
    assert ((got[1:].double() - want).abs() <= want.abs() * half_step(dtype) + smallest_half(dtype) + bound).all()
    expect = old[1, :, left].double() + weights[0]
    assert ((scores[1, :, left].double() - expect).abs() <= expect * 2.0 ** -24 + weights[0] * rel[0]).all()
    assert torch.equal(scores[1, :, some], old[1, :, some]) and torch.equal(scores[1, :, n:], old[1, :, n:])


# ------------------------------------------------------------------ eviction
def test_evict_keep_is_bounded(rib, lib):
    """`keep` beyond what the loops over rows count to is refused on the host, before its buffers are made."""
    pages, table = make_cache([40], 1, 64, 16, BF16, gen(0), fill=0.0)
    scores = torch.rand((1, 1, 48), generator=gen(1)).cuda()
    before = pages.clone()
    for keep in (0x7f000001, 2 ** 31 - 1):
        with pytest.raises(ValueError, match="keep"):
            rib.paged_evict(pages, table, i32([40]), scores, keep, table)
    assert torch.equal(pages, before) and lib.take_device_status() == 0


# ------------------------------------------------------------------ layouts
def strided(sizes, order, pad):
    """Zeros of `sizes` whose dims lie in memory in `order` (outermost first; the last dim innermost), with `pad`
    elements behind every run of the innermost dims."""
    strides, step = [0] * len(sizes), 1
    for d in reversed([*order, len(sizes) - 1]):
        strides[d] = step
        step = step * sizes[d] + pad
    return torch.zeros(step, dtype=BF16, device="cuda").as_strided(sizes, strides)


@pytest.mark.parametrize("order,pad", [
    ((0, 1, 2, 3), 8),    # padded rows, heads, halves and pages: no stride is a multiple of another
    ((0, 1, 3, 2), 0),    # rows before heads
    ((1, 0, 2, 3), 0),    # K and V as outer halves
    ((0, 3, 1, 2), 0),    # a row's K and V together
    ((2, 0, 1, 3), 0),    # a pool for each head
    ((3, 2, 1, 0), 24),   # everything the other way round
])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_in_any_order(rib, lib, order, pad, D):
    """Append, attention and eviction give the same bits whatever the order of the pages' dims in memory."""
    g = gen(31)
    nq, nkv, P, lens = 6, 3, 32, [70, 33, 0, 2000]
    base, table = make_cache(lens, nkv, D, P, BF16, g, spare=40, fill=0.0)
    free = sorted(set(range(base.shape[0])) - set(table.flatten().tolist()))
    new = i32([free[:2], free[2:4], [-1, -1], free[4:6]])
    q, k, v = (torch.randn((4, h, D), generator=g).to(BF16).cuda() for h in (nq, nkv, nkv))
    scores = torch.rand((4, nkv, table.shape[1] * P), generator=g).cuda()
    rot, row = rib.Rotary(D), i32([69, 32, -1, 1999])
    results = []
    for pages in (base.clone(), strided(base.shape, order, pad)):
        pages.copy_(base)
        sc = scores.clone()
        qr = rib.paged_append(q, k, v, i32([7, 8, 9, 10]), row, pages, table, rot)
        out = rib.paged_decode_attention(qr, pages, table, i32(lens), 0.1, scores=sc)
        rows, n = rib.paged_evict(pages, table, i32(lens), sc, 64, new, sinks=3, recent=9)
        results.append((qr, out, sc, rows, n, pages))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert lib.take_device_status() == 0
    want, _, bound, _ = attend64(results[0][0][:2], base_after_append(base, results[0][5], table, lens), table, lens[:2], 0.1)
    got = results[1][1][:2]
    assert ((got.double() - want).abs() <= want.abs() * half_step(BF16) + smallest_half(BF16) + bound).all()


def base_after_append(before, after, table, lens):
    """The pages as the attention saw them: those of the table, before the eviction wrote to others."""
    pages = before.clone()
    used = table[table >= 0].long()
    pages[used] = after[used]
    return pages


def test_append_of_broadcast_heads(rib, lib):
    """k and v as one head expanded over all KV heads, one token expanded over all sequences."""
    g = gen(32)
    nkv, D = 4, 64
    q = torch.randn((3, 8, D), generator=g).to(BF16).cuda()
    k = torch.randn((3, 1, D), generator=g).to(BF16).cuda().expand(3, nkv, D)
    v = torch.randn((1, nkv, D), generator=g).to(BF16).cuda().expand(3, nkv, D)
    table, rot, pos, row = i32([[0], [1], [2]]), rib.Rotary(D), i32([5, 6, 7]), i32([0, 3, 15])
    pages = [torch.zeros((3, 2, nkv, 16, D), dtype=BF16, device="cuda") for _ in range(2)]
    a = rib.paged_append(q, k, v, pos, row, pages[0], table, rot)
    b = rib.paged_append(q, k.contiguous(), v.contiguous(), pos, row, pages[1], table, rot)
    assert torch.equal(a, b) and torch.equal(*pages) and (pages[0][1, 1, :, 3] == v[1]).all()
    before = pages[0].clone()
    none = rib.paged_append(q[:0], k[:0], v[:0], pos[:0], row[:0], pages[0], table, rot)
    assert none.shape == (0, 8, D) and torch.equal(pages[0], before)
    assert lib.take_device_status() == 0


# ------------------------------------------------------------------ many heads, bounds on lengths
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (FP16, 128)])
@pytest.mark.parametrize("nq,nkv", [(128, 1), (129, 1), (272, 1), (290, 2)])
def test_attention_row_weights_of_many_heads(rib, lib, nq, nkv, D, dtype):
    """More than 128 query heads to a KV head: their weights of a row are summed in several passes, of whole and of
    joined units."""
    check_attention(rib, lib, [1, 17, 0, 250], nq=nq, nkv=nkv, D=D, page_rows=16, dtype=dtype, scores=True)
    check_attention(rib, lib, [5000, 33, 0, 1200], nq=nq, nkv=nkv, D=D, page_rows=16, dtype=dtype, scores=True, seed=1)


@pytest.mark.parametrize("max_len", [200, 256, 257, 1000, None])
@pytest.mark.parametrize("scores", [False, True])
def test_attention_with_any_bound_on_the_lengths(rib, lib, max_len, scores):
    """max_len chooses how units are split, and with it the order of the sums; every choice is within the bounds."""
    check_attention(rib, lib, [200, 3, 0, 77], nq=8, nkv=2, D=128, page_rows=16, dtype=BF16, max_len=max_len, width=80,
                    scores=scores)
