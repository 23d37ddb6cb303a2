"""GPU: the paged-cache operators against their definitions in 64 bits (paged_ref.py).

Tolerances: every result is rounded to its type once, so it may be off by half a step of that type
(torch.finfo(t).eps / 2 relative) plus the FP32 arithmetic before it, whose bound is written where it
is used.  Selections of rows and moved values must be exact."""
from __future__ import annotations

import importlib
import math

import pytest
import torch

from paged_ref import attend64, half_step, kept_rows, make_cache, rotate64, smallest_half

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


def close(got, want, slack):
    """|got - want| <= half a step of got's type + slack, element by element."""
    d = (got.double() - want).abs()
    lim = want.abs() * half_step(got.dtype) + smallest_half(got.dtype) + slack
    bad = ~(d <= lim)
    assert not bad.any(), (int(bad.sum()), float((d / lim)[bad].max()), bad.nonzero()[:3].tolist())


# ------------------------------------------------------------------ rotary positions
# FP32 arithmetic of a rotation, in units of 2^-24 of |a| + |b|: the norm's sum over 256 values in
# chains of 16 and its shuffles (20 additions, halved by the root), root, quotient and two products (4),
# the angle (half a turn rounded to FP32 is off by 2^-25 turns, 3.2 units of 2^-24 radians) and its sine
# (2 ulp each), gain, two products and a sum (4): under 28 in all.
ROT = 28 * 2.0 ** -24

ROTATIONS = [
    dict(head_dim=128), dict(head_dim=64, interleaved=True), dict(head_dim=128, rotary_dim=64),
    dict(head_dim=64, rotary_dim=48, interleaved=True), dict(head_dim=96, rotary_dim=32, base=1e4),
    dict(head_dim=256, rotary_dim=16), dict(head_dim=80, base=1e4), dict(head_dim=32, interleaved=True),
    dict(head_dim=128, scaling="linear", factor=4.0), dict(head_dim=128, scaling="ntk", factor=8.0),
    dict(head_dim=128, scaling="yarn", factor=4.0, original_length=4096, interleaved=True),
    dict(head_dim=256, scaling="yarn", factor=32.0, original_length=32768),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("spec", ROTATIONS, ids=lambda s: "-".join(str(v) for v in s.values()))
def test_rotary(rib, spec, dtype):
    rot = rib.Rotary(**spec)
    D = spec["head_dim"]
    for tokens, heads in [(1, 1), (5, 3), (67, 33)]:
        x = torch.randn((tokens, heads, D), generator=gen(tokens)).to(dtype).cuda()
        pos = torch.randint(0, 1 << 21, (tokens,), generator=gen(1), dtype=torch.int32).cuda()
        pos[0] = 0
        want, size = rotate64(x, pos, rot.frequencies, rot.gain, rot.rotary_dim, rot.interleaved)
        got = rib.rotary(x, pos, rot)
        assert got.dtype == dtype and got.shape == x.shape
        close(got, want, size * ROT)
        assert torch.equal(got[..., rot.rotary_dim:], x[..., rot.rotary_dim:])  # the rest passes bit for bit
        same = x.clone()
        assert rib.rotary(same, pos, rot, out=same) is same and torch.equal(same, got)  # in place
    assert rib.rotary(x[:0], pos[:0], rot).shape == (0, heads, D)


def test_rotary_far_positions_and_strides(rib):
    """The largest positions, and x as a transposed view into a wider buffer."""
    rot = rib.Rotary(128)
    wide = torch.randn((6, 9, 160), generator=gen(0)).to(BF16).cuda()
    x = wide.transpose(0, 1)[:, 1:5, 16:144]
    pos = i32([0, 1, 2 ** 17 + 1, 2 ** 24 + 1, 2 ** 31 - 1, -1, -70000, 12345, 2 ** 30])
    before = wide.clone()
    out = torch.zeros((4, 9, 128), dtype=BF16, device="cuda").transpose(0, 1)
    got = rib.rotary(x, pos, rot, out=out)
    want, size = rotate64(x, pos, rot.frequencies, rot.gain, 128, False)
    close(got, want, size * ROT)
    assert torch.equal(wide, before)


# ------------------------------------------------------------------ append
def check_append(rib, lib, *, T, nq, nkv, D, page_rows, dtype, norm, seqs, first, rot, seed=0, pages_view=None):
    g = gen(seed)
    share = -(-T // seqs)
    seq = [t // share for t in range(T)]
    row = [first + t % share for t in range(T)]
    width = (first + share - 1) // page_rows + 2
    total = seqs * width
    pages = torch.randn((total + 2, 2, nkv, page_rows, D), generator=g).to(dtype).cuda()
    if pages_view:
        pages = pages_view(pages)
    table = torch.randperm(total, generator=g).to(torch.int32).view(seqs, width).cuda()
    qkv = torch.randn((T, (nq + 2 * nkv) * D), generator=g).to(dtype).cuda()
    q, k, v = (s.view(T, -1, D) for s in qkv.split([nq * D, nkv * D, nkv * D], 1))
    pos = torch.randint(0, 200000, (T,), generator=g, dtype=torch.int32).cuda()  # rows are not positions
    qw = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() if norm else None
    kw = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() if norm else None
    want = pages.clone()
    got_q = rib.paged_append(q, k, v, pos, i32(row), pages, table, rot, seq=i32(seq), qw=qw, kw=kw)
    args = (pos, rot.frequencies, rot.gain, rot.rotary_dim, rot.interleaved)
    q64, qs = rotate64(q, *args, w=qw)
    k64, ks = rotate64(k, *args, w=kw)
    close(got_q, q64, qs * ROT)
    page = table[i32(seq).long(), i32(row).long() // page_rows].long()
    slot = i32(row).long() % page_rows
    close(pages[page, 0, :, slot], k64, ks * ROT)
    assert torch.equal(pages[page, 1, :, slot], v)
    want[page, :, :, slot] = pages[page, :, :, slot]
    assert torch.equal(pages, want)  # nothing else was written
    assert lib.take_device_status() == 0


APPENDS = [
    dict(T=1, nq=16, nkv=8, D=128, page_rows=16, dtype=BF16, norm=True, seqs=1, first=513),
    dict(T=1, nq=1, nkv=1, D=64, page_rows=16, dtype=FP16, norm=False, seqs=1, first=0),
    dict(T=5, nq=16, nkv=8, D=128, page_rows=64, dtype=BF16, norm=True, seqs=5, first=63),
    dict(T=33, nq=6, nkv=2, D=64, page_rows=32, dtype=FP16, norm=True, seqs=2, first=30),
    dict(T=300, nq=20, nkv=1, D=128, page_rows=16, dtype=BF16, norm=False, seqs=3, first=7),
    dict(T=257, nq=4, nkv=4, D=256, page_rows=1, dtype=BF16, norm=True, seqs=1, first=0),
    dict(T=9, nq=3, nkv=3, D=96, page_rows=5, dtype=FP16, norm=True, seqs=2, first=11),
    dict(T=3001, nq=32, nkv=8, D=128, page_rows=256, dtype=FP16, norm=True, seqs=1, first=1),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"T{c['T']}-{c['nq']}x{c['nkv']}x{c['D']}-p{c['page_rows']}")
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(rib, lib, case, interleaved):
    D = case["D"]
    check_append(rib, lib, rot=rib.Rotary(D, interleaved=interleaved), **case)
    check_append(rib, lib, rot=rib.Rotary(D, rotary_dim=D // 2 // 16 * 16, interleaved=interleaved, scaling="yarn",
                                          factor=4.0, original_length=8192), **case, seed=1)


def test_append_into_one_layer_of_a_pool(rib, lib):
    """Pages that are a slice of a larger tensor: every stride differs from the contiguous one."""
    def view(pages):
        pool = torch.randn((pages.shape[0], 3, 2, pages.shape[2], pages.shape[3], 2 * pages.shape[4]),
                           generator=gen(9)).to(pages.dtype).cuda()
        return pool[:, 1, ..., :pages.shape[4]]
    check_append(rib, lib, rot=rib.Rotary(128), T=40, nq=4, nkv=2, D=128, page_rows=16, dtype=BF16, norm=True, seqs=4,
                 first=10, pages_view=view)


def test_append_padding_and_missing_pages(rib, lib):
    """A negative row writes nothing; a row, sequence or page that is not there writes nothing and is reported."""
    rot = rib.Rotary(64)
    pages = torch.zeros((3, 2, 2, 16, 64), dtype=BF16, device="cuda")
    table = i32([[0, 1], [2, -1]])
    x = torch.randn((6, 2, 64), generator=gen(0)).to(BF16).cuda()

    def call(seq, row):
        pages.zero_()
        q = rib.paged_append(x[:len(row)], x[:len(row)], x[:len(row)], i32([7] * len(row)), i32(row), pages, table,
                             rot, seq=i32(seq))
        assert torch.equal(q, rib.rotary(x[:len(row)], i32([7] * len(row)), rot))
        return lib.take_device_status(), int((pages != 0).any(-1).any(1).any(1).sum())
    assert call([0, 0, 1], [0, -1, -5]) == (0, 1)
    assert call([0, 1], [17, 15]) == (0, 2)
    for seq, row in [([0], [32]), ([1], [16]), ([2], [0]), ([-1], [3]), ([0], [2 ** 31 - 1])]:
        assert call(seq, row) == (lib.RIB_ECAPACITY, 0)
    table[0, 0] = 3  # outside the pool
    assert call([0], [0]) == (lib.RIB_ECAPACITY, 0)


# ------------------------------------------------------------------ attention
def check_attention(rib, lib, lens, *, nq, nkv, D, page_rows, dtype, scores=False, seed=0, q_scale=1.0, fill=math.nan,
                    max_len=None, width=None):
    g = gen(seed)
    B = len(lens)
    pages, table = make_cache(lens, nkv, D, page_rows, dtype, g, fill=fill, width=width)
    q = (torch.randn((B, nq, D), generator=g) * q_scale).to(dtype).cuda()
    scale = D ** -0.5
    want, weights, bound, rel = attend64(q, pages, table, lens, scale)
    kw = {}
    if scores:
        room = table.shape[1] * page_rows
        old = torch.rand((B, nkv, room + 3), generator=g).cuda()
        new = torch.full_like(old, -7.0)
        kw = dict(scores=old, scores_out=new)
    got = rib.paged_decode_attention(q, pages, table, i32(lens), scale, max_len=max_len, **kw)
    assert lib.take_device_status() == 0
    close(got, want, bound)
    if scores:
        for b, n in enumerate(lens):
            expect = old[b, :, :n].double() + weights[b]
            assert ((new[b, :, :n].double() - expect).abs() <= expect * 2.0 ** -24 + weights[b] * rel[b]).all()
            assert (new[b, :, n:] == -7.0).all()
        again = old.clone()
        out = rib.paged_decode_attention(q, pages, table, i32(lens), scale, max_len=max_len, scores=again)
        assert torch.equal(out, got)
        for b, n in enumerate(lens):
            assert torch.equal(again[b, :, :n], new[b, :, :n]) and torch.equal(again[b, :, n:], old[b, :, n:])
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (16, 8), (10, 2), (8, 1), (18, 2), (20, 1)])
def test_attention_heads_and_types(rib, lib, nq, nkv, D, dtype):
    check_attention(rib, lib, [1, 15, 16, 17, 0, 33, 200], nq=nq, nkv=nkv, D=D, page_rows=16, dtype=dtype, scores=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,nkv", [(9, 1), (16, 1), (17, 1), (32, 1), (30, 2), (40, 1)])
def test_attention_more_than_eight_heads_to_a_kv_head(rib, lib, nq, nkv, D, dtype):
    """Units of 16 query heads, whole, in pieces and in runs, with partly filled units."""
    check_attention(rib, lib, [1, 17, 0, 250], nq=nq, nkv=nkv, D=D, page_rows=16, dtype=dtype, scores=True)
    check_attention(rib, lib, [5000, 33, 0, 1200], nq=nq, nkv=nkv, D=D, page_rows=16, dtype=dtype, scores=True, seed=1)
    check_attention(rib, lib, [40000], nq=nq, nkv=nkv, D=D, page_rows=64, dtype=dtype, scores=nq < 20, seed=2, q_scale=3.0)


@pytest.mark.parametrize("page_rows", [16, 32, 48, 64, 256])
def test_attention_pages_that_end_inside(rib, lib, page_rows):
    check_attention(rib, lib, [page_rows - 1, page_rows, page_rows + 1, 3 * page_rows + 5, 1], nq=4, nkv=2, D=128,
                    page_rows=page_rows, dtype=BF16, scores=page_rows == 48)


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf, 3e38])
def test_attention_ignores_what_lies_behind(rib, lib, fill):
    """Rows behind the last one and pages no sequence names may hold anything."""
    dtype = BF16
    check_attention(rib, lib, [1, 9, 31, 130], nq=4, nkv=2, D=128, page_rows=32, dtype=dtype, fill=fill, scores=True)


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [1], [4097], [0, 5000, 0, 3, 0], [16 * 8 + 1], [20000]])
@pytest.mark.parametrize("scores", [False, True])
def test_attention_lengths(rib, lib, lens, scores):
    check_attention(rib, lib, lens, nq=4, nkv=2, D=128, page_rows=64, dtype=BF16, scores=scores)


@pytest.mark.parametrize("B", [129, 700])
def test_attention_many_sequences(rib, lib, B):
    """More sequences than a CTA has threads, most of one tile, some empty."""
    lens = [(b * 7919) % 40 if b % 5 else 0 for b in range(B)]
    lens[B // 2] = 900
    check_attention(rib, lib, lens, nq=2, nkv=1, D=64, page_rows=16, dtype=FP16, scores=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention_sharp_and_large_scores(rib, lib, dtype):
    """Scores in the hundreds: one row takes nearly all the weight, the running maximum moves."""
    check_attention(rib, lib, [1000, 77], nq=4, nkv=2, D=128, page_rows=16, dtype=dtype, q_scale=40.0, scores=True)


@pytest.mark.parametrize("B,high", [(1, 256), (40, 17), (700, 40), (1500, 1), (333, 256)])
@pytest.mark.parametrize("scores", [False, True])
def test_attention_short_tables(rib, lib, B, high, scores):
    """Tables of at most 256 rows: units are never split; several units to a CTA, and empty sequences."""
    lens = [(b * 7919) % (high + 1) for b in range(B)]
    lens[-1] = high
    check_attention(rib, lib, lens, nq=4, nkv=2, D=64 if B > 1 else 128, page_rows=16, dtype=BF16, scores=scores)


@pytest.mark.parametrize("lens", [[4719], [4720], [4737], [4736, 1], [16 * 148], [300] * 12, [3000, 0, 1, 1700]])
def test_attention_between_pieces_and_runs(rib, lib, lens):
    """Few tiles are cut into pieces of units, one to a CTA; more than fill the GPU into equal runs."""
    check_attention(rib, lib, lens, nq=16, nkv=8, D=128, page_rows=16, dtype=FP16, scores=True)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("gap", [12.0, 17.0, 19.0])
@pytest.mark.parametrize("n", [200, 30000])
def test_attention_many_small_weights_behind_one_large(rib, lib, n, gap, dtype):
    """One row takes nearly all the weight and has V = 0, so the output is what all the others (weights
    of exp(-gap) each, V near 1) add up to: they must not be lost in the type of P."""
    g = gen(12)
    D = 64
    pages, table = make_cache([n], 1, D, 16, dtype, g)
    at = torch.arange(n, device="cuda")
    page, slot = table[0, at // 16].long(), at % 16
    pages[page, 0, 0, slot] = 0
    pages[page, 1, 0, slot] = (1 + torch.rand((n, D), generator=g).cuda() / 8).to(dtype)
    pages[page[n // 3], 0, 0, slot[n // 3], 0] = gap
    pages[page[n // 3], 1, 0, slot[n // 3]] = 0
    q = torch.zeros((1, 2, D), dtype=dtype, device="cuda")
    q[:, :, 0] = 8.0
    scores = torch.zeros((1, 1, table.shape[1] * 16), device="cuda")
    want, weights, bound, rel = attend64(q, pages, table, [n], 0.125)
    got = rib.paged_decode_attention(q, pages, table, i32([n]), 0.125, scores=scores)
    close(got, want, bound)
    assert ((scores[0, :, :n].double() - weights[0]).abs() <= weights[0] * (rel[0] + 2.0 ** -24)).all()


def test_attention_max_len_and_wide_table(rib, lib):
    check_attention(rib, lib, [40, 100], nq=2, nkv=1, D=128, page_rows=16, dtype=BF16, max_len=100, width=50, scores=True)


def test_attention_lengths_out_of_range_are_clamped(rib, lib):
    g = gen(3)
    pages, table = make_cache([64, 64], 1, 64, 16, BF16, g)
    q = torch.randn((2, 2, 64), generator=g).to(BF16).cuda()
    want = rib.paged_decode_attention(q, pages, table, i32([64, 0]), 0.125)
    assert lib.take_device_status() == 0
    got = rib.paged_decode_attention(q, pages, table, i32([65, -3]), 0.125)
    assert lib.take_device_status() == lib.RIB_ECAPACITY
    assert torch.equal(got, want)


def test_attention_missing_page_is_reported(rib, lib):
    g = gen(4)
    pages, table = make_cache([64, 48], 1, 64, 16, BF16, g)
    q = torch.randn((2, 2, 64), generator=g).to(BF16).cuda()
    want = rib.paged_decode_attention(q, pages, table, i32([64, 48]), 0.125)
    for bad in (-1, pages.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[1, 1] = bad
        got = rib.paged_decode_attention(q, pages, t, i32([64, 48]), 0.125)
        assert lib.take_device_status() == lib.RIB_EINVAL
        assert torch.equal(got[0], want[0]) and torch.isfinite(got[1]).all()


def test_attention_strided_inputs(rib, lib):
    """q as a view of a projection, one layer of a pool, a table inside a wider one, a shared page."""
    g = gen(5)
    lens, nkv, D = [70, 33], 2, 128
    pages, table = make_cache(lens, nkv, D, 16, BF16, g)
    pool = torch.full((pages.shape[0], 3, 2, nkv, 16, 2 * D), math.nan, dtype=BF16, device="cuda")
    pool[:, 1, ..., :D] = pages
    table[1, 0] = table[0, 0]  # two sequences share their first page
    wide = torch.full((2, 11), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + table.shape[1]] = table
    qkv = torch.randn((2, 8 * D), generator=g).to(BF16).cuda()
    q = qkv[:, :4 * D].view(2, 4, D)
    got = rib.paged_decode_attention(q, pool[:, 1, ..., :D], wide[:, 3:3 + table.shape[1]], i32(lens), 0.09)
    want, _, bound, _ = attend64(q, pages, table, lens, 0.09)
    close(got, want, bound)
    assert lib.take_device_status() == 0


def test_attention_beyond_32_bit_offsets(rib, lib):
    """Pages whose first value lies past 2^31 values (4 GB) from the pool's start."""
    g = gen(6)
    pages, table = make_cache([100, 37], 2, 128, 64, BF16, g)
    far = (1 << 31) // pages[0].numel() + 5
    pool = torch.empty((far + pages.shape[0], *pages.shape[1:]), dtype=BF16, device="cuda")
    pool[far:] = pages
    q = torch.randn((2, 4, 128), generator=g).to(BF16).cuda()
    want = rib.paged_decode_attention(q, pages, table, i32([100, 37]), 0.09)
    assert torch.equal(rib.paged_decode_attention(q, pool, (table + (table >= 0) * far).int(), i32([100, 37]), 0.09), want)
    # and the append and the eviction there
    rot = rib.Rotary(128)
    kv = torch.randn((2, 2, 128), generator=g).to(BF16).cuda()
    rib.paged_append(q, kv, kv, i32([5, 6]), i32([99, 36]), pages, table, rot)
    rib.paged_append(q, kv, kv, i32([5, 6]), i32([99, 36]), pool, (table + (table >= 0) * far).int(), rot)
    assert torch.equal(pool[far:].nan_to_num(), pages.nan_to_num())
    scores = torch.rand((2, 2, 128), generator=g).cuda()
    free = [p for p in range(pages.shape[0]) if p not in table.tolist()[0] + table.tolist()[1]][:2]
    new = i32([[free[0]], [free[1]]])
    for t, pg, nt in ((table, pages, new), ((table + (table >= 0) * far).int(), pool, new + far)):
        rows, n = rib.paged_evict(pg, t, i32([100, 37]), scores, 40, nt, sinks=2, recent=5)
        assert n.tolist() == [40, 37]
    assert torch.equal(pool[far:].nan_to_num(), pages.nan_to_num())
    assert lib.take_device_status() == 0


def test_attention_same_bits_every_time_and_on_every_stream(rib, lib):
    """Results depend on nothing but the inputs: two streams at once, each with scratch of its own."""
    g = gen(7)
    lens = [3000, 1, 0, 700, 2049]
    pages, table = make_cache(lens, 2, 128, 16, BF16, g)
    q = torch.randn((5, 8, 128), generator=g).to(BF16).cuda()
    want = rib.paged_decode_attention(q, pages, table, i32(lens), 0.09)
    L = i32(lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(rib.paged_decode_attention(q, pages, table, L, 0.09))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_capture_and_replay(rib, lib):
    """A captured decode step (append, attention with scores) replays with what its buffers hold, and
    two graphs captured one after the other run at the same time on two streams."""
    g = gen(8)
    nq, nkv, D, B = 4, 2, 128, 3
    lens = [30, 500, 64]
    rot = rib.Rotary(D)

    def build(seed):
        s = gen(seed)
        pages, table = make_cache([n + 8 for n in lens], nkv, D, 16, BF16, s, fill=0.0)
        st = dict(pages=pages, table=table, qkv=torch.zeros((B, (nq + 2 * nkv) * D), dtype=BF16, device="cuda"),
                  pos=i32(lens), n=i32([x + 1 for x in lens]),
                  scores=torch.zeros((B, nkv, table.shape[1] * 16), device="cuda"))
        return st

    def step(st):
        q, k, v = (x.view(B, -1, D) for x in st["qkv"].split([nq * D, nkv * D, nkv * D], 1))
        q = rib.paged_append(q, k, v, st["pos"], st["pos"], st["pages"], st["table"], rot)
        out = rib.paged_decode_attention(q, st["pages"], st["table"], st["n"], 0.09, scores=st["scores"])
        st["pos"].add_(1)
        st["n"].add_(1)
        return out

    eager, captured = [build(1), build(2)], [build(1), build(2)]
    inputs = [torch.randn((B, (nq + 2 * nkv) * D), generator=g).to(BF16).cuda() for _ in range(4)]
    want = []
    for i, st in enumerate(eager):
        want.append([])
        for x in inputs:
            st["qkv"].copy_(x)
            want[i].append(step(st).clone())
    graphs, outs = [], []
    for st in captured:
        graph = torch.cuda.CUDAGraph()
        keep = {k: st[k].clone() for k in ("pages", "pos", "n", "scores")}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(st)
        torch.cuda.current_stream().wait_stream(side)
        for k, t in keep.items():
            st[k].copy_(t)
        with torch.cuda.graph(graph):
            outs.append(step(st))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for x in inputs:
        for i, st in enumerate(captured):
            with torch.cuda.stream(streams[i]):
                st["qkv"].copy_(x)
                graphs[i].replay()
                got[i].append(outs[i].clone())
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(got[i], want[i]):
            assert torch.equal(a, b)
        assert torch.equal(captured[i]["scores"], eager[i]["scores"])
        assert torch.equal(captured[i]["pages"], eager[i]["pages"])
    assert lib.take_device_status() == 0


# ------------------------------------------------------------------ eviction
def check_evict(rib, lib, lens, *, nkv, D, page_rows, dtype, keep, sinks, recent, scores=None, seed=0, extra=0):
    g = gen(seed)
    B = len(lens)
    new_need = [-(-min(n, keep) // page_rows) for n in lens]
    pages, table = make_cache(lens, nkv, D, page_rows, dtype, g, spare=sum(new_need) + 1, fill=0.5)
    free = sorted(set(range(pages.shape[0])) - set(table.flatten().tolist()))
    width = max(1, -(-keep // page_rows))
    new_table = torch.full((B, width), -1, dtype=torch.int32)
    for b, m in enumerate(new_need):
        for i in range(m):
            new_table[b, i] = free.pop()
    new_table = new_table.cuda()
    room = table.shape[1] * page_rows
    if scores is None:
        scores = torch.rand((B, nkv, room), generator=g).cuda()
    new_scores = torch.full((B, nkv, keep + extra), 9.0, device="cuda")
    before, old_scores = pages.clone(), scores.clone()
    rows, new_lens = rib.paged_evict(pages, table, i32(lens), scores, keep, new_table, sinks=sinks, recent=recent,
                                     new_scores=new_scores)
    assert lib.take_device_status() == 0
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    want = before.clone()
    host = scores.cpu()
    for b, n in enumerate(lens):
        for h in range(nkv):
            kept = kept_rows(host[b, h], n, keep, sinks, recent)
            assert rows[b, h].tolist() == kept + [-1] * (keep - len(kept)), (b, h)
            src = torch.tensor(kept, dtype=torch.long, device="cuda")
            dst = torch.arange(len(kept), device="cuda")
            want[new_table[b, dst // page_rows].long(), :, h, dst % page_rows] = \
                before[table[b, src // page_rows].long(), :, h, src % page_rows]
            assert torch.equal(new_scores[b, h, :len(kept)].nan_to_num(-3), scores[b, h, src].nan_to_num(-3))
            assert (new_scores[b, h, len(kept):] == 0).all()
    assert torch.equal(pages, want)  # the old pages, and rows behind the kept ones, are as they were
    assert torch.equal(scores.nan_to_num(-3), old_scores.nan_to_num(-3))
    return rows


@pytest.mark.parametrize("dtype,D,nkv,page_rows", [(BF16, 128, 2, 16), (FP16, 64, 3, 32), (BF16, 64, 1, 48)])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (40, 4, 8), (40, 20, 20), (100, 0, 99),
                                               (64, 3, 0)])
def test_evict(rib, lib, dtype, D, nkv, page_rows, keep, sinks, recent):
    check_evict(rib, lib, [0, 1, keep, keep + 1, 300, 7], nkv=nkv, D=D, page_rows=page_rows, dtype=dtype, keep=keep,
                sinks=sinks, recent=recent, extra=5)


@pytest.mark.parametrize("n,keep", [(1000, 300), (1900, 1899), (5000, 1234), (20001, 20000), (33000, 700), (280000, 1000)])
def test_evict_long(rib, lib, n, keep):
    check_evict(rib, lib, [n, n // 3], nkv=2, D=64, page_rows=64, dtype=BF16, keep=keep, sinks=4, recent=keep // 8)


def test_evict_many_heads(rib, lib):
    """More (sequence, head) pairs than fit the GPU at once, of up to 1024 and up to 2048 rows."""
    for high in (700, 1500):
        check_evict(rib, lib, [high - 3 * b for b in range(100)], nkv=7, D=64, page_rows=64, dtype=BF16, keep=128, sinks=1,
                    recent=16)


def test_evict_ties_infinities_and_nan(rib, lib):
    """Equal scores go by the lower row, infinities rank as values, NaN lowest, -0 as 0."""
    B, nkv, n = 6, 2, 160
    s = torch.zeros((B, nkv, n))
    s[1] = 1.0
    s[2] = torch.arange(n) % 3
    s[3] = torch.tensor([math.inf, -math.inf, 0.0, math.nan, -0.0, 5.0, -5.0, 1e-45]).repeat(n // 8)
    s[4] = math.nan
    s[5] = -torch.arange(n).float() * 1e30
    s[:, 1] = s[:, 1].flip(-1)
    for keep, sinks, recent in [(50, 3, 7), (81, 0, 0), (100, 1, 1), (159, 0, 0)]:
        check_evict(rib, lib, [n] * B, nkv=nkv, D=64, page_rows=16, dtype=BF16, keep=keep, sinks=sinks, recent=recent,
                    scores=s.cuda())


def test_evict_keep_beyond_the_table(rib, lib):
    """keep may exceed what any sequence has: every row moves, and the new table holds just those."""
    g = gen(3)
    pages, table = make_cache([40, 16], 2, 64, 16, BF16, g, spare=4, fill=0.0)
    free = sorted(set(range(pages.shape[0])) - set(table.flatten().tolist()))
    new = i32([[free[0], free[1], free[2]], [free[3], -1, -1]])
    scores = torch.rand((2, 2, 48), generator=g).cuda()
    before = pages.clone()
    rows, n = rib.paged_evict(pages, table, i32([40, 16]), scores, 1000, new)
    assert n.tolist() == [40, 16] and lib.take_device_status() == 0
    assert torch.equal(rows[0, :, :40], torch.arange(40, device="cuda", dtype=torch.int32).expand(2, 40))
    assert (rows[0, :, 40:] == -1).all() and (rows[1, :, 16:] == -1).all()
    for b, m in enumerate((40, 16)):
        at = torch.arange(m, device="cuda")
        assert torch.equal(pages[new[b, at // 16].long(), :, :, at % 16], before[table[b, at // 16].long(), :, :, at % 16])


@pytest.mark.parametrize("make", ["zero_stride", "odd_stride"])
def test_dimensions_of_one_element_have_no_stride(rib, lib, make):
    """One page, one KV head, one token: their strides are never used, whatever they are."""
    g = gen(4)
    base = torch.randn((1, 2, 1, 16, 64), generator=g).to(BF16).cuda()
    odd = 0 if make == "zero_stride" else 3
    pages = base.as_strided(base.shape, (odd, 1024, odd, 64, 1))
    table = i32([0]).as_strided((1, 1), (odd, 1))
    q = torch.randn((1, 2, 64), generator=g).to(BF16).cuda()
    one = q.as_strided((1, 2, 64), (odd, 64, 1))
    want, _, bound, _ = attend64(q, base, i32([[0]]), [9], 0.125)
    close(rib.paged_decode_attention(one, pages, table, i32([9]), 0.125), want, bound)
    rot = rib.Rotary(64)
    k = q[:, :1]
    got = rib.paged_append(one, k, k, i32([5]), i32([9]), pages, table, rot)
    assert torch.equal(got, rib.rotary(q, i32([5]), rot))
    assert torch.equal(base[0, 1, 0, 9], k[0, 0]) and torch.equal(base[0, 0, 0, 9], rib.rotary(k, i32([5]), rot)[0, 0])
    assert lib.take_device_status() == 0


def test_outputs_that_overlap_are_refused(rib, lib):
    g = gen(5)
    pages, table = make_cache([32, 32], 2, 64, 16, BF16, g)
    q = torch.randn((2, 4, 64), generator=g).to(BF16).cuda()
    n = i32([32, 32])
    scores = torch.zeros((2, 2, 64), device="cuda")
    for kw in (dict(scores=scores[..., :40], scores_out=scores[..., 8:48]),
               dict(scores=scores, scores_out=scores[:1, :1].expand(2, 2, 64)), dict(scores_out=scores),
               dict(scores=scores[..., :31]), dict(scores=scores.double()), dict(out=q[:, :2]), dict(max_len=33),
               dict(max_len=0), dict(out=torch.empty((2, 8, 64), dtype=BF16, device="cuda")[:, ::2])):
        with pytest.raises(ValueError):
            rib.paged_decode_attention(q, pages, table, n, 0.125, **kw)
    with pytest.raises(ValueError):
        rib.paged_evict(pages, table, n, scores, 16, table, new_scores=scores[..., 32:])
    with pytest.raises(ValueError):
        rib.paged_append(q, q[:, :2], q[:, :2], n, n, pages[:1].expand(3, -1, -1, -1, -1), table, rib.Rotary(64))
    with pytest.raises(ValueError):
        rib.rotary(q, n, rib.Rotary(64), out=q[:, :1].expand(2, 4, 64))
    for bad in (q.float(), q[..., :32], q.transpose(1, 2), q[0]):
        with pytest.raises(ValueError):
            rib.paged_decode_attention(bad, pages, table, n, 0.125)
    for bad in (table.long(), table[0], table[:1], table[:, :0], table.cpu()):
        with pytest.raises(ValueError):
            rib.paged_decode_attention(q, pages, bad, n, 0.125)
    for bad in (n.long(), n[:1], n.cpu()):
        with pytest.raises(ValueError):
            rib.paged_decode_attention(q, pages, table, bad, 0.125)
    for bad in (pages.float(), pages[:, :1], pages[..., :32], pages[:, :, :, :8], pages[0]):
        with pytest.raises(ValueError):
            rib.paged_decode_attention(q, bad, table, n, 0.125)
    with pytest.raises(ValueError):  # 16-byte alignment
        rib.rotary(torch.zeros(129, dtype=BF16, device="cuda")[1:].view(1, 2, 64), i32([0]), rib.Rotary(64))
    out = rib.paged_decode_attention(q, pages, table, n, 0.125)
    same = q.clone()
    assert rib.paged_decode_attention(same, pages, table, n, 0.125, out=same) is same and torch.equal(same, out)
    assert lib.take_device_status() == 0


@pytest.mark.parametrize("n,keep", [(900, 300), (5000, 700), (70000, 5000)])
def test_evict_captured_and_on_two_streams(rib, lib, n, keep):
    """A captured eviction replays with what its buffers hold, while another runs on its own stream."""
    g = gen(21)
    nkv, D, P = 2, 64, 64

    def state(seed):
        s = gen(seed)
        pages, table = make_cache([n], nkv, D, P, BF16, s, spare=-(-keep // P), fill=0.25)
        free = sorted(set(range(pages.shape[0])) - set(table.flatten().tolist()))
        return dict(pages=pages, table=table, lens=i32([n]), new=i32([free]), kept=torch.zeros((1, nkv, keep), device="cuda"),
                    scores=torch.zeros((1, nkv, table.shape[1] * P), device="cuda"))

    def call(st):
        return rib.paged_evict(st["pages"], st["table"], st["lens"], st["scores"], keep, st["new"], sinks=2, recent=9,
                               new_scores=st["kept"])
    states, graphs, outs = [state(1), state(2)], [], []
    for st in states:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(st)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(st))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(3):
        lens = [n - 7 * step, keep + step]
        inputs = [torch.randn((1, nkv, states[0]["scores"].shape[2]), generator=g).cuda() for _ in states]
        torch.cuda.synchronize()
        for st, graph, stream, x, m in zip(states, graphs, streams, inputs, lens):
            with torch.cuda.stream(stream):
                st["scores"].copy_(x)
                st["lens"].fill_(m)
                graph.replay()
        torch.cuda.synchronize()
        for st, (rows, new_lens), x, m in zip(states, outs, inputs, lens):
            assert new_lens.tolist() == [min(m, keep)]
            for h in range(nkv):
                at = kept_rows(x[0, h].cpu(), m, keep, 2, 9)
                assert rows[0, h].tolist() == at
                at = torch.tensor(at, device="cuda")
                to = torch.arange(keep, device="cuda")
                assert torch.equal(st["pages"][st["new"][0, to // P].long(), :, h, to % P],
                                   st["pages"][st["table"][0, at // P].long(), :, h, at % P])
                assert torch.equal(st["kept"][0, h], x[0, h, at])
    assert lib.take_device_status() == 0


def test_evict_reports_missing_pages(rib, lib):
    g = gen(2)
    pages, table = make_cache([64], 1, 64, 16, BF16, g, spare=2, fill=0.0)
    free = sorted(set(range(pages.shape[0])) - set(table.flatten().tolist()))
    scores = torch.rand((1, 1, 64), generator=g).cuda()
    before = pages.clone()
    rib.paged_evict(pages, table, i32([64]), scores, 32, i32([[free[0], -1]]))
    assert lib.take_device_status() == lib.RIB_ECAPACITY
    pages[free[0]] = before[free[0]]
    assert torch.equal(pages, before)
    rows, n = rib.paged_evict(pages, table, i32([65]), scores, 32, i32([free]))
    assert lib.take_device_status() == lib.RIB_ECAPACITY and n.tolist() == [32]


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype,D,nq,nkv", [(BF16, 128, 4, 2), (FP16, 64, 6, 2)])
def test_decode_with_eviction(rib, lib, dtype, D, nq, nkv):
    """Append, attend and evict as a decode loop runs them, followed row by row in 64 bits: what a head
    attends to after an eviction is exactly the rows that its scores kept."""
    g = gen(11)
    B, page_rows, keep, steps = 2, 16, 24, 60
    rot = rib.Rotary(D)
    pages = torch.zeros((40, 2, nkv, page_rows, D), dtype=dtype, device="cuda")
    free = list(range(40))
    width = 4
    table = [[free.pop()] for _ in range(B)]
    lens, pos = [0] * B, [0] * B
    scores = torch.zeros((B, nkv, width * page_rows), device="cuda")
    model = [[([], [], []) for _ in range(nkv)] for _ in range(B)]  # per head: keys, values, scores in FP64

    def dev(t):
        return i32([r + [-1] * (width - len(r)) for r in t])
    for step in range(steps):
        for b in range(B):
            if lens[b] == len(table[b]) * page_rows:
                table[b].append(free.pop())
        q, k, v = (torch.randn((B, h, D), generator=g).to(dtype).cuda() for h in (nq, nkv, nkv))
        qr = rib.paged_append(q, k, v, i32(pos), i32(lens), pages, dev(table), rot)
        k64, _ = rotate64(k, i32(pos), rot.frequencies, 1.0, D, False)
        lens = [n + 1 for n in lens]
        pos = [p + 1 + (b == 1) for b, p in enumerate(pos)]
        out = rib.paged_decode_attention(qr, pages, dev(table), i32(lens), D ** -0.5, scores=scores)
        for b in range(B):
            for h in range(nkv):
                keys, vals, sc = model[b][h]
                keys.append(k64[b, h].to(dtype).double())
                vals.append(v[b, h].double())
                sc.append(0.0)
                K, V = torch.stack(keys), torch.stack(vals)
                grp = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
                p = torch.softmax(qr[b, grp].double() @ K.T * D ** -0.5, -1)
                # keys here are rounded from 64 bits, in the cache from 32: at most one step apart, so a
                # score is off by at most 2 half steps of sum |q k|, and a weight by twice that
                size = (qr[b, grp].double().abs() @ K.abs().T).amax().item() * D ** -0.5
                e = 2 * 2 * half_step(dtype) * size + 2.0 ** -16
                close(out[b, grp], p @ V, (p @ V.abs()) * e)
                w = p.sum(0)
                sc[:] = [a + x for a, x in zip(sc, w.tolist())]
                got = scores[b, h, :lens[b]].double().cpu()
                assert ((got - torch.tensor(sc, dtype=torch.float64)).abs() <= torch.tensor(sc) * (e + 1e-5)).all()
        if step % 20 == 19 or max(lens) == width * page_rows:
            new = [[free.pop() for _ in range(-(-min(n, keep) // page_rows))] for n in lens]
            kept = torch.zeros_like(scores)
            rows, n = rib.paged_evict(pages, dev(table), i32(lens), scores, keep, dev(new), sinks=2, recent=6,
                                      new_scores=kept)
            for b in range(B):
                for h in range(nkv):
                    at = [r for r in rows[b, h].tolist() if r >= 0]
                    assert at == kept_rows(scores[b, h].cpu(), lens[b], keep, 2, 6)
                    for lst in model[b][h][:2]:
                        lst[:] = [lst[r] for r in at]
                    model[b][h][2][:] = kept[b, h, :len(at)].tolist()
            lens, scores = n.tolist(), kept
            for b in range(B):
                free.extend(table[b])
            table = new
    assert lib.take_device_status() == 0
