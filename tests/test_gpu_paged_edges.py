"""GPU: the paged-cache operators where the other tests do not reach.  Tolerances as in test_gpu_paged.py, or
derived where they are used."""
from __future__ import annotations

import importlib
import math

import pytest
import torch

from paged_ref import attend64, half_step, make_cache, smallest_half

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
