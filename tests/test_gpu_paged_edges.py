"""GPU: the paged-cache operators where the other tests do not reach.  Tolerances as in test_gpu_paged.py, or
derived where they are used."""
from __future__ import annotations

import importlib
import math

import pytest
import torch

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
