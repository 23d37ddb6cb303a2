"""The paged-cache operators from their definitions, in 64 bits, for the tests of the kernels."""
from __future__ import annotations

import math

import torch


def half_step(dtype) -> float:
    """A rounding to `dtype` is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def smallest_half(dtype) -> float:
    """... and by at most this where the value is subnormal (half the smallest step)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rotate64(x, pos, freq, gain, rotary_dim, interleaved, w=None, eps=1e-6):
    """(rotated x, the sum |a| + |b| of each element's pair) in FP64; freq in radians per position."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    r = rotary_dim
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    ang = pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = (ang.cos() * gain)[:, None], (ang.sin() * gain)[:, None]
    z, size = y.clone(), y.abs()
    a, b = y[..., first], y[..., second]
    z[..., first], z[..., second] = a * c - b * s, a * s + b * c
    pair = (a.abs() + b.abs()) * gain
    size[..., first], size[..., second] = pair, pair
    return z, size


def rows_of(pages, table_row, n):
    """K, V [nkv, n, D] of one sequence's first n rows, in FP64."""
    page_rows = pages.shape[3]
    used = table_row[:-(-n // page_rows)].long()
    kv = pages[used].double().permute(1, 2, 0, 3, 4)           # [2, nkv, pages, page_rows, D]
    kv = kv.reshape(2, pages.shape[2], -1, pages.shape[4])[:, :, :n]
    return kv[0], kv[1]


def attend64(q, pages, table, lens, scale):
    """(out [B, nq, D], weights as a list of [nkv, n], error bound of out without its last rounding,
    relative error bound of a weight) in FP64.

    The bounds are sums of the roundings that an FP32 kernel makes: a score is a sum of D products,
    each addition off by at most 2^-23 of the sum of the |q k| (the tensor cores may truncate), so a
    weight is off by twice that (score and maximum), the exponential by 2^-22, the weight entering P.V
    by 2^-17 (two BF16 parts), and a sum over n weights, added 16 at a time, by 2^-23 a step."""
    B, nq, D = q.shape
    nkv = pages.shape[2]
    out = torch.zeros((B, nq, D), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    weights, rel = [], []
    for b, n in enumerate(lens):
        if n == 0:
            weights.append(torch.zeros((nkv, 0), dtype=torch.float64, device=q.device))
            rel.append(0.0)
            continue
        K, V = rows_of(pages, table[b], n)
        qb = q[b].double().view(nkv, nq // nkv, D)
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", qb, K) * scale, -1)
        size = torch.einsum("hgd,hnd->hgn", qb.abs(), K.abs()).amax().item() * scale
        e = 2 * size * (D + 2) * 2.0 ** -23 + 2.0 ** -17 + 2.0 ** -22 + 2 * (n / 16 + 40) * 2.0 ** -23
        out[b] = torch.einsum("hgn,hnd->hgd", p, V).reshape(nq, D)
        bound[b] = torch.einsum("hgn,hnd->hgd", p, V.abs()).reshape(nq, D) * e
        weights.append(p.sum(1))
        rel.append(e)
    return out, weights, bound, rel


def kept_rows(scores, n, keep, sinks, recent):
    """Rows that one KV head keeps of its n, from the definition."""
    if n <= keep:
        return list(range(n))
    val = [(-math.inf if math.isnan(v) else v) for v in scores[:n].tolist()]
    nan = [math.isnan(v) for v in scores[:n].tolist()]
    middle = sorted(range(sinks, n - recent), key=lambda i: (nan[i], -val[i], i))[:keep - sinks - recent]
    return sorted(list(range(sinks)) + middle + list(range(n - recent, n)))


def make_cache(lens, nkv, D, page_rows, dtype, gen, *, spare=3, width=None, fill=float("nan"), device="cuda"):
    """Pages with normal values in the rows that `lens` names and `fill` everywhere else, and a table
    of pages in mixed order with -1 behind each sequence's last page."""
    need = [-(-n // page_rows) for n in lens]
    width = max(1, max(need)) if width is None else width
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen)
    pages = torch.full((total, 2, nkv, page_rows, D), fill, dtype=dtype)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        for i in range(need[b]):
            page = int(order[at])
            at += 1
            table[b, i] = page
            m = min(page_rows, n - i * page_rows)
            pages[page, :, :, :m] = torch.randn((2, nkv, m, D), generator=gen).to(dtype)
    return pages.to(device), table.to(device)
