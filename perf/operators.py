"""Measured cases of the paged-cache operators: appending rotated keys and values to pages, attention of
one new token over pages, and eviction of the rows that gathered the least attention.

Cache pages are [num_pages, 2, kv_heads, page_rows, head_dim] (K, then V); `table` [sequences, pages] names
the pages of each sequence in order, so row r of a sequence lies in page table[s, r // page_rows]."""
import importlib
import math

import torch

own = False  # True: run() calls the framework's operators; False: their plain form

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GOLDEN = 0.6180339887498949
EPS = 1e-6
MOST_BYTES = 4.0e9  # what a drawn case reads and writes, at most


def listed():
    return [
        # one sequence decodes one token far into its context: the call whose latency counts
        _append("append_token", tokens=1, seqs=1, first=32768, nq=16, nkv=8, dim=128, rotary=128,
                page=16, dtype="bf16", norm=True),
        # one decode step of a full batch, angles stretched for a longer context by frequency bands
        _append("append_step", tokens=256, seqs=256, first=5000, nq=16, nkv=8, dim=128, rotary=128, page=64,
                dtype="bf16", norm=True, scaling="yarn", factor=4.0),
        # the prompts of three requests in one call: interleaved pairs over half of the head, no norm
        _append("append_prompts", tokens=4093, seqs=3, first=0, nq=32, nkv=8, dim=128, rotary=64, page=32,
                dtype="fp16", norm=False, interleaved=True),
        # a long prompt, positions compressed
        _append("append_long_prompt", tokens=32768, seqs=1, first=0, nq=16, nkv=8, dim=128, rotary=128, page=256,
                dtype="bf16", norm=True, scaling="linear", factor=2.0),
        # one sequence, short context
        _attend("attend_short", seqs=1, low=513, high=513, nq=16, nkv=8, dim=128, page=16, dtype="bf16"),
        # one sequence, long context: few rows, a long axis to split
        _attend("attend_long", seqs=1, low=32769, high=32769, nq=16, nkv=8, dim=128, page=64, dtype="bf16"),
        # a ragged serving batch that also sums up the weight each row gets (for eviction)
        _attend("attend_ragged_scores", seqs=64, low=512, high=4096, nq=16, nkv=8, dim=128, page=16, dtype="bf16",
                scores=True),
        # eight query heads share a KV head
        _attend("attend_grouped", seqs=32, low=8191, high=8191, nq=64, nkv=8, dim=128, page=32, dtype="fp16"),
        # the largest batch: more cache than anything else in the step, small heads, pages of 128 rows
        _attend("attend_large", seqs=64, low=30011, high=32768, nq=16, nkv=8, dim=64, page=128, dtype="bf16"),
        # one sequence drops half of its rows
        _evict("evict_one", seqs=1, low=4097, high=4097, nkv=8, dim=128, page=16, dtype="bf16", keep=2048, sinks=4,
               recent=256),
        # a ragged batch, some of whose sequences are short enough to keep every row
        _evict("evict_ragged", seqs=32, low=300, high=8192, nkv=8, dim=128, page=32, dtype="fp16", keep=1024,
               sinks=4, recent=128),
        # long contexts cut to a quarter
        _evict("evict_long", seqs=8, low=65536, high=65536, nkv=8, dim=128, page=64, dtype="bf16", keep=16384,
               sinks=16, recent=1024),
    ]


def _append(name, *, tokens, seqs, first, nq, nkv, dim, rotary, page, dtype, norm, interleaved=False, scaling="",
            factor=1.0):
    return {"name": name, "op": "append", "tokens": tokens, "seqs": seqs, "first": first, "nq": nq, "nkv": nkv,
            "dim": dim, "rotary": rotary, "page": page, "dtype": dtype, "norm": norm, "interleaved": interleaved,
            "scaling": scaling, "factor": factor}


def _attend(name, *, seqs, low, high, nq, nkv, dim, page, dtype, scores=False):
    return {"name": name, "op": "attend", "seqs": seqs, "low": low, "high": high, "nq": nq, "nkv": nkv, "dim": dim,
            "page": page, "dtype": dtype, "scores": scores}


def _evict(name, *, seqs, low, high, nkv, dim, page, dtype, keep, sinks, recent):
    return {"name": name, "op": "evict", "seqs": seqs, "low": low, "high": high, "nkv": nkv, "dim": dim,
            "page": page, "dtype": dtype, "keep": keep, "sinks": sinks, "recent": recent}


def _spread(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "attend", "evict"])
        nkv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 6, 8])
        same = {"nkv": nkv, "dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
                "dtype": rng.choice(["bf16", "fp16"])}
        if op == "append":
            tokens = _spread(rng, 1, 40000)
            step = tokens <= 512 and rng.random() < 0.6
            scaling = rng.choice(["", "linear", "ntk", "yarn"])
            case = _append("", tokens=tokens, seqs=tokens if step else min(tokens, rng.randint(1, 8)),
                           first=_spread(rng, 1, 100000) - 1, nq=nkv * group,
                           rotary=rng.choice([same["dim"], same["dim"], same["dim"] // 2, 48]),
                           norm=rng.random() < 0.5, interleaved=rng.random() < 0.4, scaling=scaling,
                           factor=rng.choice([2.0, 4.0, 8.0]) if scaling else 1.0, **same)
        else:
            high = _spread(rng, 1 if op == "attend" else 64, 70000)
            low = rng.choice([high, max(1, round(high * rng.uniform(0.05, 1.0)))])
            seqs = _spread(rng, 1, 96)
            if op == "attend":
                case = _attend("", seqs=seqs, low=low, high=high, nq=nkv * group, scores=rng.random() < 0.4, **same)
            else:
                keep = max(8, round(high * rng.uniform(0.1, 0.9)))
                sinks = rng.choice([0, 1, 4])
                case = _evict("", seqs=seqs, low=low, high=high, keep=keep, sinks=sinks,
                              recent=rng.randint(0, (keep - sinks) // 2), **same)
        del case["name"]
        if work(case)["bytes"] <= MOST_BYTES:
            return case


def _lens(case):
    """Sequence lengths: spread evenly over [low, high] in a mixed order, the same for every seed."""
    low, high = case["low"], case["high"]
    return [high if b == 0 else low + int((b * GOLDEN % 1.0) * (high - low + 1)) for b in range(case["seqs"])]


def _shares(case):
    """How many of an append's tokens each sequence gets; its first one goes to row `first`."""
    share = -(-case["tokens"] // case["seqs"])
    return [max(0, min(share, case["tokens"] - b * share)) for b in range(case["seqs"])]


def work(case):
    item, dim, nkv = 2, case["dim"], case["nkv"]
    if case["op"] == "append":
        heads = case["tokens"] * (case["nq"] + 2 * nkv)
        table = sum((case["first"] + n - 1) // case["page"] - case["first"] // case["page"] + 1
                    for n in _shares(case) if n)
        weights = 2 * dim * item if case["norm"] else 0
        return {"bytes": 2 * heads * dim * item + 12 * case["tokens"] + 4 * table + weights,
                "flops": 3 * case["tokens"] * (case["nq"] + nkv) * case["rotary"]}
    lens = _lens(case)
    if case["op"] == "attend":
        rows = sum(lens) * nkv
        table = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": rows * 2 * dim * item + 2 * len(lens) * case["nq"] * dim * item + 4 * table + 4 * len(lens)
                + (8 * rows if case["scores"] else 0),
                "flops": 4 * sum(lens) * case["nq"] * dim}
    kept = sum(min(n, case["keep"]) for n in lens) * nkv
    table = sum(-(-n // case["page"]) for n in lens) + sum(-(-min(n, case["keep"]) // case["page"]) for n in lens)
    out = len(lens) * nkv * case["keep"] * 8  # the kept rows' numbers and scores
    return {"bytes": 4 * nkv * sum(n for n in lens if n > case["keep"]) + 2 * kept * 2 * dim * item + out + 4 * table
            + 8 * len(lens), "flops": 0}


def _rng(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1_000_003 + 17)
    return g


def _normal(shape, dtype, g):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _cuda(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to("cuda")


def _table(need, width, g, start=0):
    """Pages for need[s] pages of each sequence, in mixed order; -1 where a sequence has none."""
    total = sum(need)
    order = (torch.randperm(total, generator=g, device="cuda") + start).to(torch.int32)
    count = _cuda(need, torch.int64)[:, None]
    at = torch.cumsum(count, 0) - count + torch.arange(width, device="cuda")
    used = torch.arange(width, device="cuda") < count
    return torch.where(used, order[torch.where(used, at, 0)], -1).to(torch.int32).contiguous()


def prepare(case, seed):
    g, dtype = _rng(case, seed), DTYPES[case["dtype"]]
    nkv, dim, page = case["nkv"], case["dim"], case["page"]
    s = {"case": case}
    if case["op"] == "append":
        nq, tokens, shares = case["nq"], case["tokens"], _shares(case)
        # the pages of the rows before `first`, which the call does not touch, are left out
        first = case["first"] // page
        real = [(case["first"] + n - 1) // page + 1 - first if n else 0 for n in shares]
        s["table"] = torch.cat([torch.full((case["seqs"], first), -1, dtype=torch.int32, device="cuda"),
                                _table(real, max(1, max(real)), g)], 1).contiguous()
        s["pages"] = _normal((sum(real), 2, nkv, page, dim), dtype, g)
        # one projection's output, of which q, k and v are views
        qkv = _normal((tokens, (nq + 2 * nkv) * dim), dtype, g)
        s["q"] = qkv[:, :nq * dim].view(tokens, nq, dim)
        s["k"] = qkv[:, nq * dim:(nq + nkv) * dim].view(tokens, nkv, dim)
        s["v"] = qkv[:, (nq + nkv) * dim:].view(tokens, nkv, dim)
        token = torch.arange(tokens, dtype=torch.int32, device="cuda")
        s["seq"], s["row"] = token // shares[0], case["first"] + token % shares[0]
        s["pos"] = s["row"]
        s["qw"] = s["kw"] = None
        if case["norm"]:
            s["qw"] = (1 + 0.1 * _normal((dim,), torch.float32, g)).to(dtype)
            s["kw"] = (1 + 0.1 * _normal((dim,), torch.float32, g)).to(dtype)
        if own:
            rib = importlib.import_module("roofline-inference_b200")
            s["rib"] = rib
            s["rotary"] = rib.Rotary(dim, 1e6, rotary_dim=case["rotary"], interleaved=case["interleaved"],
                                     scaling=case["scaling"] or None, factor=case["factor"], original_length=32768,
                                     device="cuda")
        return s
    lens = _lens(case)
    need = [-(-n // page) for n in lens]
    width = max(need)
    s["lens"], s["table"] = _cuda(lens), _table(need, width, g)
    if own:
        s["rib"] = importlib.import_module("roofline-inference_b200")
    if case["op"] == "attend":
        s["pages"] = _normal((sum(need) + 1, 2, nkv, page, dim), dtype, g)
        s["q"] = _normal((len(lens), case["nq"], dim), dtype, g)
        s["scale"] = dim ** -0.5
        s["scores"] = s["scores_out"] = None
        if case["scores"]:
            s["scores"] = torch.empty((len(lens), nkv, width * page), device="cuda").exponential_(generator=g)
            s["scores_out"] = torch.zeros_like(s["scores"])
        return s
    # an eviction moves the kept rows to pages of their own; the old pages are free afterwards
    kept = [-(-min(n, case["keep"]) // page) for n in lens]
    s["new_table"] = _table(kept, max(kept), g, start=sum(need))
    s["pages"] = _normal((sum(need) + sum(kept), 2, nkv, page, dim), dtype, g)
    # accumulated weights have a heavy tail, and rows that never got any are equal
    shape = (len(lens), nkv, width * page)
    scores = torch.empty(shape, device="cuda").normal_(generator=g).mul_(2.5).exp_()
    s["scores"] = scores.mul_(torch.rand(shape, generator=g, device="cuda") > 0.1)
    s["new_scores"] = torch.zeros((len(lens), nkv, case["keep"]), device="cuda")
    return s


def run(state):
    op = state["case"]["op"]
    if op == "append":
        return _run_append(state)
    return _run_attend(state) if op == "attend" else _run_evict(state)


def _frequencies(case):
    """Radians a position for each rotated pair, and the factor on cosine and sine."""
    dim, base, factor, length = case["rotary"], 1e6, case["factor"], 32768
    i = torch.arange(0, dim, 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk":
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-i / dim)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] != "yarn":
        return f, 1.0
    # pairs that turn less than once over the original length are stretched, those that turn often are not
    edge = [dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), dim - 1)
    ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rotated(x, cos, sin, case):
    r = case["rotary"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([c, d], -1).flatten(-2) if case["interleaved"] else torch.cat([c, d], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _run_append(s):
    if own:
        q = s["rib"].paged_append(s["q"], s["k"], s["v"], s["pos"], s["row"], s["pages"], s["table"], s["rotary"],
                                  seq=s["seq"], qw=s["qw"], kw=s["kw"])
        return {"q": q, "pages": s["pages"]}
    case, dtype = s["case"], s["q"].dtype
    freq, mag = _frequencies(case)
    angle = s["pos"].double()[:, None] * freq  # positions go far: 32 bits would lose the angle
    cos, sin = (angle.cos() * mag).float()[:, None], (angle.sin() * mag).float()[:, None]
    q = _rotated(_normed(s["q"], s["qw"]), cos, sin, case).to(dtype)
    k = _rotated(_normed(s["k"], s["kw"]), cos, sin, case).to(dtype)
    page = s["table"][s["seq"].long(), (s["row"] // case["page"]).long()].long()
    slot = (s["row"] % case["page"]).long()
    s["pages"][page, 0, :, slot] = k
    s["pages"][page, 1, :, slot] = s["v"]
    return {"q": q, "pages": s["pages"]}


def _run_attend(s):
    case = s["case"]
    if own:
        out = s["rib"].paged_decode_attention(s["q"], s["pages"], s["table"], s["lens"], s["scale"],
                                              scores=s["scores"], scores_out=s["scores_out"])
        return {"out": out, "scores": s["scores_out"]} if case["scores"] else {"out": out}
    seqs, nkv, dim = case["seqs"], case["nkv"], case["dim"]
    kv = s["pages"][s["table"].clamp(min=0).long()]                       # [B, pages, 2, nkv, page, dim]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, seqs, nkv, -1, dim)
    q = s["q"].float().view(seqs, nkv, -1, dim)
    live = torch.arange(kv.shape[3], device="cuda") < s["lens"][:, None]
    logits = torch.matmul(q, kv[0].float().transpose(-1, -2)) * s["scale"]
    logits = torch.where(live[:, None, None], logits, -math.inf)
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, kv[1].float()).view(seqs, -1, dim).to(s["q"].dtype)
    if not case["scores"]:
        return {"out": out}
    s["scores_out"].copy_(torch.where(live[:, None], s["scores"] + p.sum(2), s["scores_out"]))
    return {"out": out, "scores": s["scores_out"]}


def _run_evict(s):
    case, keep = s["case"], s["case"]["keep"]
    if own:
        rows, lens = s["rib"].paged_evict(s["pages"], s["table"], s["lens"], s["scores"], keep, s["new_table"],
                                          sinks=case["sinks"], recent=case["recent"], new_scores=s["new_scores"])
        return {"rows": rows, "lens": lens, "scores": s["new_scores"], "pages": s["pages"]}
    page, table = case["page"], s["table"].long()
    lens = s["lens"].long()[:, None, None]
    n = s["scores"].shape[2]
    at = torch.arange(n, device="cuda")
    score = torch.where((at < case["sinks"]) | (at >= lens - case["recent"]), math.inf, s["scores"])
    score = torch.where(at < lens, score, -1.0)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]  # ties: the lowest row
    best = torch.where(torch.arange(best.shape[2], device="cuda") < lens, best, n)
    rows = torch.sort(best, dim=-1).values
    rows = torch.cat([rows, rows.new_full((*rows.shape[:2], keep - rows.shape[2]), n)], -1)
    live = rows < n
    src = torch.where(live, rows, 0)
    s["new_scores"].copy_(torch.where(live, s["scores"].gather(2, src), 0.0))
    old = table.gather(1, (src // page).flatten(1)).view_as(src)
    to = torch.arange(keep, device="cuda")
    new = s["new_table"].long()[:, (to // page).clamp(max=s["new_table"].shape[1] - 1)]
    b, h, j = live.nonzero(as_tuple=True)
    s["pages"][new[b, j], :, h, to[j] % page] = s["pages"][old[b, h, j], :, h, (src % page)[b, h, j]]
    return {"rows": torch.where(live, rows, -1).to(torch.int32), "lens": s["lens"].clamp(max=keep),
            "scores": s["new_scores"], "pages": s["pages"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    return _exact_attend(case, s) if case["op"] == "attend" else _exact_evict(case, s)


def _exact_append(case, s):
    rot, half = case["rotary"], case["rotary"] // 2
    base = 1e6 * (case["factor"] ** (rot / (rot - 2)) if case["scaling"] == "ntk" else 1.0)
    speeds, gain = [], 1.0
    for i in range(half):
        w = math.exp(-2 * i / rot * math.log(base))
        if case["scaling"] == "linear":
            w /= case["factor"]
        elif case["scaling"] == "yarn":
            turns = lambda t: rot * math.log(32768 / (t * math.tau)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), rot - 1)
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            w = w * (1 - part) + w / case["factor"] * part
            gain = 1.0 + math.log(case["factor"]) / 10
        speeds.append(w)
    turn = torch.polar(torch.tensor(gain, dtype=torch.float64, device="cuda"),
                       torch.outer(s["pos"].double(), torch.tensor(speeds, dtype=torch.float64, device="cuda")))

    def turned(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["dim"] + EPS) * w.double()
        z = y.clone()
        first = slice(0, rot, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, rot, 2) if case["interleaved"] else slice(half, rot)
        c = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn[:, None]
        z[..., first], z[..., second] = c.real, c.imag
        return z

    pages = s["pages"].double()
    k = turned(s["k"], s["kw"])
    flat = pages.permute(0, 3, 1, 2, 4).reshape(-1, 2, case["nkv"], case["dim"])  # a copy: row by row
    row = s["row"].long()
    at = torch.div(row, case["page"], rounding_mode="floor")
    at = s["table"][s["seq"].long(), at].long() * case["page"] + row % case["page"]
    flat[at] = torch.stack([k, s["v"].double()], 1)
    pages = flat.view(-1, case["page"], 2, case["nkv"], case["dim"]).permute(0, 2, 3, 1, 4)
    return {"q": turned(s["q"], s["qw"]), "pages": pages}


def _exact_attend(case, s):
    outs, sums, nkv = [], None, case["nkv"]
    if case["scores"]:
        sums = s["scores_out"].double()
    for b, n in enumerate(_lens(case)):
        used = s["table"][b, :-(-n // case["page"])].long()
        rows = s["pages"][used].double().transpose(0, 2)                   # [nkv, 2, pages, page, dim]
        rows = rows.transpose(0, 1).reshape(2, nkv, -1, case["dim"])[:, :, :n]
        q = s["q"][b].double().view(nkv, -1, case["dim"])
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, rows[0]) / math.sqrt(case["dim"]), -1)
        outs.append(torch.einsum("hgn,hnd->hgd", p, rows[1]).reshape(-1, case["dim"]))
        if sums is not None:
            sums[b, :, :n] = s["scores"][b, :, :n].double() + p.sum(1)
    out = {"out": torch.stack(outs)}
    if sums is not None:
        out["scores"] = sums
    return out


def _exact_evict(case, s):
    nkv, keep, page, lens = case["nkv"], case["keep"], case["page"], _lens(case)
    rows = torch.full((len(lens), nkv, keep), -1, dtype=torch.int32, device="cuda")
    scores = torch.zeros((len(lens), nkv, keep), dtype=torch.float64, device="cuda")
    pages = s["pages"].clone()
    for b, n in enumerate(lens):
        for h in range(nkv):
            mine = s["scores"][b, h, :n]
            kept = torch.arange(n, device="cuda")
            if n > keep:
                middle = mine[case["sinks"]:n - case["recent"]]
                order = torch.argsort(-middle, stable=True)[:keep - case["sinks"] - case["recent"]]
                mark = torch.ones(n, dtype=torch.bool, device="cuda")
                mark[case["sinks"]:n - case["recent"]] = False
                mark[order + case["sinks"]] = True
                kept = mark.nonzero()[:, 0]
            m = kept.numel()
            rows[b, h, :m], scores[b, h, :m] = kept.int(), mine[kept].double()
            to = torch.arange(m, device="cuda")
            source = s["pages"][s["table"][b, kept // page].long(), :, h, kept % page]
            pages[s["new_table"][b, to // page].long(), :, h, to % page] = source
    return {"rows": rows, "lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32), "scores": scores,
            "pages": pages}
