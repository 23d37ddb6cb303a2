"""Batched decode of the Qwen3 forward over a paged cache: the paged operators (paged.py) as the decode
path of batch.py's SlotDecoder, with sequences that grow page by page, may run past the trained context
(a scaled Rotary), and may be held to a bounded number of rows by evicting those that gathered the least
attention.

The reference decodes one sequence over one contiguous cache (agent-test/v2/engine.py:33-55, 145-163).

  PagePool(n_layers, n_kv, pages, page_rows)     pages [layers, pages, 2, n_kv, page_rows, 128], free list
  PagedDecoder(engine, pool, slots, max_rows)    decode steps over the slots' sequences
      .add(prompt) -> slot      prefill, pages, first token      .remove(slot)
      .step()                   next greedy token of every slot  .capture()  the step as a CUDA graph
"""
from __future__ import annotations

import torch

from . import _lib
from ._tensors import HEAD_DIM, stream_handle
from .attention import attention
from .batch import _linear as _linear_rows
from .cache import Cache
from .kernels import add_rms, argmax, embedding, gemv, rms_norm
from .model import _linear
from .paged import Rotary, paged_append, paged_decode_attention, paged_evict
from .pool import PoolFull


class PagePool:
    """`pages` pages of `page_rows` rows for every layer, and the list of free ones.  A page number
    names the same place of every layer, so a sequence has one table for all layers."""

    def __init__(self, n_layers: int, n_kv: int, pages: int, page_rows: int = 64, head_dim: int = HEAD_DIM,
                 dtype=torch.bfloat16, device=None):
        if n_layers < 1 or n_kv < 1 or pages < 1:
            raise ValueError("n_layers, n_kv and pages must be positive")
        if page_rows not in (16, 32, 64, 128, 256):
            raise ValueError("page_rows must be 16, 32, 64, 128 or 256")
        self.page_rows, self.n_kv = page_rows, n_kv
        # never read behind a sequence's rows, so the contents need no clearing
        self.storage = torch.empty((n_layers, pages, 2, n_kv, page_rows, head_dim), dtype=dtype, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._used: set[int] = set()

    @classmethod
    def for_engine(cls, engine, pages: int, page_rows: int = 64) -> "PagePool":
        return cls(engine.cfg.num_layers, engine.n_kv, pages, page_rows, device=engine.device)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, i: int) -> torch.Tensor:
        return self.storage[i]

    def pages_for(self, rows: int) -> int:
        return -(-rows // self.page_rows)

    def take(self, n: int) -> list[int]:
        """n free pages; PoolFull (and none taken) when there are fewer."""
        if n > len(self._free):
            raise PoolFull(f"{n} pages wanted, {len(self._free)} free")
        ids = [self._free.pop() for _ in range(n)]
        self._used.update(ids)
        return ids

    def give(self, ids: list[int]) -> None:
        """Returns pages; work on the current stream may still read them, later work reuses them."""
        if len(set(ids)) != len(ids) or not self._used.issuperset(ids):
            raise ValueError("pages that were not taken from this pool (or given back already)")
        self._used.difference_update(ids)
        self._free.extend(reversed(ids))


class PagedDecoder:
    """Decode steps over `slots` sequences of at most `max_rows` cached rows each.

    rotary: the rotation (default: the engine's base, whole head).  keep: with it, a sequence that has
    filled max_rows is cut to its `keep` best rows before the next step (its first `sinks`, its last
    `recent` and those that decode steps gave the most attention, per layer and KV head; a prompt's rows
    start with none, so one that fills max_rows is cut, before its first step, to its lowest rows between
    those); without it such a sequence raises "KV capacity exceeded"."""

    def __init__(self, engine, pool: PagePool, slots: int, max_rows: int, *, rotary: Rotary | None = None,
                 keep: int | None = None, sinks: int = 4, recent: int = 32):
        if engine.world != 1:
            raise ValueError("paged decode runs on one GPU")
        cfg, dev = engine.cfg, engine.device
        if pool.storage.shape[0] != cfg.num_layers or pool.n_kv != engine.n_kv or pool.storage.shape[5] != HEAD_DIM \
                or pool.storage.dtype != torch.bfloat16:
            raise ValueError("the pool does not match the engine's layers / KV heads")
        if pool.storage.device != dev:
            raise ValueError(f"the pool is on {pool.storage.device}, the engine on {dev}")
        if rotary is not None and (rotary.head_dim != HEAD_DIM or rotary.device != dev):
            raise ValueError(f"rotary must rotate heads of {HEAD_DIM} dims on {dev}")
        if slots < 1 or max_rows < 1:
            raise ValueError("need at least one slot and max_rows >= 1")
        if keep is not None and (not 1 <= keep < max_rows or sinks < 0 or recent < 0 or sinks + recent > keep):
            raise ValueError("need 1 <= keep < max_rows, sinks >= 0, recent >= 0 and sinks + recent <= keep")
        self.e, self.pool, self.device, self.B, self.L = engine, pool, dev, slots, _lib.load()
        self.max_rows, self.keep, self.sinks, self.recent = max_rows, keep, sinks, recent
        self.rotary = Rotary(HEAD_DIM, engine.base, device=dev) if rotary is None else rotary
        width = pool.pages_for(max_rows)
        i32 = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((slots, width), -1, **i32)
        self.pos = torch.zeros(slots, **i32)             # position of the next token
        self.row = torch.full((slots,), -1, **i32)       # its cache row; -1: an idle slot, nothing is written
        self.lens = torch.zeros(slots, **i32)            # rows it attends to; 0: an idle slot, zeros
        self.active = torch.zeros(slots, **i32)
        self.tok = torch.zeros(slots, **i32)             # next input tokens
        self.next = torch.empty(slots, **i32)
        self.scores = None
        if keep is not None:
            room = width * pool.page_rows
            self.scores = torch.zeros((cfg.num_layers, slots, engine.n_kv, room), device=dev)
            self._kept = torch.empty((cfg.num_layers, 1, engine.n_kv, room), device=dev)
        self.pages: list[list[int] | None] = [None] * slots   # host side: each slot's pages,
        self.rows = [0] * slots                                 # rows,
        self.positions = [0] * slots                            # and next position
        self.graph = None

    # ---------------------------------------------------------------- membership
    def free_slots(self) -> list[int]:
        return [i for i, p in enumerate(self.pages) if p is None]

    def add(self, prompt: list[int]) -> int:
        """Prefills `prompt` into pages of its own; returns its slot, whose next input (`tok`) is the
        prompt's greedy continuation."""
        free = self.free_slots()
        if not free:
            raise ValueError("no free slot")
        n = len(prompt)
        if not prompt or min(prompt) < 0 or max(prompt) >= self.e.cfg.vocab_size:
            raise ValueError("the prompt needs tokens inside the vocabulary")
        if n > self.max_rows:
            raise ValueError("KV capacity exceeded")
        i, ids = free[0], self.pool.take(self.pool.pages_for(n))
        try:
            first = argmax(self._prefill(torch.tensor(prompt, dtype=torch.int32, device=self.device), ids))
        except BaseException:
            self.pool.give(ids)
            raise
        self.tok[i:i + 1].copy_(first)
        self.pages[i], self.rows[i], self.positions[i] = ids, n, n
        self.table[i].fill_(-1)
        self.table[i, :len(ids)] = torch.tensor(ids, dtype=torch.int32).to(self.device)
        self.active[i] = 1
        self.pos[i] = n
        self._set_rows(i, n)
        if self.scores is not None:
            self.scores[:, i].zero_()
        return i

    def remove(self, i: int) -> None:
        """Slot i goes idle; its pages return to the pool."""
        if self.pages[i] is None:
            raise ValueError(f"slot {i} is idle")
        self.pool.give(self.pages[i])
        self.pages[i] = None
        self.active[i] = 0
        self.pos[i] = 0
        self.row[i] = -1
        self.lens[i] = 0
        self.table[i].fill_(-1)

    def _set_rows(self, i: int, n: int) -> None:
        self.rows[i] = n
        self.row[i] = n
        self.lens[i] = n + 1

    # ---------------------------------------------------------------- prefill
    def _prefill(self, tokens, ids: list[int]):
        """The prompt's forward over one layer's contiguous scratch cache, which is one large page to the append and
        serves every layer in turn: its rows go to the sequence's pages before the next layer's overwrite them.
        Returns the FP32 logits of the last row."""
        e, n, P = self.e, tokens.numel(), self.pool.page_rows
        kv = Cache(1, e.n_kv, HEAD_DIM, n, device=self.device).kv[0]
        pos = torch.arange(n, dtype=torch.int32, device=self.device)
        seq = torch.zeros_like(pos)
        one_page = torch.zeros((1, 1), dtype=torch.int32, device=self.device)
        where = torch.tensor(ids, dtype=torch.int64).to(self.device)
        q = torch.empty((e.nq_local, (n + 31) // 32 * 32, HEAD_DIM), dtype=torch.bfloat16, device=self.device)
        h = embedding(e.embed, tokens)
        x = rms_norm(h, e.layers[0]["in_norm"])
        for l, w in enumerate(e.layers):
            self._append(_linear(x, w["qkv"]), w, pos, pos, kv[None], one_page, seq, q.transpose(0, 1)[:n])
            self.pool.layer(l)[where] = kv.view(2, e.n_kv, -1, P, HEAD_DIM)[:, :, :len(ids)].permute(2, 0, 1, 3, 4)
            o = attention(q, kv[0], kv[1], n, n, e.scale)
            last = l == len(e.layers) - 1
            if last:  # only the final row feeds the logits
                o, h = o[n - 1:], h[n - 1:]
            h, x = add_rms(h, _linear(o, w["o"]), w["post_norm"])
            r = _linear(_linear(x, w["gu"], "swiglu"), w["down"])
            if last:
                h = h + r
            else:
                h, x = add_rms(h, r, e.layers[l + 1]["in_norm"])
        return gemv(e.embed, h.reshape(-1), nw=e.final_norm, out_float=True)

    def _append(self, qkv, w, pos, row, pages, table, seq, out):
        """Norm, rotation and append of the rows of one layer's QKV projection; returns q."""
        nq, nkv = self.e.nq_local, self.e.n_kv
        q, k, v = (t.view(qkv.shape[0], -1, HEAD_DIM)
                   for t in qkv.split([nq * HEAD_DIM, nkv * HEAD_DIM, nkv * HEAD_DIM], 1))
        return paged_append(q, k, v, pos, row, pages, table, self.rotary, seq=seq, qw=w["q_norm"], kw=w["k_norm"],
                            out=out)

    # ---------------------------------------------------------------- the step
    def _forward(self):
        """The device work of one step on the input tokens; returns the FP32 logits [S, vocab].
        Positions, rows and lengths of active slots advance on the device."""
        e, B = self.e, self.B
        h = embedding(e.embed, self.tok)
        x = rms_norm(h, e.layers[0]["in_norm"])
        for l, w in enumerate(e.layers):
            pages = self.pool.layer(l)
            q = self._append(_linear_rows(x, w["qkv"]), w, self.pos, self.row, pages, self.table, None, None)
            o = paged_decode_attention(q, pages, self.table, self.lens, e.scale,
                                       scores=None if self.scores is None else self.scores[l])
            h, x = add_rms(h, _linear_rows(o.view(B, -1), w["o"]), w["post_norm"])
            r = _linear_rows(_linear_rows(x, w["gu"], "swiglu"), w["down"])
            if l == len(e.layers) - 1:
                h = h + r
            else:
                h, x = add_rms(h, r, e.layers[l + 1]["in_norm"])
        out = torch.mm(rms_norm(h, e.final_norm), e.embed.t(), out_dtype=torch.float32)
        for t in (self.pos, self.row, self.lens):
            t.add_(self.active)
        return out

    def _argmax(self, logits):
        _lib.check(self.L.rib_argmax_rows_f32(logits.data_ptr(), self.B, logits.shape[1], self.next.data_ptr(),
                                              stream_handle(self.device)), "argmax_rows")

    def _make_room(self) -> None:
        """Before a step: sequences at max_rows are cut to `keep`, and each gets the page its next row
        needs.  Raises, with nothing changed, when the pool has too few free pages."""
        live = [i for i, p in enumerate(self.pages) if p is not None]
        full = [i for i in live if self.rows[i] == self.max_rows]
        if full and self.keep is None:
            raise ValueError("KV capacity exceeded")
        P = self.pool.page_rows
        growing = [i for i in live if i not in full and self.rows[i] == len(self.pages[i]) * P]
        # what the loops below take and give, in their order: an eviction takes its new pages before it gives the
        # old ones back, which the next eviction, and then the growing sequences, can use
        free = self.pool.free_pages
        wants = self.pool.pages_for(self.keep) if full else 0
        for i in full:
            if wants > free:
                raise PoolFull(f"{wants} pages wanted for an eviction, {free} free")
            free += len(self.pages[i]) - wants
        grow = len(growing) + (len(full) if full and self.keep == wants * P else 0)
        if grow > free:
            raise PoolFull(f"{grow} pages wanted, {free} free")
        for i in full:
            self._evict(i)
            if self.keep == len(self.pages[i]) * P:
                growing.append(i)
        for i in growing:
            page = self.pool.take(1)[0]
            self.table[i, len(self.pages[i])] = page
            self.pages[i].append(page)

    def _evict(self, i: int) -> None:
        ids = self.pool.take(self.pool.pages_for(self.keep))
        new = torch.full_like(self.table[i:i + 1], -1)
        new[0, :len(ids)] = torch.tensor(ids, dtype=torch.int32).to(self.device)
        lens = self.row[i:i + 1]  # rows in the cache: the next token's row
        try:
            for l in range(len(self.e.layers)):
                paged_evict(self.pool.layer(l), self.table[i:i + 1], lens, self.scores[l, i:i + 1], self.keep, new,
                            sinks=self.sinks, recent=self.recent, new_scores=self._kept[l])
        except BaseException:  # the sequence is as it was: its own pages and scores were only read
            self.pool.give(ids)
            raise
        self.scores[:, i:i + 1].copy_(self._kept)
        self.table[i:i + 1].copy_(new)
        self.pool.give(self.pages[i])
        self.pages[i] = ids
        self._set_rows(i, self.keep)

    def _advance_host(self) -> None:
        for i, p in enumerate(self.pages):
            if p is not None:
                self.rows[i] += 1
                self.positions[i] += 1

    def capture(self):
        """Records one step in a CUDA graph; later steps replay it.  Every input of the step lives in a
        fixed buffer (tables, rows, lengths, scores), so the graph serves every membership, every page
        and every eviction.  Captured while no slot is active, so nothing has to be wound back."""
        if any(p is not None for p in self.pages):
            raise ValueError("capture before the first sequence is added")
        dev, stream = self.device, torch.cuda.current_stream(self.device)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(device=dev)
        side.wait_stream(stream)
        with torch.cuda.stream(side):
            self._argmax(self._forward())  # warm-up outside the graph
        stream.wait_stream(side)
        torch.cuda.synchronize(dev)
        with torch.cuda.graph(graph, stream=side):
            self.graph_logits = self._forward()
            self._argmax(self.graph_logits)
            self.tok.copy_(self.next)
        stream.wait_stream(side)
        torch.cuda.synchronize(dev)
        self.graph = graph
        return self

    def step(self) -> torch.Tensor:
        """One step of every active slot on the tokens in `tok`; returns the next greedy tokens (int32
        [slots], the caller's own, which also become the next inputs; idle slots' entries are meaningless)."""
        self._make_room()
        if self.graph is None:
            self._argmax(self._forward())
            self.tok.copy_(self.next)
        else:
            self.graph.replay()
        self._advance_host()
        return self.next.clone()

    def logits(self) -> torch.Tensor:
        """One eager step; returns the FP32 logits [slots, vocab] and leaves `tok` alone."""
        self._make_room()
        out = self._forward()
        self._advance_host()
        return out
