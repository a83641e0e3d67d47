"""Serving over a paged key/value cache.

`PagedKVCache` holds the keys and values of all layers in pages that sequences
take as they grow, share after a fork (the last, partly filled page is copied
when one of them writes on) and give back when they end. `PagedBatchingEngine`
is the scheduler over it: prompts of different lengths are prefilled together in
one packed row without padding, every step decodes one token for each active
sequence at its own position, and no admission waits for the others' length
(ContinuousBatchingEngine shares one write column over a dense cache).

Operators: ops.flash_attention_packed, ops.paged_attention,
ops.paged_kv_append, ops.copy_pages, ops.token_logprobs.
"""

from __future__ import annotations

import heapq
import operator
import threading
from typing import Callable, Dict, List, Optional, Sequence, Tuple

import torch

from .. import ops
from .engine import GenerationConfig, check_tokens, sample_token


class _Step:
    """Where one forward's tokens go, shared by all layers."""

    __slots__ = ("table", "positions", "seq_ids", "lens")

    def __init__(self, table, positions, seq_ids, lens):
        self.table = table
        self.positions = positions
        self.seq_ids = seq_ids
        self.lens = lens


class PagedLayer:
    """One layer of a PagedKVCache for one forward, in the place of a KVCache
    (models/transformer.py)."""

    paged = True
    graph_mode = False
    pos_dev = None

    def __init__(self, k: torch.Tensor, v: torch.Tensor, step: _Step,
                 max_len: int):
        self.k = k
        self.v = v
        self.step = step
        self.max_len = max_len

    @property
    def positions(self) -> torch.Tensor:
        return self.step.positions

    def append(self, k: torch.Tensor, v: torch.Tensor):
        s = self.step
        ops.paged_kv_append(k, v, self.k, self.v, s.table, s.positions,
                            s.seq_ids)

    def attend(self, q: torch.Tensor, scale: float) -> torch.Tensor:
        return ops.paged_attention(q, self.k, self.v, self.step.table,
                                   self.step.lens, scale)


class PagedKVCache:
    """Pages [layers, pages, kv_heads, page_size, width] for keys and values,
    and for each of `max_seqs` slots its page numbers and its length. Tables are
    kept on the host and copied to the device when they change."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int,
                 pages: int, page_size: int = 64, max_seqs: int = 8,
                 max_len: int = 2048, dtype: torch.dtype = torch.bfloat16,
                 device: Optional[torch.device] = None):
        if not 16 <= page_size <= 4096 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to "
                             f"4096, got {page_size}")
        if pages < 1 or max_seqs < 1 or max_len < 1:
            raise ValueError("pages, max_seqs and max_len must be positive")
        self.page_size = page_size
        self.max_len = max_len
        shape = (num_layers, pages, num_kv_heads, page_size,
                 ops.page_width(head_dim))
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.device = self.k.device
        self.lens = [0] * max_seqs
        self.tables: List[List[int]] = [[] for _ in range(max_seqs)]
        self._refs = [0] * pages
        self._free = list(range(pages))
        self._table = torch.zeros(max_seqs, self.pages_for(max_len),
                                  dtype=torch.int32, device=self.device)

    # ------------------------------------------------------------- pages
    @property
    def pages(self) -> int:
        return self.k.shape[1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages_for(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def pages_needed(self, slots: Sequence[int], counts: Sequence[int]) -> int:
        """Pages that counts[i] more tokens of slots[i] take, the copies of
        shared pages that they would write into among them: of k slots that
        share one, the last to write keeps it."""
        need, left = 0, {}
        for slot, count in zip(slots, counts):
            n, table = self.lens[slot], self.tables[slot]
            need += max(0, self.pages_for(n + count) - len(table))
            if count > 0 and n % self.page_size:
                p = table[n // self.page_size]
                left[p] = left.get(p, self._refs[p])
                if left[p] > 1:
                    left[p] -= 1
                    need += 1
        return need

    def extend(self, slots: Sequence[int], counts: Sequence[int]):
        """Makes room for counts[i] more tokens of slots[i]; a shared page that
        would be written into is copied first, all of them in one call. Raises
        before anything changes if there is no room."""
        if len(set(slots)) < len(slots):
            raise ValueError("a slot is named twice")
        if len(slots) != len(counts) or min(counts, default=0) < 0:
            raise ValueError("each slot needs a count of 0 or more")
        for slot, count in zip(slots, counts):
            if self.lens[slot] + count > self.max_len:
                raise ValueError(f"slot {slot} would pass max_len "
                                 f"{self.max_len}")
        if self.pages_needed(slots, counts) > self.free_pages:
            raise MemoryError("the page pool is full")
        src, dst = [], []
        for slot, count in zip(slots, counts):
            table, n = self.tables[slot], self.lens[slot]
            at = n // self.page_size
            shared = (count > 0 and n % self.page_size != 0
                      and self._refs[table[at]] > 1)
            if shared:
                src.append(table[at])
                dst.append(self._take())
                self._drop(table[at])
                table[at] = dst[-1]
            new = max(0, self.pages_for(n + count) - len(table))
            table.extend(self._take() for _ in range(new))
            if new or shared:
                self._upload(slot)
        if src:
            ops.copy_pages([self.k, self.v], src, dst)

    def fork(self, src: int, dst: int):
        """Slot dst continues what slot src holds, on the same pages."""
        if self.tables[dst]:
            raise ValueError(f"slot {dst} is in use")
        # room that was made ahead stays with src: nothing of it is written yet
        self.tables[dst] = self.tables[src][:self.pages_for(self.lens[src])]
        self.lens[dst] = self.lens[src]
        for p in self.tables[dst]:
            self._refs[p] += 1
        self._upload(dst)

    def free(self, slot: int):
        for p in self.tables[slot]:
            self._drop(p)
        self.tables[slot] = []
        self.lens[slot] = 0

    def compact(self) -> int:
        """Moves the live pages to the front of the pool; returns how many."""
        live = [p for p, r in enumerate(self._refs) if r]
        src = [p for p in live if p >= len(live)]
        dst = [p for p in range(len(live)) if not self._refs[p]]
        if not src:
            return 0
        ops.copy_pages([self.k, self.v], src, dst)
        moved = dict(zip(src, dst))
        for a, b in moved.items():
            self._refs[a], self._refs[b] = 0, self._refs[a]
        self._free = list(range(len(live), self.pages))
        for slot, table in enumerate(self.tables):
            if any(p in moved for p in table):
                self.tables[slot] = [moved.get(p, p) for p in table]
                self._upload(slot)
        return len(src)

    def resize(self, pages: int):
        """Grows or shrinks the pool; the live pages are compacted first."""
        live = self.pages - self.free_pages
        if pages < max(live, 1):
            raise ValueError(f"{live} pages are in use, {pages} do not hold "
                             "them")
        self.compact()
        keep = min(pages, self.pages)
        for name in ("k", "v"):
            old = getattr(self, name)
            new = old.new_zeros(old.shape[0], pages, *old.shape[2:])
            new[:, :keep] = old[:, :keep]
            setattr(self, name, new)
        self._refs = self._refs[:keep] + [0] * (pages - keep)
        self._free = list(range(live, pages))

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._refs[p] = 1
        return p

    def _drop(self, p: int):
        self._refs[p] -= 1
        if self._refs[p] == 0:
            heapq.heappush(self._free, p)

    def _upload(self, slot: int):
        t = self.tables[slot]
        if t:
            self._table[slot, :len(t)] = torch.tensor(t, dtype=torch.int32)

    # ------------------------------------------------------------- forwards
    def _layers(self, step: _Step) -> List[PagedLayer]:
        return [PagedLayer(self.k[i], self.v[i], step, self.max_len)
                for i in range(self.k.shape[0])]

    def _int32(self, values: List[int]) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.device)

    def prefill(self, slots: Sequence[int], counts: Sequence[int]
                ) -> Tuple[List[PagedLayer], torch.Tensor]:
        """(kv_caches, cu_seqlens) of a forward over counts[i] tokens of each
        empty slot, packed."""
        if any(self.lens[s] for s in slots):
            raise ValueError("a prompt goes into an empty slot")
        self.extend(slots, counts)
        cu, ids, pos = [0], [], []
        for s, n in zip(slots, counts):
            cu.append(cu[-1] + n)
            ids += [s] * n
            pos += range(n)
            self.lens[s] = n
        step = _Step(self._table, self._int32(pos), self._int32(ids), None)
        return self._layers(step), self._int32(cu)

    def decode(self, slots: Sequence[int]) -> List[PagedLayer]:
        """kv_caches of a forward over one more token of each slot; row i of
        its [len(slots), 1] input belongs to slots[i]."""
        self.extend(slots, [1] * len(slots))
        pos = self._int32([self.lens[s] for s in slots])
        for s in slots:
            self.lens[s] += 1
        rows = torch.tensor(list(slots)).to(self.device)
        step = _Step(self._table.index_select(0, rows), pos, None, pos + 1)
        return self._layers(step)


# tokens of one packed prefill, whose activations and logits are held at once
PREFILL_TOKENS = 32768


class _Slot:
    __slots__ = ("active", "cfg", "stops", "recent", "out", "cb", "done",
                 "result", "logprobs", "error")

    def __init__(self):
        self.active = False
        self.result = None
        self.logprobs = None
        self.error = None

    def start(self, cfg, stops, recent, out, logprobs, cb):
        self.cfg = cfg
        self.stops = stops
        self.recent = recent
        self.out = out
        self.logprobs = logprobs
        self.cb = cb
        self.done = threading.Event()
        self.result = None
        self.error = None
        self.active = True


class PagedBatchingEngine:
    """Iteration-level scheduler over a PagedKVCache, with the interface of
    ContinuousBatchingEngine and forks and log probabilities besides. A slot
    that finds no page for its next token ends with what it has; the default
    pool holds max_batch sequences of max_len. A slot whose next token cannot
    be sampled ends too, with the exception in its `error`; the others go on."""

    def __init__(self, model, tokenizer, max_batch: int = 8,
                 max_len: int = 2048, page_size: int = 64,
                 pages: Optional[int] = None,
                 device: Optional[torch.device] = None):
        p = next(model.parameters())
        self.device = device or p.device
        if self.device.type == "cuda" and p.dtype != torch.bfloat16:
            raise TypeError("paged serving on the GPU needs a bf16 model, got "
                            f"{p.dtype}")
        if model.layers[0].attention.head_dim > 192:
            raise ValueError("paged serving takes head_dim up to 192")
        self.model = model.eval()
        self.tokenizer = tokenizer
        self.max_batch = max_batch
        self.max_len = max_len
        at = model.layers[0].attention
        self.cache = PagedKVCache(
            len(model.layers), at.num_kv_heads, at.head_dim,
            pages or max_batch * -(-max_len // page_size), page_size,
            max_batch, max_len, p.dtype, self.device)
        self.slots = [_Slot() for _ in range(max_batch)]
        self.last_logits: Optional[torch.Tensor] = None
        self._pad = tokenizer.pad_token_id
        self.stats = {"admitted": 0, "finished": 0, "steps": 0,
                      "tokens_out": 0}

    # --------------------------------------------------------------- state
    def n_active(self) -> int:
        return sum(1 for s in self.slots if s.active)

    def free_slots(self) -> List[int]:
        return [i for i, s in enumerate(self.slots) if not s.active]

    def can_admit(self, prompt_len: int, n: int = 1) -> bool:
        """Whether a prompt and n - 1 forks of it fit now, each with room for
        its first token."""
        return self.admissible([(prompt_len, n)]) == 1

    def admissible(self, requests: Sequence[Tuple[int, int]]) -> int:
        """How many of these (prompt length, answers), from the first on, fit
        now and go through one prefill: up to PREFILL_TOKENS, or one prompt."""
        slots, pages, tokens = len(self.free_slots()), self.cache.free_pages, 0
        for i, (length, n) in enumerate(requests):
            slots -= n
            pages -= self._pages_to_admit(length, n)
            tokens += length
            if slots < 0 or pages < 0 or length + 1 > self.max_len or \
                    i and tokens > PREFILL_TOKENS:
                return i
        return len(requests)

    def can_ever_admit(self, prompt_len: int, n: int = 1) -> bool:
        """Whether they fit when nothing else is served."""
        return n <= self.max_batch and prompt_len + 1 <= self.max_len and \
            self._pages_to_admit(prompt_len, n) <= self.cache.pages

    def _pages_to_admit(self, prompt_len: int, n: int) -> int:
        # beside the prompt's, the page that each fork writes into
        return self.cache.pages_for(prompt_len + 1) + n - 1

    # --------------------------------------------------------------- admit
    @torch.no_grad()
    def admit_many(self, prompts: Sequence[List[int]],
                   configs: Optional[Sequence[Optional[GenerationConfig]]]
                   = None,
                   callbacks: Optional[Sequence[Optional[Callable]]] = None
                   ) -> List[int]:
        """Prefills prompts of any lengths in one packed forward; returns their
        slots. The next step() decodes their first tokens."""
        if not prompts:
            return []
        configs = configs or [None] * len(prompts)
        callbacks = callbacks or [None] * len(prompts)
        if min(len(configs), len(callbacks)) < len(prompts):
            raise ValueError(f"{len(prompts)} prompts, {len(configs)} configs "
                             f"and {len(callbacks)} callbacks")
        cfgs = [c or GenerationConfig() for c in configs[:len(prompts)]]
        stops = [self._stops(c) for c in cfgs]
        slots = self.free_slots()[:len(prompts)]
        if len(slots) < len(prompts):
            raise RuntimeError("no free slot — poll can_admit first")
        ids = [p[-min(c.max_context, self.max_len - 1):] or [self._pad]
               for p, c in zip(prompts, cfgs)]
        check_tokens(ids, self.model)
        flat = [t for x in ids for t in x]
        try:
            caches, cu = self.cache.prefill(slots, [len(x) for x in ids])
            logits, _, _ = self.model(
                torch.tensor([flat], dtype=torch.long).to(self.device),
                kv_caches=caches, cu_seqlens=cu)
            last = logits[0].index_select(0, (cu[1:] - 1).long()).float()
            if self.last_logits is None:
                self.last_logits = last.new_zeros(self.max_batch,
                                                  last.shape[-1])
            for i, b in enumerate(slots):
                self.last_logits[b] = last[i]
        except Exception:
            for b in slots:
                self.cache.free(b)
            raise
        for i, b in enumerate(slots):
            self.slots[b].start(cfgs[i], stops[i], list(ids[i]), [], [],
                                callbacks[i])
        self.stats["admitted"] += len(slots)
        return slots

    def _stops(self, cfg: GenerationConfig) -> set:
        """Checks a configuration; the tokens that end its answer."""
        if cfg.logprobs is not None and not (
                isinstance(cfg.logprobs, int) and 0 <= cfg.logprobs <= 64):
            raise ValueError(f"logprobs must be 0 to 64, got {cfg.logprobs}")
        try:
            stops = {operator.index(t) for t in cfg.stop_token_ids}
        except TypeError:
            raise ValueError("stop_token_ids must be whole numbers, got "
                             f"{cfg.stop_token_ids}") from None
        return stops | {self.tokenizer.eos_token_id}

    def admit(self, prompt_ids: List[int],
              cfg: Optional[GenerationConfig] = None,
              stream_callback: Optional[Callable[[int], None]] = None) -> int:
        return self.admit_many([prompt_ids], [cfg], [stream_callback])[0]

    @torch.no_grad()
    def fork(self, slot: int, cfg: Optional[GenerationConfig] = None,
             stream_callback: Optional[Callable[[int], None]] = None) -> int:
        """A further answer that continues slot's text so far, on its pages."""
        src = self.slots[slot]
        if not src.active:
            raise ValueError(f"slot {slot} is not active")
        free = self.free_slots()
        if not free:
            raise RuntimeError("no free slot — poll can_admit first")
        b = free[0]
        cfg = cfg or src.cfg
        stops = self._stops(cfg)
        self.last_logits[b] = self.last_logits[slot]
        self.cache.fork(slot, b)
        self.slots[b].start(cfg, stops, list(src.recent), list(src.out),
                            list(src.logprobs), stream_callback)
        self.stats["admitted"] += 1
        return b

    # ---------------------------------------------------------------- step
    @torch.no_grad()
    def step(self) -> List[int]:
        """Samples one token for every active slot and decodes them all in one
        forward. Returns the slots that finished."""
        finished: List[int] = []
        tok_of: Dict[int, int] = {}
        for b, s in enumerate(self.slots):
            if not s.active:
                continue
            try:
                nid = sample_token(self.last_logits[b].clone(), s.cfg,
                                   s.recent[-s.cfg.rep_window:])
                ends = nid in s.stops or len(s.out) >= s.cfg.max_new_tokens
            except Exception as e:  # noqa: BLE001
                s.error = e
                ends = True
            if ends:
                finished.append(b)
                continue
            tok_of[b] = nid
        rows = [b for b in tok_of if self.slots[b].cfg.logprobs is not None]
        try:
            self._record_logprobs(rows, tok_of)
        except Exception as e:  # noqa: BLE001
            for b in rows:
                self.slots[b].error = e
                finished.append(b)
                del tok_of[b]
        for b, nid in tok_of.items():
            s = self.slots[b]
            s.out.append(nid)
            s.recent.append(nid)
            if s.cb is not None:
                try:
                    s.cb(nid)
                except Exception:  # noqa: BLE001
                    pass
        for b in finished:
            self._retire(b)
        live: List[int] = []
        for b in tok_of:
            if self.cache.lens[b] + 1 > self.max_len or \
                    self.cache.pages_needed(live + [b], [1] * (len(live) + 1)) \
                    > self.cache.free_pages:
                self._retire(b)
                finished.append(b)
            else:
                live.append(b)
        if live:
            x = torch.tensor([[tok_of[b]] for b in live], dtype=torch.long)
            try:
                logits, _, _ = self.model(x.to(self.device),
                                          kv_caches=self.cache.decode(live))
            except Exception:
                for b in live:
                    self._retire(b)
                raise
            rows = torch.tensor(live).to(self.device)
            self.last_logits.index_copy_(0, rows, logits[:, -1].float())
            self.stats["steps"] += 1
        self.stats["tokens_out"] += len(tok_of)
        return finished

    def _record_logprobs(self, rows: List[int], tok_of: Dict[int, int]):
        """Log probabilities of the rows' next tokens, under the model's own
        distribution (before penalties and temperature)."""
        if not rows:
            return
        k = min(max(self.slots[b].cfg.logprobs for b in rows),
                self.last_logits.shape[-1])
        r = ops.token_logprobs(
            self.last_logits.index_select(
                0, torch.tensor(rows).to(self.device)),
            torch.tensor([tok_of[b] for b in rows]).to(self.device), k)
        lp, ids, top = (t.tolist() for t in (r.logprobs, r.top_ids,
                                             r.top_logprobs))
        for i, b in enumerate(rows):
            n = self.slots[b].cfg.logprobs
            self.slots[b].logprobs.append(
                {"token": tok_of[b], "logprob": lp[i],
                 "top": list(zip(ids[i][:n], top[i][:n]))})

    def _retire(self, b: int):
        s = self.slots[b]
        s.active = False
        s.result = list(s.out)
        self.cache.free(b)
        self.stats["finished"] += 1
        if s.done is not None:
            s.done.set()

    # ------------------------------------------------------------- convenience
    def run_to_completion(self, requests: List, configs=None,
                          admit_schedule: Optional[List[int]] = None
                          ) -> List[List[int]]:
        """Drives admit_many / step until every request finishes;
        admit_schedule[i] is the step at which request i arrives."""
        n = len(requests)
        cfgs = configs if isinstance(configs, list) else [configs] * n
        sched = admit_schedule or [0] * n
        slot_of: Dict[int, int] = {}
        results: List[Optional[List[int]]] = [None] * n
        waiting = sorted(range(n), key=lambda i: sched[i])
        t = 0
        while None in results:
            now = [i for i in waiting if sched[i] <= t]
            now = now[:self.admissible(
                [(min(len(requests[i]), self.max_len - 1), 1) for i in now])]
            if not now and not slot_of and sched[waiting[0]] <= t:
                raise RuntimeError("the page pool does not hold a prompt of "
                                   f"{len(requests[waiting[0]])} tokens")
            for i, b in zip(now, self.admit_many([requests[i] for i in now],
                                                 [cfgs[i] for i in now])):
                slot_of[i] = b
                waiting.remove(i)
            self.step()
            for i, b in list(slot_of.items()):
                if not self.slots[b].active:
                    if self.slots[b].error is not None:
                        raise self.slots[b].error
                    results[i] = self.slots[b].result
                    del slot_of[i]
            t += 1
        return results  # type: ignore[return-value]
