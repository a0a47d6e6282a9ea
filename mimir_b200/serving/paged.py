"""Decoding over the 8-bit paged cache: the serving operators put together.

:class:`PagedCache` owns the pool of all layers, the page table and the counts, and hands out
:class:`Batch` objects: the new tokens of some slots, packed one after the other.  A model's attention
calls :meth:`Batch.attend` with its unrotated q, k and v: ``ops.cache_append`` rotates and writes,
``ops.cache_attention`` attends.  :class:`PagedDecoder` generates with the Transformers Mimir2 model
(:mod:`mimir_b200.export.transformers_mimir2`): prompts of any lengths run packed, without padding; ``n``
completions of a prompt share its pages (``ops.cache_fork``); every request has its own penalties,
biases and allowed tokens (``ops.process_logits``); finished sequences give their pages back; a pool that is
full moves into a larger one (``ops.cache_compact``).

The reference serves with its patched vLLM (``src/mimir/serving/server.py:12-75``); the cache there is
vLLM's own.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Iterator, Optional

import torch

from mimir_b200 import ops
from mimir_b200.ops._ext import KernelTimeout
from mimir_b200.ops.kv_cache import BLOCK, MAX_SEQUENCES, cache_status, check_cache_status


def rotary_tables(positions: int, dim: int, theta: float, device) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 cos and sin ``[positions, dim]`` (halves duplicated), as the model's own rope computes them."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, dim, 2, dtype=torch.float32, device=device) / dim))
    angle = torch.arange(positions, dtype=torch.float32, device=device)[:, None] * inv_freq
    angle = torch.cat((angle, angle), dim=-1)
    return angle.cos(), angle.sin()


class PagedCache:
    """An 8-bit cache of ``slots`` sequences for every attention layer; it grows when its pages run out."""

    def __init__(self, layers: int, slots: int, max_len: int, kv_heads: int, head_dim: int, *, theta: float = 10000.0,
                 page_size: int = 64, pages: Optional[int] = None, device="cpu"):
        self.page_size, self.max_len = page_size, max_len
        width = -(-max_len // page_size)
        pages = pages if pages is not None else max(slots * min(width, 8), 1)
        self.pages, self.scales = self._pool(layers, pages, kv_heads, head_dim, page_size, device)
        self.page_table = torch.full((slots, width), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.ref_counts = torch.zeros(pages, dtype=torch.int32, device=device)
        self.cos, self.sin = rotary_tables(width * page_size, head_dim, theta, device)

    @staticmethod
    def _pool(layers, pages, kv_heads, head_dim, page_size, device):
        shape = (layers, pages, 2, kv_heads, page_size, head_dim)
        # (no byte of a fresh pool is NaN; what lies beyond a sequence is not read in any case)
        return (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                torch.zeros((*shape[:4], page_size // BLOCK), device=device))

    @property
    def device(self):
        return self.pages.device

    def _growing(self, call) -> None:
        """``call`` returns the number of pages that lack: once more then, with as many."""
        for again in (False, True):
            missing = int(call())
            if missing < 0:
                raise ValueError("a sequence of the paged cache would be longer than its page table")
            if missing == 0:
                return
            if again:
                raise RuntimeError(f"the paged cache lacks {missing} pages after it has grown")
            self.resize(self.pages.shape[1] + max(missing, self.pages.shape[1] // 2))

    def reserve(self, slots, counts) -> None:
        """Room for ``counts[i]`` more tokens of ``slots[i]``; the pool grows if its pages run out."""
        self._growing(lambda: ops.cache_reserve(self.page_table, self.seq_lens, self.ref_counts, slots, counts, self.page_size))

    def fork(self, src, dst) -> None:
        """``dst[i]`` becomes a copy of ``src[i]``: whole pages are shared."""
        self._growing(lambda: ops.cache_fork(self.pages, self.scales, self.page_table, self.seq_lens, self.ref_counts, src, dst))

    def free(self, slots) -> None:
        ops.cache_free(self.page_table, self.seq_lens, self.ref_counts, slots)

    def resize(self, pages: int) -> None:
        """Move into a pool of ``pages`` pages (at least as many as are held)."""
        layers, _, _, kv_heads, page_size, head_dim = self.pages.shape
        new = (*self._pool(layers, pages, kv_heads, head_dim, page_size, self.device), torch.empty_like(self.page_table),
               torch.zeros(pages, dtype=torch.int32, device=self.device))
        missing = int(ops.cache_compact(self.pages, self.scales, self.page_table, self.ref_counts, out=new))
        if missing:
            raise ValueError(f"the paged cache holds {missing} pages more than {pages}")
        self.pages, self.scales, self.page_table, self.ref_counts = new

    def batch(self, slots, counts, *, prompts: bool = False) -> "Batch":
        """The last ``counts[i]`` tokens of ``slots[i]``, which :meth:`reserve` has made room for.  ``prompts``:
        they are whole prompts, and every token of one sees all of it."""
        return Batch(self, [int(s) for s in slots], [int(c) for c in counts], prompts)


class Batch:
    """New tokens of some slots, packed: row ``cu_new[i]`` is the first of ``slots[i]``."""

    def __init__(self, cache: PagedCache, slots: list[int], counts: list[int], prompts: bool):
        self.cache, self.slots, self.counts = cache, slots, counts
        self.max_new, self.total = max(counts), sum(counts)
        bounds = [0]
        for c in counts:
            bounds.append(bounds[-1] + c)
        both = torch.tensor(slots + bounds + (counts if prompts else []), dtype=torch.int32).to(cache.device)  # one copy
        n = len(slots)
        self.seqs, self.cu_new = both[:n], both[n:2 * n + 1]
        self.prefix_lens = both[2 * n + 1:].contiguous() if prompts else None
        self.last_rows = self.cu_new[1:].long() - 1

    def positions(self) -> torch.Tensor:
        """Positions ``[total]`` of the new tokens in their sequences."""
        starts = self.cache.seq_lens[self.seqs.long()] - (self.cu_new[1:] - self.cu_new[:-1])
        rows = torch.arange(self.total, device=self.cache.device)
        at = torch.searchsorted(self.cu_new, rows, right=True) - 1
        return rows - self.cu_new[at] + starts[at]

    def attend(self, layer: int, q, k, v):
        """``q [total, heads, d]``, ``k`` and ``v [total, kv_heads, d]`` before their rotation -> attention."""
        c = self.cache
        pages, scales = c.pages[layer], c.scales[layer]
        q = ops.cache_append(q, k, v, c.cos, c.sin, pages, scales, c.page_table, c.seq_lens, self.seqs, self.cu_new)
        return ops.cache_attention(q, pages, scales, c.page_table, c.seq_lens, self.seqs, self.cu_new, self.prefix_lens,
                                   max_new=self.max_new)


FLOAT32_MAX = torch.finfo(torch.float32).max
LEAST = 1e-30              # temperature (logits divided by it stay in float32) and top_p (not rounded to zero)
MAX_COMPLETIONS = 128      # of one request, and of a server's batch: each takes a slot of the cache


@dataclass
class Request:
    """One prompt and its decoding rule (OpenAI's fields; ``repetition_penalty`` as Transformers has it)."""
    ids: list[int]
    max_tokens: int = 16
    temperature: float = 0.0           # 0: greedy
    top_p: float = 1.0
    n: int = 1
    seed: Optional[int] = None
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    repetition_penalty: float = 1.0
    logit_bias: dict = field(default_factory=dict)
    allowed_token_ids: Optional[list] = None

    def check(self, vocab: int, max_len: int) -> None:
        if not self.ids or any(not 0 <= i < vocab for i in self.ids):
            raise ValueError("a prompt needs tokens of the vocabulary")
        if len(self.ids) + 1 > max_len:
            raise ValueError(f"a prompt of {len(self.ids)} tokens does not fit {max_len} positions")
        if self.n < 1 or self.max_tokens < 1 or self.repetition_penalty <= 0:
            raise ValueError("n, max_tokens and repetition_penalty must be positive")
        if self.n > MAX_COMPLETIONS:
            raise ValueError(f"n is at most {MAX_COMPLETIONS}")
        # (comparisons that NaN does not pass)
        if not -FLOAT32_MAX <= self.temperature <= FLOAT32_MAX or 0 < self.temperature < LEAST:
            raise ValueError(f"temperature must be zero (greedy) or at least {LEAST}, and finite")
        if not self.top_p >= LEAST:
            raise ValueError(f"top_p must be at least {LEAST}")
        if not 2.0 ** -126 <= self.repetition_penalty <= 2.0 ** 126:
            raise ValueError("repetition_penalty and its inverse must be float32 numbers")
        if not all(abs(x) <= FLOAT32_MAX for x in (self.presence_penalty, self.frequency_penalty)):
            raise ValueError("presence_penalty and frequency_penalty must be finite float32 numbers")
        if any(not 0 <= int(i) < vocab for i in self.logit_bias):
            raise ValueError("logit_bias names tokens of the vocabulary")
        if any(not v <= FLOAT32_MAX for v in self.logit_bias.values()):
            raise ValueError("logit_bias holds finite float32 numbers, or -inf")
        if self.seed is not None and not -2 ** 63 <= self.seed <= 2 ** 64 - self.n:
            raise ValueError("seed must lie in 64 bits, with one for each of the n completions")
        if self.allowed_token_ids is not None and not any(0 <= int(i) < vocab for i in self.allowed_token_ids):
            raise ValueError("allowed_token_ids allows no token of the vocabulary")


class PagedDecoder:
    """Generates with a Transformers Mimir2 model over a :class:`PagedCache`."""

    def __init__(self, model, *, page_size: int = 64, pages: Optional[int] = None, slots: int = 16):
        cfg = model.config
        device = next(model.parameters()).device
        if device.type == "cuda":
            if cfg.head_dim != 128:
                raise ValueError(f"the 8-bit paged cache needs a head dimension of 128, not {cfg.head_dim}")
            if model.dtype not in (torch.bfloat16, torch.float16):
                raise ValueError(f"the 8-bit paged cache needs a bfloat16 or float16 model, not {model.dtype}")
        self.model, self.config, self.device = model, cfg, device
        self.layers = cfg.num_layers_per_stack * cfg.H_cycles * (cfg.L_cycles + 1)
        self.page_size, self.pages = page_size, pages
        self._running = False
        self._make(slots)

    def _make(self, slots: int) -> None:
        cfg = self.config
        self.cache = PagedCache(self.layers, slots, cfg.max_position_embeddings, cfg.num_key_value_heads, cfg.head_dim,
                                theta=float(cfg.rope_parameters.get("rope_theta", 10000.0)), page_size=self.page_size,
                                pages=self.pages, device=self.device)
        # every slot's prompt and generated tokens: the n-gram memory's context and the penalties' history
        self.history = torch.zeros(slots, self.cache.page_table.shape[1] * self.page_size, dtype=torch.int32, device=self.device)

    def _rules(self, rows: list[tuple[Request, int]], vocab: int) -> dict:
        """``ops.process_logits`` arguments of the requests that share a step (one row a completion)."""
        reqs = [r for r, _ in rows]
        kw = {}
        prompt = torch.tensor([len(r.ids) for r in reqs], dtype=torch.int32)
        if any(r.presence_penalty or r.frequency_penalty or r.repetition_penalty != 1.0 for r in reqs):
            table = torch.tensor([[r.repetition_penalty, r.presence_penalty, r.frequency_penalty] for r in reqs])
            kw["prompt_lens"] = prompt.to(self.device)
            kw["repetition"], kw["presence"], kw["frequency"] = table.t().contiguous().to(self.device)
        if any(r.logit_bias for r in reqs):
            offsets, ids, values = [0], [], []
            for r in reqs:
                ids += [int(i) for i in r.logit_bias]
                values += [float(v) for v in r.logit_bias.values()]
                offsets.append(len(ids))
            kw["bias"] = (torch.tensor(offsets, dtype=torch.int32).to(self.device),
                          torch.tensor(ids, dtype=torch.int32).to(self.device), torch.tensor(values).to(self.device))
        if any(r.allowed_token_ids is not None for r in reqs):
            mask = torch.full((len(reqs), -(-vocab // 32) * 32), True)
            for row, r in zip(mask, reqs):
                if r.allowed_token_ids is not None:
                    row.fill_(False)
                    row[[int(i) for i in r.allowed_token_ids if 0 <= int(i) < vocab]] = True
            words = (mask.view(len(reqs), -1, 32).long() << torch.arange(32)).sum(-1)
            kw["allowed"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).to(self.device)
        return kw

    @staticmethod
    def _sample(logits: torch.Tensor, reqs: list[Request], generators: list) -> list[Optional[int]]:
        """A token of each row; None where there is none to choose: NaN among the logits, or everything forbidden.
        (Such rows do not come to ``torch.multinomial``, which reports them by an assertion on the device.)"""
        best = logits.max(-1)  # NaN where one is among them; of equal ones the first
        out = []
        for i, (r, top, token) in enumerate(zip(reqs, *torch.stack((best.values.double(), best.indices.double())).tolist())):
            if r.temperature <= 0:
                out.append(int(token) if top > -math.inf else None)
                continue
            if not abs(top / r.temperature) < 2.0 ** 127:  # softmax is finite where its largest argument is
                out.append(None)
                continue
            p = torch.softmax(logits[i] / r.temperature, -1)
            if r.top_p < 1.0:
                order = p.argsort(descending=True, stable=True)
                ahead = p[order].cumsum(-1) - p[order]
                p = p.index_fill(0, order[ahead >= r.top_p], 0.0)
            out.append(int(torch.multinomial(p, 1, generator=generators[i])))
        return out

    @torch.no_grad()
    def run(self, requests: list[Request], eos: Optional[int] = None,
            failed: Optional[dict] = None) -> Iterator[tuple[int, int, int]]:
        """Yields ``(request, completion, token)`` as tokens are generated (the end token included), all
        completions of all requests side by side.  A request that has no token to choose leaves the batch with an
        exception, which ``failed`` takes at its number; without ``failed`` it is raised."""
        vocab = self.config.vocab_size
        limit = min(self.config.max_position_embeddings, self.history.shape[1])
        for r in requests:
            r.check(vocab, limit)
        slots = sum(r.n for r in requests)
        if not requests:
            return
        if slots > MAX_SEQUENCES:
            raise ValueError(f"{slots} completions side by side are more than {MAX_SEQUENCES}")
        if self._running:
            raise RuntimeError("a batch of this decoder is not finished (nor closed): it holds the slots")
        if slots > self.cache.page_table.shape[0]:
            self._make(slots)
        cache, used = self.cache, list(range(slots))
        first = [sum(r.n for r in requests[:i]) for i in range(len(requests))]
        generators = {(i, w): torch.Generator(self.device).manual_seed(r.seed + w)
                      for i, r in enumerate(requests) if r.seed is not None for w in range(r.n)}
        self._running, reported = True, False
        try:
            # ---- prompts, packed; then a slot for each further completion
            counts = [len(r.ids) for r in requests]
            cache.reserve(first, counts)
            packed = torch.tensor([i for r in requests for i in r.ids]).to(self.device)
            batch = cache.batch(first, counts, prompts=self.config.prefix_lm)
            hidden = self.model.model.forward_paged(packed, batch)
            logits = self.model.lm_head(hidden[batch.last_rows])
            for slot, r in zip(first, requests):
                for w in range(r.n):
                    self.history[slot + w, :len(r.ids)] = torch.tensor(r.ids, dtype=torch.int32)
            pairs = [(f, f + w) for f, r in zip(first, requests) for w in range(1, r.n)]
            if pairs:
                cache.fork([a for a, _ in pairs], [b for _, b in pairs])
            live = [(i, w) for i, r in enumerate(requests) for w in range(r.n)]
            logits = logits[torch.tensor([i for i, _ in live], device=self.device)]
            made = {key: 0 for key in live}
            # ---- one token of every completion at a time
            while True:
                rows = [(requests[i], w) for i, w in live]
                at = [first[i] + w for i, w in live]
                kw = self._rules(rows, vocab)
                if "prompt_lens" in kw:
                    where = torch.tensor(at, device=self.device)
                    kw["token_lens"] = cache.seq_lens[where]
                    kw["tokens"] = self.history[where, :max(len(r.ids) + made[k] for (r, _), k in zip(rows, live))]
                tokens = self._sample(ops.process_logits(logits, **kw), [r for r, _ in rows], [generators.get(k) for k in live])
                check_cache_status(self.device)  # the host has waited for the step
                lost = {}
                for row, ((i, _), token) in enumerate(zip(live, tokens)):
                    if token is None and not bool(torch.isfinite(logits[row]).all()):
                        lost[i] = RuntimeError("the model's logits are not finite")
                    elif token is None:
                        lost.setdefault(i, ValueError("the rules of the request leave no token to choose"))
                if lost and failed is None:
                    raise next(iter(lost.values()))
                if lost:
                    failed.update(lost)
                still, ended = [], []
                for key, token in zip(live, tokens):
                    if key[0] in lost:
                        ended.append((key, None))
                        continue
                    made[key] += 1
                    yield key[0], key[1], token
                    r = requests[key[0]]
                    full = made[key] >= r.max_tokens or len(r.ids) + made[key] >= limit
                    (ended if full or token == eos else still).append((key, token))
                gone = [first[i] + w for (i, w), _ in ended]
                if gone:
                    cache.free(gone)
                    used = [s for s in used if s not in set(gone)]
                if not still:
                    return
                live = [key for key, _ in still]
                at = [first[i] + w for i, w in live]
                ids = torch.tensor([t for _, t in still], dtype=torch.int32)
                lens = [len(requests[i].ids) + made[(i, w)] for i, w in live]
                self.history[torch.tensor(at), torch.tensor(lens) - 1] = ids.to(self.device)
                cache.reserve(at, [1] * len(at))
                batch = cache.batch(at, [1] * len(at))
                batch.ngram_history, batch.ngram_lens = self.history, lens
                logits = self.model.lm_head(self.model.model.forward_paged(ids.to(self.device, torch.long), batch))
        except KernelTimeout:
            reported = True
            raise
        finally:
            self._running = False
            if used:
                cache.free(used)
            if reported:
                cache_status(self.device)  # what freeing a bad page reports is this batch's too, not the next one's

    def generate(self, requests: list[Request], eos: Optional[int] = None,
                 failed: Optional[dict] = None) -> list[list[list[int]]]:
        """Generated tokens of every completion of every request (``failed`` as :meth:`run` has it)."""
        out = [[[] for _ in range(r.n)] for r in requests]
        for i, w, token in self.run(requests, eos, failed):
            out[i][w].append(token)
        return out
