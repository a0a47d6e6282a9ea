"""The serving operators over an 8-bit paged key/value cache, as cases to be measured.

Four groups, reached through ``mimir_b200.ops``:

* ``attention``: attention of new tokens over the cache (``cache_attention``);
* ``append``: rotary embedding of q and k, and k and v written to the cache (``cache_append``);
* ``pages``: bookkeeping and movement of pages (``cache_free``, ``cache_reserve``, ``cache_fork``,
  ``cache_compact``);
* ``logits``: repetition penalties, biases and grammar masks (``process_logits``).

Cache layout: pages e4m3 ``[pages, 2, kv_heads, page_size, head_dim]`` (k, then v; a leading layer
dimension for the page operations), scales fp32 ``[pages, 2, kv_heads, page_size / 16]``, each a
power of two for 16 tokens of one head; page table int32 ``[slots, width]`` with -1 for no page;
sequence lengths int32 ``[slots]``; reference counts int32 ``[pages]``.

A case's lengths follow from the case alone, its values and the order of its pages from the seed.
"""
import math
import random

import torch

own = False

BLOCK = 16      # tokens that share a scale
HEAD_DIM = 128  # every size preset of this repository
E4M3_MAX = 448.0
MIN_EXP = -32   # smallest scale is 2**MIN_EXP


# ---------------------------------------------------------------------------------- the cases
def listed():
    return [
        # One user, one short conversation: the smallest call of a decoding loop, latency only.
        dict(name="decode one", op="attention", seqs=1, context=333, new=1, ragged=False, heads=16, kv_heads=4,
             page=64, dtype="bfloat16", prefix="none"),
        # A full serving batch, conversations of very different lengths, one new token each.
        dict(name="decode batch", op="attention", seqs=64, context=8000, new=1, ragged=True, heads=16, kv_heads=4,
             page=64, dtype="bfloat16", prefix="none"),
        # Long documents: the cache's bytes are all that counts.
        dict(name="decode long", op="attention", seqs=8, context=100001, new=1, ragged=True, heads=16, kv_heads=4,
             page=128, dtype="bfloat16", prefix="none"),
        # A model without grouped heads takes a few tokens at a time (drafted tokens, short turns).
        dict(name="drafts ungrouped", op="attention", seqs=24, context=2100, new=7, ragged=True, heads=20, kv_heads=20,
             page=16, dtype="float16", prefix="none"),
        # Prompts: bidirectional over the whole prompt, all of it new.
        dict(name="prompts", op="attention", seqs=5, context=4096, new=4096, ragged=True, heads=16, kv_heads=4,
             page=64, dtype="bfloat16", prefix="prompt"),
        # One decoding step of a full batch writes one token a sequence.
        dict(name="append batch", op="append", seqs=64, context=2000, new=1, ragged=True, heads=16, kv_heads=4, page=64,
             dtype="bfloat16"),
        # Prompts are written at once.
        dict(name="append prompts", op="append", seqs=5, context=4096, new=4096, ragged=True, heads=16, kv_heads=4,
             page=64, dtype="bfloat16"),
        # Finished conversations leave and new prompts enter a pool of pages.
        dict(name="turnover", op="pages", do="turnover", slots=256, seqs=48, context=4000, ragged=True, layers=1,
             kv_heads=1, page=64, dtype="bfloat16"),
        # Four prompts, eight completions each: whole pages shared, the last one copied in every layer.
        dict(name="fork", op="pages", do="fork", slots=64, seqs=32, context=1500, ragged=True, layers=24, kv_heads=4,
             page=64, dtype="bfloat16"),
        # A half empty pool moves into a smaller one.
        dict(name="compact", op="pages", do="compact", slots=32, seqs=16, context=1700, ragged=True, layers=24,
             kv_heads=4, page=64, dtype="bfloat16"),
        # One user's next token with penalties and a short history.
        dict(name="logits one", op="logits", rows=1, vocab=65536, history=300, bias=8, mask=False, dtype="bfloat16"),
        # A batch with long histories, the most biases that requests may carry, and a grammar.
        dict(name="logits batch", op="logits", rows=128, vocab=65536, history=4000, bias=300, mask=True,
             dtype="bfloat16"),
    ]


def _span(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    # No drawn case reads more of a cache, holds more scores or moves more pages than the largest listed one.
    op = rng.choice(["attention", "attention", "attention", "attention", "append", "append", "pages", "pages", "logits", "logits"])
    kv = rng.choice([1, 2, 3, 4, 5, 8, 20])
    group = rng.choice([1, 2, 3, 4, 5, 8]) if kv < 20 else 1
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if op == "attention":
        kind = rng.choice(["decode", "decode", "drafts", "prompts"])
        if kind == "prompts":
            seqs, new = _span(rng, 1, 6), _span(rng, 65, 3500)
            context = new + (rng.choice([0, 0, _span(rng, 1, 500)]))
            while seqs * context * new * kv * group > 5 * 4096 * 4096 * 16:
                seqs, kv, group = max(1, seqs // 2), max(1, kv // 2), max(1, group // 2)
            prefix = rng.choice(["prompt", "half", "none"])
        else:
            new = 1 if kind == "decode" else _span(rng, 2, 40)
            seqs = _span(rng, 1, 128)
            context = max(new, _span(rng, 1, 60000))
            while seqs * context * kv > 8 * 100001 * 4:
                context = max(new, context // 2)
            prefix = "none"
        return dict(op=op, seqs=seqs, context=context, new=new, ragged=rng.random() < 0.8, heads=kv * group, kv_heads=kv,
                    page=page, dtype=dtype, prefix=prefix)
    if op == "append":
        new = rng.choice([1, _span(rng, 2, 4000)])
        seqs = _span(rng, 1, 128)
        while seqs * new * kv * (group + 2) > 5 * 4096 * 4 * 6:
            seqs, new = max(1, seqs // 2), max(1, new // 2)
        context = new + rng.choice([0, _span(rng, 1, 2000)])
        while seqs * context * kv > 2000000:
            seqs = seqs // 2
        return dict(op=op, seqs=seqs, context=context, new=new,
                    ragged=rng.random() < 0.8, heads=kv * group, kv_heads=kv, page=page, dtype=dtype)
    if op == "pages":
        do = rng.choice(["turnover", "fork", "compact"])
        seqs, kv = _span(rng, 1, 24), min(kv, 4)
        slots = 2 * seqs + rng.randrange(0, 16)
        layers = 1 if do == "turnover" else _span(rng, 1, 24)
        return dict(op=op, do=do, slots=slots, seqs=seqs, context=_span(rng, 1, 1500), ragged=rng.random() < 0.8,
                    layers=layers, kv_heads=kv, page=page, dtype="bfloat16")
    return dict(op=op, rows=_span(rng, 1, 128), vocab=_span(rng, 500, 65536) + rng.randrange(0, 2), history=_span(rng, 1, 4000),
                bias=rng.choice([0, _span(rng, 1, 300)]), mask=rng.random() < 0.6, dtype=rng.choice(["bfloat16", "float16", "float32"]))


def _lengths(case):
    """(lengths of the cached sequences with their new tokens, numbers of new tokens)."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["context"], case.get("new", 1)))
    n, new = case["seqs"], case.get("new", 1)
    if not case["ragged"]:
        return [case["context"]] * n, [new] * n
    counts = [new] + [max(1, round(new * rng.uniform(0.3, 1.0))) for _ in range(n - 1)]
    old = case["context"] - new
    if old <= 0:
        return counts, counts
    lens = [old + new] + [c + round(old * rng.random() ** 2) for c in counts[1:]]
    return lens, counts


def _prefixes(case, lens):
    kind = case.get("prefix", "none")
    return None if kind == "none" else [n if kind == "prompt" else n // 2 for n in lens]


# ---------------------------------------------------------------------------------- inputs
def _exponent(amax):
    """Smallest e >= MIN_EXP with amax <= 448 * 2**e."""
    mant, exp = torch.frexp(amax)
    return torch.clamp(exp - 9 + (mant > 0.875), min=MIN_EXP)


def _pool(shape, gen):
    """Cached values ``[..., tokens, head_dim]`` of uneven size, in 8 bits, and their scales."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((*shape[:-1], 1), generator=gen, device="cuda"))
    blocks = x.unflatten(-2, (-1, BLOCK))
    e = _exponent(blocks.abs().amax((-1, -2)))
    scales = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    return (blocks / scales[..., None, None]).to(torch.float8_e4m3fn).reshape(shape), scales


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(lens, page, pages, width, gen):
    """Page table rows whose pages lie in any order in the pool."""
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    need = torch.tensor([-(-n // page) for n in lens], device="cuda")
    first = need.cumsum(0) - need
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col).clamp_max(pages - 1)
    return torch.where(col < need[:, None], order[at], -1).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    st = dict(case=case)
    if case["op"] == "logits":
        rows, vocab, most = case["rows"], case["vocab"], case["history"]
        st["logits"] = (3.0 * torch.randn(rows, vocab, generator=gen, device="cuda")).to(dtype)
        u = torch.rand(rows, most, generator=gen, device="cuda")
        st["tokens"] = (vocab * u ** 3).to(torch.int32).clamp_max(vocab - 1)  # a few tokens are repeated often
        st["token_lens"] = torch.randint(most // 2, most + 1, (rows,), generator=gen, device="cuda").to(torch.int32)
        st["prompt_lens"] = st["token_lens"] // 3
        st["repetition"] = 1.0 + 0.3 * torch.rand(rows, generator=gen, device="cuda")
        st["presence"] = torch.rand(rows, generator=gen, device="cuda")
        st["frequency"] = 0.1 * torch.rand(rows, generator=gen, device="cuda")
        b = case["bias"]
        st["bias_offsets"] = torch.arange(rows + 1, device="cuda", dtype=torch.int32) * b
        st["bias_ids"] = torch.randint(0, vocab, (rows * b,), generator=gen, device="cuda").to(torch.int32)
        st["bias_values"] = 4.0 * torch.randn(rows * b, generator=gen, device="cuda")
        st["allowed"] = None
        if case["mask"]:
            words = -(-vocab // 32)
            st["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=gen, device="cuda").to(torch.int32)
        return st
    page, kv = case["page"], case["kv_heads"]
    lens, counts = _lengths(case)
    if case["op"] == "pages":
        return _prepare_pages(st, lens, gen)
    need = sum(-(-n // page) for n in lens)
    width = max(-(-n // page) for n in lens) + 1
    pages = need + need // 8 + 1
    st["table"] = _table(lens, page, pages, width, gen)
    st["seq_lens"], st["seqs"] = _ints(lens), torch.arange(len(lens), device="cuda", dtype=torch.int32)
    st["cu_new"] = torch.cat([_ints([0]), _ints(counts).cumsum(0).to(torch.int32)])
    st["max_new"], st["max_len"], st["total"] = max(counts), max(lens), sum(counts)
    st["pages"], st["scales"] = _pool((pages, 2, kv, page, HEAD_DIM), gen)
    q = torch.randn(st["total"], case["heads"], HEAD_DIM, generator=gen, device="cuda")
    st["q"] = q.to(dtype)
    if case["op"] == "attention":
        prefixes = _prefixes(case, lens)
        st["prefix_lens"] = None if prefixes is None else _ints(prefixes)
        return st
    size = torch.exp(0.5 * torch.randn(st["total"], kv, 1, generator=gen, device="cuda"))
    st["k"] = (size * torch.randn(st["total"], kv, HEAD_DIM, generator=gen, device="cuda")).to(dtype)
    st["v"] = (size * torch.randn(st["total"], kv, HEAD_DIM, generator=gen, device="cuda")).to(dtype)
    angle = torch.outer(torch.arange(width * page, device="cuda", dtype=torch.float32),
                        10000.0 ** (-torch.arange(0, HEAD_DIM, 2, device="cuda", dtype=torch.float32) / HEAD_DIM))
    angle = torch.cat((angle, angle), -1)
    st["cos"], st["sin"] = angle.cos(), angle.sin()
    return st


def _pages_plan(case):
    """(length of each slot, source slots, destination slots, tokens that enter) of a page case."""
    lens, _ = _lengths(case)
    slots, n = case["slots"], case["seqs"]
    if case["do"] == "fork":
        sources = max(1, n // 8)
        held = lens[:sources] + [0] * n  # the destinations hold nothing yet
        return held + [0] * (slots - len(held)), [i % sources for i in range(n)], [sources + i for i in range(n)], None
    if case["do"] == "turnover":
        held = [lens[i % n] for i in range(slots)]
        return held, None, [(2 * i + 1) % slots if 2 * n <= slots else i for i in range(n)], lens[::-1]
    held = [lens[i // 2] if i % 2 == 0 and i // 2 < n else 0 for i in range(slots)]
    return held, None, None, None


def _prepare_pages(st, lens, gen):
    case = st["case"]
    page, layers, kv = case["page"], case["layers"], case["kv_heads"]
    held, src, dst, enter = _pages_plan(case)
    need = sum(-(-n // page) for n in held)
    width = max(-(-n // page) for n in held + lens) + 1
    pages = 2 * need + case["seqs"]
    table = _table(held, page, pages, width, gen)
    st["table"], st["seq_lens"] = table, _ints(held)
    st["refs"] = torch.zeros(pages + 1, dtype=torch.int32, device="cuda").index_add_(
        0, table.flatten().long() % (pages + 1), torch.ones(table.numel(), dtype=torch.int32, device="cuda"))[:pages]
    st["refs"] = st["refs"].contiguous()
    if case["do"] != "turnover":
        st["pages"], st["scales"] = _pool((layers * pages, 2, kv, page, HEAD_DIM), gen)
        st["pages"] = st["pages"].unflatten(0, (layers, pages))
        st["scales"] = st["scales"].unflatten(0, (layers, pages))
    if case["do"] == "compact":
        fewer = need + need // 8 + 1
        st["out"] = dict(pages=torch.zeros((layers, fewer, 2, kv, page, HEAD_DIM), dtype=torch.float8_e4m3fn, device="cuda"),
                         scales=torch.zeros((layers, fewer, 2, kv, page // BLOCK), device="cuda"),
                         table=torch.empty_like(table), refs=torch.zeros(fewer, dtype=torch.int32, device="cuda"))
    st["src"] = None if src is None else _ints(src)
    st["dst"] = None if dst is None else _ints(dst)
    st["enter"] = None if enter is None else _ints(enter)
    return st


# ---------------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    return (_run_own if own else _run_plain)[case["op"]](st)


def _own_attention(st):
    from mimir_b200 import ops
    return ops.cache_attention(st["q"], st["pages"], st["scales"], st["table"], st["seq_lens"], st["seqs"], st["cu_new"],
                               prefix_lens=st["prefix_lens"], max_new=st["max_new"])


def _own_append(st):
    from mimir_b200 import ops
    q = ops.cache_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["pages"], st["scales"], st["table"],
                         st["seq_lens"], st["seqs"], st["cu_new"])
    return dict(q=q, pages=st["pages"], scales=st["scales"])


def _own_pages(st):
    from mimir_b200 import ops
    do, page = st["case"]["do"], st["case"]["page"]
    if do == "turnover":
        ops.cache_free(st["table"], st["seq_lens"], st["refs"], st["dst"])
        missing = ops.cache_reserve(st["table"], st["seq_lens"], st["refs"], st["dst"], st["enter"], page)
        return dict(table=st["table"], seq_lens=st["seq_lens"], refs=st["refs"], missing=missing)
    if do == "fork":
        missing = ops.cache_fork(st["pages"], st["scales"], st["table"], st["seq_lens"], st["refs"], st["src"], st["dst"])
        return dict(table=st["table"], seq_lens=st["seq_lens"], refs=st["refs"], missing=missing, pages=st["pages"],
                    scales=st["scales"])
    out = st["out"]
    missing = ops.cache_compact(st["pages"], st["scales"], st["table"], st["refs"],
                                out=(out["pages"], out["scales"], out["table"], out["refs"]))
    return dict(out, missing=missing)


def _own_logits(st):
    from mimir_b200 import ops
    return ops.process_logits(st["logits"], tokens=st["tokens"], token_lens=st["token_lens"],
                              prompt_lens=st["prompt_lens"], repetition=st["repetition"], presence=st["presence"],
                              frequency=st["frequency"],
                              bias=(st["bias_offsets"], st["bias_ids"], st["bias_values"]), allowed=st["allowed"])


_run_own = dict(attention=_own_attention, append=_own_append, pages=_own_pages, logits=_own_logits)


# ---------------------------------------------------------------------------------- plain forms
def _plain_attention(st):
    """Gathers every sequence's pages, padded to the longest, and goes through all scores at once."""
    pages, scales, q, lens, cu = st["pages"], st["scales"], st["q"], st["seq_lens"].long(), st["cu_new"].long()
    page, kv, heads = pages.shape[3], pages.shape[2], q.shape[1]
    n, most = lens.numel(), st["max_new"]
    width = -(-st["max_len"] // page)
    at = st["table"][st["seqs"].long(), :width].long().clamp_min(0)                      # [n, width]
    both = pages[at].to(torch.float32).unflatten(-2, (-1, BLOCK)) * scales[at][..., None, None]
    both = both.flatten(-3, -2).permute(2, 0, 3, 1, 4, 5).flatten(3, 4)                  # [2, n, kv, keys, d]
    counts = cu[1:] - cu[:-1]
    j = torch.arange(most, device=q.device)
    row = (cu[:-1, None] + j).clamp_max(q.shape[0] - 1)                                  # [n, most]
    rows = q[row].to(torch.float32).unflatten(2, (kv, heads // kv)).permute(0, 2, 3, 1, 4)  # [n, kv, group, most, d]
    pos = lens[:, None] - counts[:, None] + j
    limit = pos + 1
    if st["prefix_lens"] is not None:
        prefix = st["prefix_lens"].long()[:, None]
        limit = torch.where(pos < prefix, torch.maximum(prefix, limit), limit)
    limit = torch.minimum(limit, lens[:, None])
    seen = torch.arange(both.shape[3], device=q.device) < limit[..., None]               # [n, most, keys]
    s = torch.matmul(rows.flatten(2, 3), both[0].transpose(-1, -2)).unflatten(2, (-1, most)) / math.sqrt(q.shape[-1])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), both[1]).unflatten(2, (-1, most)) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                           # [n, most, heads, d]
    out = torch.zeros(q.shape[0] + 1, heads, q.shape[-1], device=q.device)
    out[torch.where(j < counts[:, None], row, q.shape[0])] = o
    return out[:-1].to(q.dtype)


def _rotate(x, cos, sin):
    x = x.to(torch.float32)
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat((-x[..., half:], x[..., :half]), -1) * sin[:, None]


def _plain_append(st):
    pages, scales, cu = st["pages"], st["scales"], st["cu_new"].long()
    count, _, kv, page, d = pages.shape
    per = page // BLOCK
    t = torch.arange(st["total"], device=pages.device)
    i = torch.searchsorted(cu, t, right=True) - 1
    slot = st["seqs"].long()[i]
    first = st["seq_lens"].long()[slot] - (cu[1:] - cu[:-1])[i]   # where the new tokens of a sequence start
    pos = first + t - cu[:-1][i]
    cos, sin = st["cos"][pos], st["sin"][pos]
    both = torch.stack((_rotate(st["k"], cos, sin), st["v"].to(torch.float32)), 1)       # [tokens, 2, kv, d]
    block = st["table"][slot, pos // page].long() * per + pos % page // BLOCK            # [tokens]
    amax = torch.full((count * per, 2, kv), -1.0, device=pages.device)
    amax.scatter_reduce_(0, block[:, None, None].expand(-1, 2, kv), both.abs().amax(-1), "amax")
    touched = amax >= 0                                                                  # of all heads or of none
    older = torch.zeros(count * per, dtype=torch.int64, device=pages.device)             # tokens a block held before
    older.scatter_reduce_(0, block, torch.clamp(first - pos // BLOCK * BLOCK, 0, BLOCK), "amax")
    old_scales = scales.permute(0, 3, 1, 2).flatten(0, 1)                                # [blocks, 2, kv]
    new_scales = torch.ldexp(torch.ones_like(amax), _exponent(amax.clamp_min(0.0)))
    keep = (older > 0)[:, None, None]
    new_scales = torch.where(keep, torch.maximum(new_scales, old_scales), new_scales)
    new_scales = torch.where(touched, new_scales, old_scales)
    held = pages.unflatten(3, (per, BLOCK)).permute(0, 3, 1, 2, 4, 5).flatten(0, 1).to(torch.float32)  # [blocks, 2, kv, 16, d]
    before = torch.arange(BLOCK, device=pages.device) < older[:, None]                   # tokens to round again
    ratio = torch.where(before[:, None, None], (torch.where(keep, old_scales, new_scales) / new_scales)[..., None], 1.0)
    again = (held * ratio[..., None]).to(pages.dtype)
    old = again.unflatten(0, (count, per)).permute(0, 2, 3, 1, 4, 5).flatten(3, 4)
    pages.copy_(old)
    bytes_ = (both / new_scales[block][..., None]).to(pages.dtype)
    pages.view(torch.uint8).permute(0, 3, 1, 2, 4)[block // per, pos % page] = bytes_.view(torch.uint8)
    scales.copy_(new_scales.unflatten(0, (count, per)).permute(0, 2, 3, 1))
    return dict(q=_rotate(st["q"], cos, sin).to(st["q"].dtype), pages=pages, scales=scales)


def _take(refs, need):
    """[rows, width] pages for rows that need ``need`` pages each: the free ones, lowest first."""
    free = torch.sort((refs != 0).to(torch.int8), stable=True).indices
    return free, need.cumsum(0) - need


def _drop(table, lens, refs, slots):
    gone = table[slots].long()
    refs.scatter_add_(0, gone.clamp_min(0).flatten(), -(gone >= 0).to(torch.int32).flatten())
    table[slots] = -1
    lens[slots] = 0


def _plain_pages(st):
    case, table, refs, lens = st["case"], st["table"], st["refs"], st["seq_lens"]
    page, width = case["page"], table.shape[1]
    col = torch.arange(width, device="cuda")
    if case["do"] == "turnover":
        dst = st["dst"].long()
        _drop(table, lens, refs, dst)
        need = (st["enter"].long() + page - 1) // page
        free, first = _take(refs, need)
        missing = (need.sum() - (refs == 0).sum()).clamp_min(0)
        used = (col < need[:, None]) & (missing == 0)
        new = free[(first[:, None] + col).clamp_max(refs.numel() - 1)]
        table[dst] = torch.where(used, new, -1).to(torch.int32)
        refs.scatter_add_(0, new.flatten(), used.to(torch.int32).flatten())
        lens[dst] = torch.where(missing == 0, st["enter"], 0)
        return dict(table=table, seq_lens=lens, refs=refs, missing=missing.to(torch.int32).reshape(1))
    pages, scales = st["pages"], st["scales"]
    if case["do"] == "fork":
        src, dst = st["src"].long(), st["dst"].long()
        _drop(table, lens, refs, dst)
        n = lens[src].long()
        whole, part = n // page, (n % page != 0).long()
        free, first = _take(refs, part)
        shared = col < whole[:, None]
        row = table[src]
        refs.scatter_add_(0, row.clamp_min(0).long().flatten(), shared.to(torch.int32).flatten())
        fresh = free[first.clamp_max(refs.numel() - 1)]
        refs.scatter_add_(0, fresh, part.to(torch.int32))
        new = torch.where((col == whole[:, None]) & (part[:, None] > 0), fresh[:, None].to(torch.int32), -1)
        table[dst] = torch.where(shared, row, new)
        lens[dst] = lens[src]
        last = row.gather(1, whole[:, None]).squeeze(1).long()
        first_page = row[:, 0].clamp_min(0).long()          # a row without a last page copies this page to itself
        a, b = torch.where(part > 0, last, first_page), torch.where(part > 0, fresh, first_page)
        pages.view(torch.uint8)[:, b] = pages.view(torch.uint8)[:, a]
        scales[:, b] = scales[:, a]
        missing = torch.zeros(1, dtype=torch.int32, device="cuda")
        return dict(table=table, seq_lens=lens, refs=refs, missing=missing, pages=pages, scales=scales)
    out = st["out"]
    live = refs != 0
    count, at = live.sum(), torch.arange(refs.numel(), device="cuda")
    holes = torch.sort(((live | (at >= count))).to(torch.int8), stable=True).indices   # free pages below count, lowest first
    rank = ((live & (at >= count)).cumsum(0) - 1).clamp_min(0)
    to = torch.where(at < count, at, holes[rank])                                       # where a live page goes
    fewer = out["refs"].numel()
    back = torch.full((fewer + 1,), -1, dtype=torch.int64, device="cuda")
    back[torch.where(live, to, fewer)] = at
    back = back[:fewer]
    fill = back >= 0
    new = pages.view(torch.uint8)[:, back.clamp_min(0)]
    out["pages"].view(torch.uint8).copy_(torch.where(fill[:, None, None, None, None], new, out["pages"].view(torch.uint8)))
    out["scales"].copy_(torch.where(fill[:, None, None, None], scales[:, back.clamp_min(0)], out["scales"]))
    out["table"].copy_(torch.where(table >= 0, to[table.clamp_min(0).long()].to(torch.int32), -1))
    out["refs"].copy_(torch.where(fill, refs[back.clamp_min(0)], 0))
    return dict(out, missing=(count - fewer).clamp_min(0).to(torch.int32).reshape(1))


def _plain_logits(st):
    x = st["logits"].to(torch.float32)
    rows, vocab = x.shape
    col = torch.arange(st["tokens"].shape[1], device="cuda")
    held = col < st["token_lens"][:, None]
    made = held & (col >= st["prompt_lens"][:, None])
    ids = st["tokens"].long()
    seen = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, ids, held.to(torch.float32)) > 0
    count = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, ids, made.to(torch.float32))
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0)
    at = torch.searchsorted(st["bias_offsets"], torch.arange(st["bias_ids"].numel(), device="cuda", dtype=torch.int32), right=True) - 1
    x = x + torch.zeros_like(x).index_put_((at, st["bias_ids"].long()), st["bias_values"], accumulate=True)
    if st["allowed"] is not None:
        v = torch.arange(vocab, device="cuda")
        bit = (st["allowed"][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        x = torch.where(bit != 0, x, -math.inf)
    return x


_run_plain = dict(attention=_plain_attention, append=_plain_append, pages=_plain_pages, logits=_plain_logits)


# ---------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        read = rows * (vocab * size + case["history"] * 3 + case["bias"] * 8 + (vocab // 8 if case["mask"] else 0))
        return dict(bytes=read + rows * vocab * 4, flops=rows * vocab)
    lens, counts = _lengths(case)
    kv, page = case["kv_heads"], case["page"]
    if case["op"] == "attention":
        prefixes = _prefixes(case, lens) or [0] * len(lens)
        pairs = 0
        for n, c, p in zip(lens, counts, prefixes):
            old, inside = n - c, max(0, min(p, n) - (n - c))
            pairs += inside * min(p, n) + sum(range(old + inside + 1, n + 1))
        held = sum(lens) * kv * 2 * (HEAD_DIM + 4 / BLOCK)
        return dict(bytes=held + 2 * sum(counts) * case["heads"] * HEAD_DIM * size, flops=4 * HEAD_DIM * pairs * case["heads"])
    if case["op"] == "append":
        tokens = sum(counts)
        rows = tokens * HEAD_DIM * (2 * case["heads"] * size + 2 * kv * (size + 1))
        return dict(bytes=rows + tokens * 8 * HEAD_DIM, flops=tokens * (case["heads"] + kv) * HEAD_DIM * 3)
    held, src, dst, enter = _pages_plan(case)
    piece = case["layers"] * 2 * kv * page * (HEAD_DIM + 4 / BLOCK)
    width = max(-(-n // page) for n in held + lens) + 1
    pages = 2 * sum(-(-n // page) for n in held) + case["seqs"]
    if case["do"] == "turnover":
        moved = 4 * (sum(-(-held[d] // page) for d in dst) * 3 + sum(-(-n // page) for n in enter) * 2 + pages)
    elif case["do"] == "fork":
        parts = [s for s in src if held[s] % page]
        moved = piece * (len(parts) + len(set(parts))) + 4 * (sum(-(-held[s] // page) for s in src) * 3 + pages)
    else:
        moved = piece * 2 * sum(-(-n // page) for n in held) + 4 * (2 * len(held) * width + 2 * pages)
    return dict(bytes=moved, flops=moved / 64)


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return dict(attention=_exact_attention, append=_exact_append, pages=_exact_pages, logits=_exact_logits)[case["op"]](st)


def _exact_attention(st):
    """One head of one sequence at a time."""
    q, cu, lens = st["q"].double(), st["cu_new"].tolist(), st["seq_lens"].tolist()
    kv, page = st["pages"].shape[2], st["pages"].shape[3]
    group = q.shape[1] // kv
    prefixes = st["prefix_lens"].tolist() if st["prefix_lens"] is not None else [0] * len(lens)
    out = torch.zeros_like(q)
    for i, n in enumerate(lens):
        rows = st["table"][i, :-(-n // page)].long()
        a, b = cu[i], cu[i + 1]
        at = torch.arange(n - (b - a), n, device="cuda")
        limit = torch.where(at < prefixes[i], max(prefixes[i], 0), at + 1).clamp(min=at + 1, max=torch.full_like(at, n))
        hidden = torch.arange(n, device="cuda")[None] >= limit[:, None]
        for h in range(kv):
            k, v = (st["pages"][rows, w, h].double().reshape(-1, HEAD_DIM)[:n]
                    * st["scales"][rows, w, h].double().repeat_interleave(BLOCK)[:n, None] for w in (0, 1))
            for g in range(h * group, (h + 1) * group):
                s = (q[a:b, g] @ k.T) * HEAD_DIM ** -0.5
                out[a:b, g] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
    return out


def _two(e):
    return torch.ldexp(torch.ones_like(e), e.to(torch.int32))


def _grid(x):
    """The e4m3 value nearest to ``x`` (ties to even)."""
    step = _two(torch.frexp(x.abs().clamp_min(2.0 ** -6)).exponent.to(x.dtype) - 4)
    return torch.round(x / step) * step


def _exact_append(st):
    """One block of 16 tokens at a time, all heads."""
    pages, scales = st["pages"].double(), st["scales"].double()
    page = pages.shape[3]
    cu, lens, table = st["cu_new"].tolist(), st["seq_lens"].tolist(), st["table"].tolist()
    pos = torch.cat([torch.arange(n - (b - a), n) for n, a, b in zip(lens, cu, cu[1:])]).cuda()

    def turn(x):
        c, s = st["cos"].double()[pos][:, None, :64], st["sin"].double()[pos][:, None, :64]
        lo, hi = x.double()[..., :64], x.double()[..., 64:]
        return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)

    new = torch.stack((turn(st["k"]), st["v"].double()), 1)  # [tokens, 2, kv, d]
    if sum(-(-n // BLOCK) for n in lens) > 40000:
        return None
    for i, n in enumerate(lens):
        t, p = cu[i], n - (cu[i + 1] - cu[i])
        while p < n:
            end = min(n, p // BLOCK * BLOCK + BLOCK)
            x = new[t:t + end - p].permute(1, 2, 0, 3)       # [2, kv, tokens, d]
            which, at = table[i][p // page], p % page // BLOCK
            first, off = p % page // BLOCK * BLOCK, p % BLOCK
            top = x.abs().amax((-1, -2))
            scale = _two(torch.floor(torch.log2(top / E4M3_MAX)).clamp_min(MIN_EXP) - 1)  # at most the one wanted
            for _ in range(3):
                scale = torch.where((top > E4M3_MAX * scale) | (scale < 2.0 ** MIN_EXP), 2 * scale, scale)
            if off:
                was = scales[which, :, :, at]
                scale = torch.maximum(scale, was)
                held = pages[which, :, :, first:first + off]
                pages[which, :, :, first:first + off] = _grid(held * (was / scale)[..., None, None])
            scales[which, :, :, at] = scale
            pages[which, :, :, first + off:first + off + end - p] = _grid(x / scale[..., None, None])
            t, p = t + end - p, end
    return dict(q=turn(st["q"]), pages=pages, scales=scales)


def _exact_pages(st):
    """Lists and sets of the host, one page at a time."""
    case, page = st["case"], st["case"]["page"]
    table, lens, refs = st["table"].tolist(), st["seq_lens"].tolist(), st["refs"].tolist()

    def leave(slot):
        for p in table[slot]:
            if p >= 0:
                refs[p] -= 1
        table[slot], lens[slot] = [-1] * len(table[slot]), 0

    def ints(v):
        return torch.tensor(v, dtype=torch.int32)

    if case["do"] == "turnover":
        for slot in st["dst"].tolist():
            leave(slot)
        free = [p for p, r in enumerate(refs) if r == 0]
        for slot, n in zip(st["dst"].tolist(), st["enter"].tolist()):
            for j in range(-(-n // page)):
                table[slot][j] = free.pop(0)
                refs[table[slot][j]] = 1
            lens[slot] = n
        return dict(table=ints(table), seq_lens=ints(lens), refs=ints(refs), missing=ints([0]))
    pages, scales = st["pages"].double(), st["scales"].double()
    if case["do"] == "fork":
        src, dst = st["src"].tolist(), st["dst"].tolist()
        for slot in dst:
            leave(slot)
        free = [p for p, r in enumerate(refs) if r == 0]
        for a, b in zip(src, dst):
            lens[b] = lens[a]
            for j in range(-(-lens[a] // page)):
                p = table[a][j]
                if (j + 1) * page > lens[a]:
                    fresh = free.pop(0)
                    pages[:, fresh], scales[:, fresh] = pages[:, p].clone(), scales[:, p].clone()
                    p = fresh
                table[b][j] = p
                refs[p] += 1
        return dict(table=ints(table), seq_lens=ints(lens), refs=ints(refs), missing=ints([0]), pages=pages, scales=scales)
    live = [p for p, r in enumerate(refs) if r]
    holes = [p for p in range(len(live)) if not refs[p]]
    to = {p: p if p < len(live) else holes.pop(0) for p in live}
    out_pages, out_scales = st["out"]["pages"].double(), st["out"]["scales"].double()
    out_refs = [0] * out_pages.shape[1]
    for p, o in to.items():
        out_pages[:, o], out_scales[:, o], out_refs[o] = pages[:, p], scales[:, p], refs[p]
    return dict(pages=out_pages, scales=out_scales, table=ints([[to.get(p, -1) for p in row] for row in table]),
                refs=ints(out_refs), missing=ints([0]))


def _exact_logits(st):
    """One row at a time on the host."""
    out = st["logits"].double().cpu()
    for i in range(out.shape[0]):
        row, n, first = out[i], int(st["token_lens"][i]), int(st["prompt_lens"][i])
        ids = st["tokens"][i, :n].long().cpu()
        r, f, p = (float(st[k][i]) for k in ("repetition", "frequency", "presence"))
        held = torch.unique(ids)
        row[held] = torch.where(row[held] > 0, row[held] / r, row[held] * r)
        made, times = torch.unique(ids[first:], return_counts=True)
        row[made] -= f * times.double() + p
        a, b = st["bias_offsets"][i:i + 2].tolist()
        row.index_add_(0, st["bias_ids"][a:b].long().cpu(), st["bias_values"][a:b].double().cpu())
        if st["allowed"] is not None:
            bits = (st["allowed"][i].cpu()[:, None] >> torch.arange(32, dtype=torch.int32)) & 1
            row[bits.flatten()[:row.numel()] == 0] = -math.inf
    return out
