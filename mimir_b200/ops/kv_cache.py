"""Serving over an 8-bit paged key/value cache: writing it, attending over it, moving its pages.

The reference decodes with a static cache in the model's type and an additive mask
(``src/mimir/model/layers.py:107-167``).  Here a cache holds e4m3 bytes in pages that sequences
share, with one power-of-two scale for 16 tokens of one head:

* ``pages`` float8_e4m3fn ``[pages, 2, kv_heads, page_size, 128]``: keys, then values.  Page operations
  take all layers at once, ``[layers, pages, ...]``; a layer's slice is what the others take.
* ``scales`` float32 ``[pages, 2, kv_heads, page_size / 16]``: a value is its byte times its scale.  A
  block of 16 that is given a value that is not finite gets the scale NaN: what sees it is NaN.
* ``page_table`` int32 ``[slots, width]``: the page of tokens ``page_size * j ...`` of a slot, -1 for none.
* ``seq_lens`` int32 ``[slots]``, ``ref_counts`` int32 ``[pages]`` (0: a free page).

A batch of new tokens is ``seqs`` (int32, the slot of each sequence, each at most once) and ``cu_new``
(int32, one more entry): sequence ``i`` has the rows ``cu_new[i]:cu_new[i + 1]``, and they are the last
tokens of its slot: :func:`cache_reserve` has counted them in ``seq_lens`` already.

On CUDA every function runs kernels of ``csrc/kv_cache.cu``, ``csrc/cache_attention.cu`` (few rows) and
``csrc/cache_prompt.cu`` (many) on the current stream and does not synchronise.  Arguments of a wrong type
or shape raise ``ValueError``; slots, pages and lengths that lie in device memory are checked by the
kernels: a bad one is skipped and reported by :func:`mimir_b200.ops._ext.check_kernel_status`.  On the
CPU the PyTorch formulations below run, which also take other head dimensions and float32 rows.
"""
from __future__ import annotations

import math

import torch

from mimir_b200.ops._ext import KernelTimeout, available, ext, kernels_enabled

BLOCK = 16       # tokens that share a scale
MIN_EXPONENT = -32
PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_SEQUENCES = 4096  # of one cache_reserve or cache_fork on CUDA


def cache_status(device: torch.device) -> int:
    """The first code that a cache kernel on ``device`` has reported since the last read (0: none).  Waits for the
    current stream."""
    if device.type != "cuda" or not available():
        return 0
    return int(ext().cache_status(device.index if device.index is not None else torch.cuda.current_device()))


def check_cache_status(device: torch.device) -> None:
    """Raise :class:`mimir_b200.ops._ext.KernelTimeout` where a cache kernel reported a call whose results are not
    valid: a slot, page or length that it does not have, or a wait that ran out."""
    code = cache_status(device)
    if code:
        raise KernelTimeout(f"kv_cache kernels reported code {code}: "
                            f"{('bad slot', 'bad page', 'bad length', 'wait timed out')[min(code, 4) - 1]}")


def _need(condition: bool, message: str) -> None:
    if not condition:
        raise ValueError(message)


def _check_ints(dev, **tensors) -> None:
    for name, (t, ndim) in tensors.items():
        _need(t.dtype == torch.int32 and t.ndim == ndim and t.is_contiguous() and t.device == dev,
              f"{name} must be a contiguous int32 tensor of {ndim} dimension(s) on {dev}")


def _check_pool(pages, scales, lead: int) -> None:
    _need(pages.dtype == torch.float8_e4m3fn and pages.ndim == 5 + lead and pages.is_contiguous(),
          f"pages must be a contiguous float8_e4m3fn tensor of {5 + lead} dimensions")
    _need(pages.shape[lead + 1] == 2, "pages must be [pages, 2, kv_heads, page_size, head_dim]")
    _need(pages.shape[lead + 3] in PAGE_SIZES,
          f"page_size must be 16, 32, 64, 128 or 256, not {pages.shape[lead + 3]}")
    _need(scales.dtype == torch.float32 and scales.is_contiguous()
          and scales.shape == (*pages.shape[:lead + 3], pages.shape[lead + 3] // BLOCK),
          "scales must be [pages, 2, kv_heads, page_size / 16]")


def _check_batch(page_table, seq_lens, seqs, cu_new, dev) -> None:
    _check_ints(dev, page_table=(page_table, 2), seq_lens=(seq_lens, 1), seqs=(seqs, 1), cu_new=(cu_new, 1))
    _need(seq_lens.shape[0] == page_table.shape[0], "seq_lens needs one length for each row of page_table")
    _need(cu_new.shape[0] == seqs.shape[0] + 1, "cu_new needs one more entry than seqs")


def _bounds(cu_new, rows: int) -> list[int]:
    bounds = cu_new.tolist()
    _need(all(0 <= a <= b <= rows for a, b in zip(bounds, bounds[1:])), f"cu_new must rise from 0 to at most {rows} rows")
    return bounds


# ---------------------------------------------------------------------------------- append
def cache_append(q, k, v, cos, sin, pages, scales, page_table, seq_lens, seqs, cu_new):
    """Rotate new q and k, write k and v to the cache and return the rotated q.

    ``q`` ``[tokens, heads, 128]``, ``k`` and ``v`` ``[tokens, kv_heads, 128]`` (bfloat16 or float16,
    any token and head strides that keep 16-byte alignment: slices of a packed projection are fine);
    ``cos`` and ``sin`` float32 ``[positions, 128]``, indexed by a token's position in its sequence.
    Rows before ``cu_new[0]`` and beyond ``cu_new[-1]`` give zeros.  Positions and sums are float32; q is rounded
    once to its type, k and v once to the 8 bits.  A block that grows beyond its scale has its older tokens
    rounded again.
    """
    if kernels_enabled(pages):
        return ext().cache_append(q, k, v, cos, sin, pages, scales, page_table, seq_lens, seqs, cu_new)
    return cache_append_reference(q, k, v, cos, sin, pages, scales, page_table, seq_lens, seqs, cu_new)


def _rotate(x, cos, sin):
    x = x.float()
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat((-x[..., half:], x[..., :half]), dim=-1) * sin[:, None]


def block_exponent(amax: torch.Tensor) -> torch.Tensor:
    """Smallest ``e >= -32`` with ``amax <= 448 * 2**e``."""
    mantissa, exponent = torch.frexp(amax)  # of zero: an exponent of zero
    e = (exponent - 9 + (mantissa > 0.875)).clamp_min(MIN_EXPONENT)
    return torch.where(amax > 0, e, torch.full_like(e, MIN_EXPONENT))


def cache_append_reference(q, k, v, cos, sin, pages, scales, page_table, seq_lens, seqs, cu_new):
    """PyTorch formulation of :func:`cache_append`, a block at a time."""
    dev = pages.device
    _check_pool(pages, scales, 0)
    _check_batch(page_table, seq_lens, seqs, cu_new, dev)
    _need(q.ndim == 3 and k.ndim == 3 and k.shape == v.shape and q.shape[0] == k.shape[0]
          and k.shape[1:] == (pages.shape[2], pages.shape[4]) and q.shape[2] == k.shape[2],
          "q, k and v must be [tokens, heads, head_dim] with as many tokens and the pages' heads")
    _need(q.shape[1] % k.shape[1] == 0,
          f"query heads {q.shape[1]} must be divisible by key/value heads {k.shape[1]}")
    _need(q.dtype == k.dtype == v.dtype, "q, k and v must have one type")
    _need(cos.shape == sin.shape and cos.ndim == 2 and cos.shape[1] == q.shape[2],
          "cos and sin must be float32 tables [positions, head_dim]")
    page = pages.shape[3]
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    bounds, slots, lens = _bounds(cu_new, q.shape[0]), seqs.tolist(), seq_lens.tolist()
    for i, slot in enumerate(slots):
        first, end = bounds[i], bounds[i + 1]
        start = lens[slot] - (end - first)
        _need(0 <= start and lens[slot] <= cos.shape[0], f"slot {slot} has no room for its new tokens or no positions")
        at = torch.arange(start, lens[slot], device=dev)
        out[first:end] = _rotate(q[first:end], cos[at], sin[at]).to(q.dtype)
        new = torch.stack((_rotate(k[first:end], cos[at], sin[at]), v[first:end].float()))  # [2, tokens, kv, d]
        pos = start
        while pos < lens[slot]:
            stop = min(lens[slot], (pos // BLOCK + 1) * BLOCK)
            which, inside = int(page_table[slot, pos // page]), pos % page
            block, off = inside // BLOCK, inside % BLOCK
            x = new[:, pos - start:stop - start].transpose(1, 2)                 # [2, kv, tokens, d]
            finite = torch.isfinite(x)
            poisoned = ~finite.all(-1).all(-1)
            x = torch.where(finite, x, torch.zeros_like(x))
            e = block_exponent(x.abs().amax((-1, -2)))
            scale = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
            bytes_ = pages[which, :, :, block * BLOCK:(block + 1) * BLOCK]       # [2, kv, 16, d]
            if off:
                was = scales[which, :, :, block]
                poisoned = poisoned | ~torch.isfinite(was)
                was = torch.where(torch.isfinite(was), was, torch.zeros_like(was))
                scale = torch.maximum(scale, was)
                older = bytes_[:, :, :off].float()
                again = older * torch.where(was > 0, was / scale, torch.ones_like(was))[..., None, None]
                bytes_[:, :, :off] = again.to(pages.dtype)
            bytes_[:, :, off:off + stop - pos] = (x / scale[..., None, None]).to(pages.dtype)
            scales[which, :, :, block] = torch.where(poisoned, torch.full_like(scale, math.nan), scale)
            pos = stop
    return out


# ---------------------------------------------------------------------------------- attention
def cache_attention(q, pages, scales, page_table, seq_lens, seqs, cu_new, prefix_lens=None, *, softmax_scale=None,
                    max_new=None):
    """Attention of the new tokens' queries over their sequences' cached keys and values.

    ``q`` ``[tokens, heads, 128]`` (rotated; bfloat16 or float16); returns the same shape and type.
    A token at position ``p`` sees the positions up to ``p``; where ``p`` lies in the first
    ``prefix_lens[i]`` (int32, optional) of its sequence it sees all of those (the prefix-LM rule of
    :func:`mimir_b200.ops.prefixlm_attention`).  A token that sees nothing, and rows before
    ``cu_new[0]`` or beyond ``cu_new[-1]``, give zeros.  ``softmax_scale`` is ``head_dim ** -0.5`` by default.

    ``max_new`` (the most new tokens of one sequence, if known on the host) lets few rows take a narrower
    kernel; it changes no result beyond rounding.
    """
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    if kernels_enabled(pages):
        return ext().cache_attention(q, pages, scales, page_table, seq_lens, seqs, cu_new, prefix_lens, softmax_scale,
                                     0 if max_new is None else max_new)
    return cache_attention_reference(q, pages, scales, page_table, seq_lens, seqs, cu_new, prefix_lens,
                                     softmax_scale=softmax_scale)


def cache_values(pages, scales, page_table, slot: int, length: int):
    """Keys and values ``[2, kv_heads, length, head_dim]`` of a slot, float32."""
    page = pages.shape[3]
    at = page_table[slot, :-(-length // page)].long()
    both = pages[at].float().unflatten(3, (-1, BLOCK)) * scales[at][..., None, None]    # [n, 2, kv, blocks, 16, d]
    return both.flatten(3, 4).permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :length]


def cache_attention_reference(q, pages, scales, page_table, seq_lens, seqs, cu_new, prefix_lens=None, *,
                              softmax_scale=None):
    """PyTorch formulation of :func:`cache_attention`, a sequence at a time."""
    dev = pages.device
    _check_pool(pages, scales, 0)
    _check_batch(page_table, seq_lens, seqs, cu_new, dev)
    kv = pages.shape[2]
    _need(q.ndim == 3 and q.shape[2] == pages.shape[4], "q must be [tokens, heads, head_dim]")
    _need(q.shape[1] % kv == 0, f"query heads {q.shape[1]} must be divisible by key/value heads {kv}")
    if prefix_lens is not None:
        _check_ints(dev, prefix_lens=(prefix_lens, 1))
        _need(prefix_lens.shape[0] == seqs.shape[0], "prefix_lens needs one length for each of seqs")
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    bounds, slots = _bounds(cu_new, q.shape[0]), seqs.tolist()
    prefixes = [0] * len(slots) if prefix_lens is None else prefix_lens.tolist()
    for i, slot in enumerate(slots):
        first, end, length = bounds[i], bounds[i + 1], int(seq_lens[slot])
        if first == end or length == 0:
            continue
        k, v = cache_values(pages, scales, page_table, slot, length)
        pos = torch.arange(length - (end - first), length, device=dev)
        limit = torch.where(pos < prefixes[i], torch.clamp_min(pos + 1, prefixes[i]), pos + 1).clamp(0, length)
        seen = torch.arange(length, device=dev) < limit[:, None]
        rows = q[first:end].float().unflatten(1, (kv, -1))                              # [t, kv, group, d]
        s = torch.einsum("tkgd,kjd->kgtj", rows, k) * scale
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        lost = torch.isnan(v)  # a poisoned block reaches the rows that see it, and no other
        p = p / torch.where(total == 0, torch.ones_like(total), total)
        o = torch.einsum("kgtj,kjd->tkgd", p, torch.where(lost, torch.zeros_like(v), v))
        if lost.any():
            reached = torch.einsum("tj,kjd->tkd", seen.float(), lost.float()) > 0
            o = o.masked_fill(reached[:, :, None], math.nan)
        out[first:end] = o.flatten(1, 2).to(q.dtype)
    return out


# ---------------------------------------------------------------------------------- pages
def _slots(value, name: str, page_table) -> torch.Tensor:
    """``value`` (int32 tensor, or slots known on the host) on the table's device."""
    if isinstance(value, torch.Tensor):
        return value
    slots = [int(s) for s in value]
    _need(all(0 <= s < page_table.shape[0] for s in slots), f"{name} must be slots of the page table")
    _need(len(set(slots)) == len(slots) or name == "src", f"{name} must name each slot once")
    return torch.tensor(slots, dtype=torch.int32).to(page_table.device, non_blocking=True)


def cache_reserve(page_table, seq_lens, ref_counts, seqs, counts, page_size: int):
    """Make room for ``counts[i]`` more tokens of slot ``seqs[i]`` and count them in ``seq_lens``.

    Free pages are taken lowest first in the order of the batch; the whole batch is served, or nothing
    changes.  Returns an int32 tensor of one: 0 (done), the number of pages that lack, or -1 (a slot,
    count or length that is not possible).  Read it where the host waits anyway.
    """
    seqs = _slots(seqs, "seqs", page_table)
    if not isinstance(counts, torch.Tensor):
        counts = torch.tensor([int(c) for c in counts], dtype=torch.int32).to(page_table.device, non_blocking=True)
    if kernels_enabled(page_table):
        return ext().cache_reserve(page_table, seq_lens, ref_counts, seqs, counts, page_size)
    dev = page_table.device
    _check_ints(dev, page_table=(page_table, 2), seq_lens=(seq_lens, 1), ref_counts=(ref_counts, 1), seqs=(seqs, 1),
                counts=(counts, 1))
    _need(page_size in PAGE_SIZES, f"page_size must be 16, 32, 64, 128 or 256, not {page_size}")
    _need(counts.shape[0] == seqs.shape[0], "counts needs one entry for each of seqs")
    lens, need = seq_lens.tolist(), []
    for slot, count in zip(seqs.tolist(), counts.tolist()):
        if not 0 <= slot < len(lens) or count < 0 or -(-(lens[slot] + count) // page_size) > page_table.shape[1]:
            return torch.full((1,), -1, dtype=torch.int32, device=dev)
        have = -(-lens[slot] // page_size)
        need += [(slot, j) for j in range(have, -(-(lens[slot] + count) // page_size))]
    free = torch.nonzero(ref_counts == 0).flatten().tolist()
    if len(free) < len(need):
        return torch.full((1,), len(need) - len(free), dtype=torch.int32, device=dev)
    for (slot, j), page in zip(need, free):
        page_table[slot, j] = page
        ref_counts[page] = 1
    seq_lens[seqs.long()] += counts
    return torch.zeros(1, dtype=torch.int32, device=dev)


def cache_free(page_table, seq_lens, ref_counts, seqs) -> None:
    """Empty the slots ``seqs``: their pages lose a holder, and are free where it was the last."""
    seqs = _slots(seqs, "seqs", page_table)
    if kernels_enabled(page_table):
        return ext().cache_free(page_table, seq_lens, ref_counts, seqs)
    _check_ints(page_table.device, page_table=(page_table, 2), seq_lens=(seq_lens, 1), ref_counts=(ref_counts, 1),
                seqs=(seqs, 1))
    at = seqs.long()
    held = page_table[at]
    ref_counts.index_add_(0, held[held >= 0].long(), torch.full_like(held[held >= 0], -1))
    page_table[at] = -1
    seq_lens[at] = 0


def cache_fork(pages, scales, page_table, seq_lens, ref_counts, src, dst):
    """Slot ``dst[i]`` becomes a copy of slot ``src[i]`` (all layers: ``pages [layers, pages, ...]``).

    What ``dst[i]`` held is freed.  Full pages are shared; a last page that is partly filled is copied
    to a free one, because both sequences write on in it.  A slot may be the source of several, but
    not both source and destination.  Returns what :func:`cache_reserve` returns; where pages
    lack, every destination is left empty.
    """
    if not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
        _need(not set(map(int, src)) & set(map(int, dst)), "a slot cannot be both source and destination")
    src, dst = _slots(src, "src", page_table), _slots(dst, "dst", page_table)
    if kernels_enabled(page_table):
        return ext().cache_fork(pages, scales, page_table, seq_lens, ref_counts, src, dst)
    dev = page_table.device
    _check_pool(pages, scales, 1)
    _need(src.shape == dst.shape, "src and dst must have as many slots")
    cache_free(page_table, seq_lens, ref_counts, dst)
    page = pages.shape[4]
    pairs, copies = list(zip(src.tolist(), dst.tolist())), []
    for a, b in pairs:
        length = int(seq_lens[a])
        whole = length // page
        page_table[b, :whole] = page_table[a, :whole]
        ref_counts.index_add_(0, page_table[a, :whole].long(), torch.ones(whole, dtype=torch.int32, device=dev))
        seq_lens[b] = length
        if length % page:
            copies.append((a, b, whole))
    free = torch.nonzero(ref_counts == 0).flatten().tolist()
    if len(free) < len(copies):
        cache_free(page_table, seq_lens, ref_counts, dst)
        return torch.full((1,), len(copies) - len(free), dtype=torch.int32, device=dev)
    for (a, b, j), fresh in zip(copies, free):
        old = int(page_table[a, j])
        page_table[b, j] = fresh
        ref_counts[fresh] = 1
        pages[:, fresh] = pages[:, old]
        scales[:, fresh] = scales[:, old]
    return torch.zeros(1, dtype=torch.int32, device=dev)


def cache_copy(pages, scales, src, dst) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every layer (int32 tensors; -1 skips an entry; no page
    may be both read and written, nor written twice)."""
    if kernels_enabled(pages):
        return ext().cache_copy(pages, scales, src, dst)
    _check_pool(pages, scales, 1)
    _check_ints(pages.device, src=(src, 1), dst=(dst, 1))
    keep = (src >= 0) & (dst >= 0)
    pages.view(torch.uint8)[:, dst[keep].long()] = pages.view(torch.uint8)[:, src[keep].long()]
    scales[:, dst[keep].long()] = scales[:, src[keep].long()]


def cache_compact(pages, scales, page_table, ref_counts, out=None):
    """Move the pages in use to the front of the pool, in place or into another pool.

    With ``n`` pages in use, those below ``n`` keep their index and the j-th one from there on goes to the
    j-th free one below.  ``out`` is ``(pages, scales, page_table, ref_counts)`` of a pool of another
    size (smaller to give memory back, larger to grow); without it the pool's own tensors change.
    Returns an int32 tensor of one: 0, or the number of pages that ``out`` lacks (nothing is written then).
    """
    to_pages, to_scales, to_table, to_counts = (pages, scales, page_table, ref_counts) if out is None else out
    if kernels_enabled(page_table):
        return ext().cache_compact(pages, scales, page_table, ref_counts, to_pages, to_scales, to_table, to_counts)
    dev = page_table.device
    _check_pool(pages, scales, 1)
    _check_pool(to_pages, to_scales, 1)
    _check_ints(dev, page_table=(page_table, 2), ref_counts=(ref_counts, 1))
    live = torch.nonzero(ref_counts).flatten()
    n = live.numel()
    if n > to_counts.numel():
        return torch.full((1,), n - to_counts.numel(), dtype=torch.int32, device=dev)
    holes = torch.nonzero(ref_counts[:n] == 0).flatten()
    to = torch.full_like(ref_counts, -1)
    to[live[live < n]] = live[live < n].to(torch.int32)
    to[live[live >= n]] = holes.to(torch.int32)
    at, counts = to[live].long(), ref_counts[live].clone()
    moved_pages, moved_scales = pages.view(torch.uint8)[:, live].clone(), scales[:, live].clone()
    to_pages.view(torch.uint8)[:, at] = moved_pages
    to_scales[:, at] = moved_scales
    to_table.copy_(torch.where(page_table >= 0, to[page_table.clamp_min(0).long()], torch.full_like(page_table, -1)))
    to_counts.zero_()
    to_counts[at] = counts
    return torch.zeros(1, dtype=torch.int32, device=dev)
