"""The kernels of the 8-bit paged key/value cache and of the logits operators against 64-bit formulas.

Tolerances are derived, element by element, from the roundings that the kernels make (see
``attention64``); bytes, scales, tables and counts have to be equal."""
import math

import pytest
import torch

from mimir_b200 import ops
from mimir_b200.ops._ext import KernelTimeout, check_kernel_status, ext, kernel_status
from mimir_b200.ops.kv_cache import BLOCK, cache_append_reference, cache_values
from mimir_b200.ops.logits import process_logits_reference

from test_kv_cache import drive_pages, ints, pool, tables

pytestmark = pytest.mark.gpu
DIM = 128
DEV = torch.device("cuda", 0)


def on_gpu(st):
    return {k: t.to(DEV) for k, t in st.items()}


def filled(lens, kv, page, seed=0, spread=1.0, extra=3, first_page=0):
    """A pool that holds ``lens`` tokens in each slot, pages in any order."""
    gen = torch.Generator(DEV).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1) + 1
    pages = sum(need) + extra
    x = torch.randn(pages, 2, kv, page // BLOCK, BLOCK, DIM, generator=gen, device=DEV)
    e = torch.round(spread * torch.randn(pages, 2, kv, page // BLOCK, generator=gen, device=DEV)).to(torch.int32) - 7
    st = dict(pages=(x * 100).clamp(-448, 448).to(torch.float8_e4m3fn).flatten(3, 4), scales=torch.ldexp(torch.ones_like(e, dtype=torch.float32), e),
              table=torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV), lens=ints(lens).to(DEV))
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32).tolist()
    for i, n in enumerate(need):
        st["table"][i, :n] = ints([order.pop() for _ in range(n)]).to(DEV)
    return st


def attention64(q, st, seqs, counts, prefix=None, softmax_scale=DIM ** -0.5, p_bits=11):
    """(64-bit attention, bound of the kernel's error), a sequence at a time.

    The bound adds up: a score is a sum of 128 exact products in fp32 (its error at most 128 * 2^-24 of the sum of
    their magnitudes, times two for the accumulator's own order, and as much again relative to the probability);
    exp2 and the sums add under 2^-18; a probability is rounded to ``p_bits`` bits, or below fp16's normal
    range, beside the largest product p * scale, to 2^-25 of it (the maximum may lag by 2^8 without loss,
    it then lies higher in the range); the result is rounded to its type."""
    kv = st["pages"].shape[2]
    out = torch.zeros_like(q, dtype=torch.float64)
    bound = torch.zeros_like(out)
    unit = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11  # half a step of 8 or 11 significant bits
    row = 0
    for i, (slot, count) in enumerate(zip(seqs, counts)):
        n = int(st["lens"][slot])
        if count and n:
            k, v = cache_values(st["pages"], st["scales"], st["table"], slot, n).double()
            pos = torch.arange(n - count, n, device=DEV)
            limit = pos + 1 if prefix is None else torch.where(pos < prefix[i], torch.clamp_min(pos + 1, prefix[i]), pos + 1)
            seen = torch.arange(n, device=DEV) < limit.clamp(0, n)[:, None]
            x = q[row:row + count].double().unflatten(1, (kv, -1))
            s = torch.einsum("tkgd,kjd->tkgj", x, k) * softmax_scale
            off = torch.einsum("tkgd,kjd->tkgj", x.abs(), k.abs()) * softmax_scale * 2.0 ** -16
            p = torch.softmax(s.masked_fill(~seen[:, None, None], -math.inf), -1)
            p = torch.nan_to_num(p)  # a row that sees nothing
            o = torch.einsum("tkgj,kjd->tkgd", p, v)
            rel = 2 * off + 2.0 ** -18 + 2.0 ** -p_bits
            err = torch.einsum("tkgj,kjd->tkgd", p * rel, v.abs()) + (p * (2 * off + 2.0 ** -18)).sum(-1)[..., None] * o.abs()
            at = st["table"][slot, :-(-n // st["pages"].shape[3])].long()
            size = st["scales"][at, 1].permute(1, 0, 2).flatten(1).double().repeat_interleave(BLOCK, 1)[:, :n]
            most = (p * size[None, :, None]).amax(-1)[..., None]
            err = err + 2.0 ** -25 * 448 * n * most
            out[row:row + count] = o.flatten(1, 2)
            bound[row:row + count] = (err + unit * (o.abs() + err)).flatten(1, 2)
        row += count
    return out, bound + 1e-30


def attend(q, st, seqs, cu, prefix=None, softmax_scale=None, max_new=None, kernel=0):
    """``ops.cache_attention``, or with ``kernel`` one of its two kernels whatever the sizes."""
    args = (q, st["pages"], st["scales"], st["table"], st["lens"], ints(seqs).to(DEV), ints(cu).to(DEV),
            None if prefix is None else ints(prefix).to(DEV))
    if kernel:
        return ext().cache_attention(*args, softmax_scale or DIM ** -0.5, max_new or 0, kernel)
    return ops.cache_attention(*args, max_new=max_new, softmax_scale=softmax_scale)


def check_attention(st, seqs, counts, heads, dtype=torch.bfloat16, prefix=None, seed=5, extra_rows=0, max_new=None, q=None,
                    softmax_scale=None, kernel=0):
    gen = torch.Generator(DEV).manual_seed(seed)
    total = sum(counts)
    if q is None:
        q = (1.5 * torch.randn(total + extra_rows, heads, DIM, generator=gen, device=DEV)).to(dtype)
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    out = attend(q, st, seqs, cu, prefix, softmax_scale, max_new, kernel)
    ref, bound = attention64(q, st, seqs, counts, prefix, softmax_scale or DIM ** -0.5, p_bits=11)
    check_kernel_status(DEV)
    assert out.dtype == q.dtype and out.shape == q.shape and torch.isfinite(out).all()
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), f"{(err / bound).max().item():.2f} of the bound"
    assert not out[total:].any()
    return q, out


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_single_tokens_at_every_edge(page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000]
    st = filled(lens, 2, page)
    check_attention(st, list(range(len(lens))), [1] * len(lens), 8, max_new=1)
    check_attention(st, list(range(len(lens)))[::-1], [1] * len(lens), 8)  # without the hint


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (5, 5), (8, 1), (16, 4), (12, 4), (24, 2), (20, 20)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_groups_and_types(heads, kv, dtype):
    st = filled([70, 9, 300], kv, 32, seed=heads)
    check_attention(st, [2, 0, 1], [1, 1, 1], heads, dtype, max_new=1)
    for kernel in (0, 1, 2):
        check_attention(st, [2, 0, 1], [5, 70, 2], heads, dtype, max_new=70, kernel=kernel)


@pytest.mark.parametrize("counts", [[2, 3, 1, 4], [0, 17, 0, 33], [64, 65, 1, 200], [300, 1, 129, 256]])
@pytest.mark.parametrize("prefix", [None, "all", "half"])
def test_several_tokens_and_prefixes(counts, prefix):
    lens = [c + old for c, old in zip(counts, [5, 0, 700, 0])]
    st = filled(lens, 2, 64, seed=sum(counts))
    p = None if prefix is None else [n if prefix == "all" else n // 2 for n in lens]
    for kernel in (0, 1, 2):
        check_attention(st, [0, 1, 2, 3], counts, 8, prefix=p, extra_rows=3, max_new=max(counts), kernel=kernel)


def test_a_long_sequence_is_split_and_many_short_ones_are_not():
    st = filled([40001], 1, 128)
    check_attention(st, [0], [1], 4, max_new=1)
    lens = [1 + i % 7 for i in range(1500)]  # more sequences than one launch takes
    st = filled(lens, 1, 16)
    check_attention(st, list(range(1500)), [1] * 1500, 2, max_new=1)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_prompts_at_every_edge(page):
    """The prompt kernel: lengths and new tokens around its tiles of 128 keys and 32 tokens, many sequences."""
    counts = [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 0, 511, 1, 300]
    old = [0, 0, 1, 200, 0, 64, 0, 128, 0, 1, 57, 5, 1, 1000, 0]
    st = filled([c + o for c, o in zip(counts, old)], 5, page, seed=page)
    for prefix in (None, [c + o for c, o in zip(counts, old)], [7 * i for i in range(15)]):
        check_attention(st, list(range(15)), counts, 20, prefix=prefix, extra_rows=2, kernel=2)


def test_many_short_prompts():
    counts = [1 + (i * 7) % 50 for i in range(1100)]  # more sequences than one launch takes
    st = filled(counts, 1, 16)
    check_attention(st, list(range(1100)), counts, 4, kernel=2)


@pytest.mark.parametrize("many", [1, 31, 32, 33])
def test_prompts_in_the_order_of_their_lengths(many):
    """Up to 32 sequences the prompt kernel takes the longest first; equal and empty ones among them."""
    counts = [(i * 37) % 150 for i in range(many - 1)] + [90]
    lens = [c + (i * 53) % 90 // 30 * 30 for i, c in enumerate(counts)]
    st = filled([max(n, 1) for n in lens], 3, 32)
    for prefix in (None, lens):
        check_attention(st, list(range(many))[::-1], counts[::-1], 12, prefix=prefix and prefix[::-1], extra_rows=5, kernel=2)


def test_results_do_not_depend_on_the_run():
    st = filled([5000, 77, 20000], 4, 64)
    q, first = check_attention(st, [0, 1, 2], [1, 1, 1], 16, max_new=1)
    for _ in range(5):
        assert torch.equal(check_attention(st, [0, 1, 2], [1, 1, 1], 16, max_new=1, q=q)[1], first)


def test_value_scales_far_apart():
    """Blocks whose scales differ by 2^40: small weights of large values and large weights of small ones."""
    st = filled([500, 33], 1, 16, spread=10.0)
    st["scales"][:, 0] = 2.0 ** -7  # keys as usual
    check_attention(st, [0, 1], [1, 1], 4, max_new=1)
    for kernel in (1, 2):
        check_attention(st, [0, 1], [40, 33], 4, max_new=40, kernel=kernel)


def test_queries_of_any_size_and_a_scale_of_ones_own():
    st = filled([200, 100], 2, 64)
    gen = torch.Generator(DEV).manual_seed(1)
    q = torch.randn(2, 8, DIM, generator=gen, device=DEV)
    for factor, scale in ((2.0 ** 20, DIM ** -0.5 * 2.0 ** -20), (2.0 ** -30, DIM ** -0.5 * 2.0 ** 30), (1.0, 0.0)):
        for kernel in (1, 2):
            check_attention(st, [0, 1], [1, 1], 8, q=(q * factor).bfloat16(), softmax_scale=scale or 1e-9, kernel=kernel)


def test_strided_queries():
    st = filled([50, 90], 2, 32)
    packed = torch.randn(9, 20, DIM, device=DEV).bfloat16()
    wide = torch.randn(8, 9, 2 * DIM, device=DEV).half().transpose(0, 1)
    for kernel in (1, 2):
        check_attention(st, [0, 1], [4, 5], 8, q=packed[:, 7:15], kernel=kernel)
        check_attention(st, [0, 1], [4, 5], 8, q=wide[..., :DIM], kernel=kernel)
    one = torch.randn(1, 8, DIM, device=DEV).bfloat16().expand(9, 8, DIM)
    check_attention(st, [0, 1], [4, 5], 8, q=one)


@pytest.mark.parametrize("kernel", [1, 2])
def test_bytes_beyond_the_length_do_not_matter(kernel):
    """NaN bytes, NaN scales and pages of others behind a sequence's end, and in pages that it does not hold."""
    for lens, counts in (([1, 17, 70], [1, 1, 1]), ([40, 150, 70], [33, 130, 2])):
        st = filled(lens, 2, 64, seed=3)
        q, want = check_attention(st, [0, 1, 2], counts, 8, kernel=kernel)
        nan = torch.tensor(0x7F, dtype=torch.uint8, device=DEV)
        held = torch.zeros(st["pages"].shape[0], dtype=torch.bool, device=DEV)
        for i, n in enumerate(lens):
            row = st["table"][i, :-(-n // 64)].long()
            held[row] = True
            inside = n - (len(row) - 1) * 64
            st["pages"].view(torch.uint8)[row[-1], :, :, inside:] = nan
            st["scales"][row[-1], :, :, -(-inside // BLOCK):] = math.nan
        st["pages"].view(torch.uint8)[~held] = nan
        st["scales"][~held] = math.nan
        got = attend(q, st, [0, 1, 2], [0, counts[0], sum(counts[:2]), sum(counts)], kernel=kernel)
        assert torch.equal(got, want)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("count,kernel", [(3, 1), (60, 1), (3, 2), (60, 2)])
def test_a_poisoned_block_reaches_the_rows_that_see_it(which, count, kernel):
    n = 100
    st = filled([n, 30], 2, 32)
    q, want = check_attention(st, [0, 1], [count, 1], 8, kernel=kernel)
    at = 98  # the block of tokens 96..99
    st["scales"][st["table"][0, at // 32].long(), which, 1, at % 32 // BLOCK] = math.nan
    got = attend(q, st, [0, 1], [0, count, count + 1], kernel=kernel)
    hit = torch.zeros(count + 1, 8, dtype=torch.bool, device=DEV)
    hit[max(0, 96 - (n - count)):count, 4:] = True  # heads of the second key/value head, from position 96 on
    assert torch.equal(torch.isnan(got).all(-1), hit) and torch.equal(torch.isnan(got).any(-1), hit)
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("kernel", [1, 2])
def test_rows_without_keys_are_zero(kernel):
    st = filled([10, 20], 1, 16)
    st["lens"][0] = 0  # an emptied slot that is still asked for
    q = torch.randn(4, 2, DIM, device=DEV).bfloat16()
    out = attend(q, st, [0, 1], [0, 1, 2], kernel=kernel)
    assert not out[0].any() and out[1].any() and not out[2:].any()
    with pytest.raises(KernelTimeout, match="kv_cache"):  # fewer tokens than new ones: reported
        check_kernel_status(DEV)
    empty = torch.zeros(0, dtype=torch.int32, device=DEV)
    out = ops.cache_attention(q, st["pages"], st["scales"], st["table"], st["lens"], empty, ints([0]).to(DEV))
    assert not out.any()


def test_offsets_beyond_32_bits():
    """Pages that lie more than 2^32 bytes into the pool."""
    page, kv, pages = 256, 4, 17000  # 256 KB each: 4.4 GB
    st = dict(pages=torch.zeros(pages, 2, kv, page, DIM, dtype=torch.float8_e4m3fn, device=DEV),
              scales=torch.full((pages, 2, kv, page // BLOCK), 2.0 ** -7, device=DEV),
              table=ints([[16999, 16990, 3]]).to(DEV), lens=ints([700]).to(DEV))
    x = (100 * torch.randn(3, 2, kv, page, DIM, device=DEV, generator=torch.Generator(DEV).manual_seed(0))).clamp(-448, 448)
    st["pages"].view(torch.uint8)[st["table"][0].long()] = x.to(torch.float8_e4m3fn).view(torch.uint8)
    check_attention(st, [0], [1], 8, max_new=1)
    for kernel in (1, 2):
        check_attention(st, [0], [300], 8, max_new=300, kernel=kernel)
    cos, sin = tables(1024, DIM)
    k = torch.randn(700, kv, DIM, device=DEV).bfloat16()
    ops.cache_append(k, k, k, cos.to(DEV), sin.to(DEV), st["pages"], st["scales"], st["table"], st["lens"],
                     ints([0]).to(DEV), ints([0, 700]).to(DEV))
    held = cache_values(st["pages"], st["scales"], st["table"], 0, 700)[1].transpose(0, 1)
    assert bool(((held - k.float()).abs() <= k.float().abs() * 2.0 ** -4 + st["scales"].max() * 2.0 ** -10).all())
    layers = st["pages"].view(2, pages // 2, 2, kv, page, DIM)
    ops.cache_copy(layers, st["scales"].view(2, pages // 2, 2, kv, -1), ints([8499, -1]).to(DEV), ints([1, 2]).to(DEV))
    assert torch.equal(layers[1, 1].view(torch.uint8), layers[1, 8499].view(torch.uint8)) and layers[1, 1].float().any()


# ---------------------------------------------------------------------------------- append
def append_both(st, q, k, v, seqs, cu, positions=2048):
    """The kernel on the GPU and the formulation on the CPU, on the same state: equal, bit for bit."""
    cos, sin = tables(positions, DIM)
    host = {name: t.cpu() for name, t in st.items()}
    want = cache_append_reference(q.cpu(), k.cpu(), v.cpu(), cos, sin, host["pages"], host["scales"], host["table"],
                                  host["lens"], ints(seqs), ints(cu))
    got = ops.cache_append(q, k, v, cos.to(DEV), sin.to(DEV), st["pages"], st["scales"], st["table"], st["lens"],
                           ints(seqs).to(DEV), ints(cu).to(DEV))
    check_kernel_status(DEV)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(st["scales"].cpu().view(torch.int32), host["scales"].view(torch.int32))
    assert torch.equal(st["pages"].cpu().view(torch.uint8), host["pages"].view(torch.uint8))
    return got


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_writes_what_the_formula_says(page, dtype):
    counts, old = [1, 5, 0, 16, 40, 1, 300], [0, 13, 9, 16, 3, 31, 1]
    heads, kv = 6, 2
    st = filled([c + o for c, o in zip(counts, old)], kv, page, spread=3.0)
    gen = torch.Generator(DEV).manual_seed(4)
    total = sum(counts) + 2  # two rows of no sequence
    size = torch.exp(3 * torch.randn(total, 1, 1, generator=gen, device=DEV))
    q, k, v = (torch.randn(total, h, DIM, generator=gen, device=DEV) for h in (heads, kv, kv))
    k, v = k * size, v * size
    v[:, :, 7] = 0
    v[20:40] = 0  # whole blocks of zeros
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    got = append_both(st, q.to(dtype), k.to(dtype), v.to(dtype), list(range(len(counts))), cu)
    assert not got[-2:].any()
    # again: nothing changes
    before = st["pages"].clone(), st["scales"].clone()
    append_both(st, q.to(dtype), k.to(dtype), v.to(dtype), list(range(len(counts))), cu)
    assert torch.equal(before[0].view(torch.uint8), st["pages"].view(torch.uint8)) and torch.equal(before[1], st["scales"])


def test_append_of_many_tokens_and_packed_projections():
    heads, kv, counts = 4, 2, [1900, 700, 3]
    st = filled([c + 10 for c in counts], kv, 64)
    packed = torch.randn(sum(counts), 2 * heads + 2 * kv, DIM, device=DEV).bfloat16()  # gate, q, k, v
    cu = [0, 1900, 2600, 2603]
    append_both(st, packed[:, heads:2 * heads], packed[:, 2 * heads:2 * heads + kv], packed[:, 2 * heads + kv:], [0, 1, 2], cu)


def test_append_of_values_that_are_not_finite():
    st = filled([33, 20], 2, 16)
    x = torch.randn(23, 2, DIM, device=DEV).bfloat16()
    k, v = x.clone(), x.clone()
    k[3, 0, 5], v[9, 1, 100], v[22, 0, 0] = math.nan, math.inf, -math.inf
    append_both(st, x, k, v, [0, 1], [0, 20, 23])
    assert torch.isnan(st["scales"]).sum() == 3
    st["lens"] += 1  # one more token into the poisoned block of the second sequence
    st["table"][1, 1] = st["table"][1, 1].clamp_min(0)
    append_both(st, x[:2], x[:2], x[:2], [1, 0], [0, 1, 2])


def test_append_extremes():
    """Zeros, the type's largest and smallest values, and a block that grows by 2^200."""
    st = filled([48], 1, 16)
    v = torch.zeros(48, 1, DIM, device=DEV)
    v[0:16] = 1e-38
    v[16, 0, 0], v[40] = 3e38, -3e38
    append_both(st, v.bfloat16(), v.bfloat16(), v.bfloat16(), [0], [0, 48])
    assert st["scales"][st["table"][0, 0].long(), 1, 0, 0] == 2.0 ** -32  # (keys of 3e38 rotate to infinities)
    st["lens"][0] = 20
    for new in (1e-12, 3e38):
        st["lens"][0] += 1
        append_both(st, v[:1].bfloat16(), v[:1].bfloat16(), torch.full((1, 1, DIM), new, device=DEV).bfloat16(), [0], [0, 1])


# ---------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("seed,slots,width,pages,page", [(0, 6, 5, 20, 16), (1, 40, 30, 500, 64), (2, 16, 300, 3001, 32)])
def test_page_operations_follow_the_model(seed, slots, width, pages, page):
    drive_pages(DEV, slots, width, pages, page, steps=50, seed=seed)
    check_kernel_status(DEV)


def test_large_bookkeeping():
    """More pages, sequences and entries than one step of the block takes."""
    slots, width, pages = 2500, 40, 60000
    table = torch.full((slots, width), -1, dtype=torch.int32, device=DEV)
    lens, refs = torch.zeros(slots, dtype=torch.int32, device=DEV), torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[::3] = 1  # held by others
    counts = [1 + (37 * i) % 600 for i in range(slots)]
    assert ops.cache_reserve(table, lens, refs, list(range(slots)), counts, 32).item() == 0
    free, at = [p for p in range(pages) if p % 3], 0
    host = table.tolist()
    for i, c in enumerate(counts):
        n = -(-c // 32)
        assert host[i] == free[at:at + n] + [-1] * (width - n)
        at += n
    assert lens.tolist() == counts and refs.sum().item() == at + 20000
    assert ops.cache_reserve(table, lens, refs, [0], [(width + 1) * 32], 32).item() == -1
    lack = ops.cache_reserve(table, lens, refs, list(range(slots)), [600] * slots, 32).item()
    need = sum(-(-(c + 600) // 32) - -(-c // 32) for c in counts)
    assert lack == need - (pages - 20000 - at) and lens.tolist() == counts
    ops.cache_free(table, lens, refs, list(range(0, slots, 2)))
    assert refs.sum().item() == 20000 + sum(-(-c // 32) for c in counts[1::2]) and (table[::2] == -1).all()


def test_bad_slots_and_pages_are_reported_and_skipped():
    st = filled([40, 40], 1, 16)
    st["table"][0, 1] = 10 ** 6
    q = torch.randn(2, 2, DIM, device=DEV).bfloat16()
    args = (st["pages"], st["scales"], st["table"], st["lens"], ints([0, 7]).to(DEV), ints([0, 1, 2]).to(DEV))
    out = ops.cache_attention(q, *args)
    assert torch.isfinite(out[1]).all() and kernel_status(DEV)["kv_cache"] in (1, 2)
    cos, sin = (t.to(DEV) for t in tables(64, DIM))
    before = st["pages"].clone()
    st["lens"][0] = 17  # the bad page
    ops.cache_append(q, q[:, :1], q[:, :1], cos, sin, *args)
    assert kernel_status(DEV)["kv_cache"] in (1, 2) and torch.equal(before.view(torch.uint8), st["pages"].view(torch.uint8))
    ops.cache_append(q, q[:, :1], q[:, :1], cos[:10], sin[:10], *args[:4], ints([1, 0]).to(DEV), args[5])
    assert kernel_status(DEV)["kv_cache"] == 3  # positions that the tables do not have
    refs = torch.ones(st["pages"].shape[0], dtype=torch.int32, device=DEV)
    ops.cache_free(st["table"], st["lens"], refs, ints([9, -1, 0]).to(DEV))
    assert kernel_status(DEV)["kv_cache"] in (1, 2)
    assert kernel_status(DEV)["kv_cache"] == 0


def test_refusals():
    st = filled([20], 2, 16)
    q, cu, seqs = torch.randn(1, 4, DIM, device=DEV).bfloat16(), ints([0, 1]).to(DEV), ints([0]).to(DEV)
    rest = (st["table"], st["lens"], seqs, cu)

    def attend(**kw):
        a = dict(q=q, pages=st["pages"], scales=st["scales"]) | kw
        return ops.cache_attention(a["q"], a["pages"], a["scales"], *kw.get("rest", rest))

    for message, kw in (("divisible", dict(q=q[:, :3])), ("bfloat16 or float16", dict(q=q.float())),
                        ("16-byte", dict(q=torch.randn(1, 4, DIM + 1, device=DEV).bfloat16()[..., 1:])),
                        ("float8", dict(pages=st["pages"].view(torch.uint8))),
                        ("scales", dict(scales=st["scales"].double())),
                        ("contiguous", dict(pages=st["pages"][:, :, :, ::2])),
                        ("int32", dict(rest=(st["table"].long(), *rest[1:]))),
                        ("on cuda", dict(rest=(st["table"].cpu(), *rest[1:]))),
                        ("one more entry", dict(rest=(*rest[:3], seqs)))):
        with pytest.raises(ValueError, match=message):
            attend(**kw)
    k, (cos, sin) = q[:, :2], (t.to(DEV) for t in tables(64, DIM))
    with pytest.raises(ValueError, match="as many tokens"):
        ops.cache_append(q, k, k[:0], cos, sin, st["pages"], st["scales"], *rest)
    with pytest.raises(ValueError, match="tables"):
        ops.cache_append(q, k, k, cos.double(), sin, st["pages"], st["scales"], *rest)
    with pytest.raises(ValueError, match="page_size"):
        ops.cache_reserve(st["table"], st["lens"], st["lens"], seqs, seqs, 48)
    with pytest.raises(ValueError, match="in place throughout"):
        layers = (st["pages"][None], st["scales"][None])
        refs = torch.zeros(st["pages"].shape[0], dtype=torch.int32, device=DEV)
        ops.cache_compact(*layers, st["table"], refs, (*layers, st["table"].clone(), refs))
    x = torch.randn(2, 40, device=DEV)
    with pytest.raises(ValueError, match="need tokens"):
        ops.process_logits(x, presence=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="ceil"):
        ops.process_logits(x, allowed=torch.zeros(2, 1, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="only where"):
        y = torch.randn(2, 80, device=DEV)
        ops.process_logits(y.view(2, 80)[:, :40], out=y.view(-1)[:80].view(2, 40))


def test_calls_follow_the_current_stream():
    """Everything of a decoding step on a side stream behind work that is still running there."""
    st = filled([600, 130], 2, 64)
    q = torch.randn(2, 8, DIM, device=DEV).bfloat16()
    cu, seqs = ints([0, 1, 2]).to(DEV), ints([0, 1]).to(DEV)
    cos, sin = (t.to(DEV) for t in tables(1024, DIM))
    k = torch.randn(2, 2, DIM, device=DEV).bfloat16()
    want = ops.cache_append(q, k, k, cos, sin, st["pages"], st["scales"], st["table"], st["lens"], seqs, cu)
    want = ops.cache_attention(want, st["pages"], st["scales"], st["table"], st["lens"], seqs, cu)
    big = torch.randn(4096, 4096, device=DEV)
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-3
        late.copy_(q)
        got = ops.cache_append(late, k, k, cos, sin, st["pages"], st["scales"], st["table"], st["lens"], seqs, cu)
        got = ops.cache_attention(got, st["pages"], st["scales"], st["table"], st["lens"], seqs, cu)
    side.synchronize()
    assert torch.equal(got, want)


def test_a_decoding_step_in_a_graph():
    st = filled([600, 130], 2, 64)
    q = torch.randn(2, 8, DIM, device=DEV).bfloat16()
    cu, seqs = ints([0, 1, 2]).to(DEV), ints([0, 1]).to(DEV)
    args = (st["pages"], st["scales"], st["table"], st["lens"], seqs, cu)
    ops.cache_attention(q, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.cache_attention(q, *args)
    for lens in ([600, 130], [3, 64], [64, 90]):
        st["lens"].copy_(ints(lens))
        q.copy_(torch.randn(2, 8, DIM))
        graph.replay()
        assert torch.equal(out, ops.cache_attention(q, *args))


# ---------------------------------------------------------------------------------- logits
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (2, 4096), (5, 4097), (2, 10007), (7, 32768)])
def test_logits_against_the_rules(rows, vocab, dtype):
    gen = torch.Generator(DEV).manual_seed(vocab)
    x = (3 * torch.randn(rows, vocab + 8, generator=gen, device=DEV)).to(dtype)[:, :vocab]  # rows with a stride
    x[0, 0] = math.inf
    x[-1, -1] = math.nan
    most = 90
    tokens = torch.randint(-2, min(vocab + 2, 40), (rows, most), generator=gen, device=DEV).to(torch.int32)
    lens = torch.randint(0, most + 1, (rows,), generator=gen, device=DEV).to(torch.int32)
    prompt = lens // 2
    rep, pres, freq = (torch.rand(rows, generator=gen, device=DEV) + a for a in (0.5, 0.0, -0.5))
    offsets = ints([0] + [40] * (rows - 1) + [67]).to(DEV) if rows > 1 else ints([3, 67]).to(DEV)
    ids = torch.randint(-1, min(vocab + 1, 9), (67,), generator=gen, device=DEV).to(torch.int32)  # many equal ones
    values = torch.randn(67, generator=gen, device=DEV)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=gen, device=DEV).to(torch.int32)
    kw = dict(tokens=tokens, token_lens=lens, prompt_lens=prompt, repetition=rep, presence=pres, frequency=freq,
              bias=(offsets, ids, values), allowed=allowed)
    for drop in ([], ["allowed"], ["bias"], ["presence", "frequency"], ["repetition"], ["token_lens", "prompt_lens"],
                 ["tokens", "token_lens", "prompt_lens", "repetition", "presence", "frequency"]):
        some = {k: v for k, v in kw.items() if k not in drop}
        got = ops.process_logits(x, **some)
        b = some.get("bias", (None, None, None))
        ref = process_logits_reference(x.double(), *(some.get(k) for k in (
            "tokens", "token_lens", "prompt_lens", "repetition", "presence", "frequency")), *b, some.get("allowed"))
        assert got.dtype == torch.float32
        # at most: a quotient, four sums and up to 67 biases, each rounded to 2^-24 of sizes under 2^8
        torch.testing.assert_close(got, ref.float(), rtol=2.0 ** -21, atol=72 * 2.0 ** -24 * 2.0 ** 8, equal_nan=True)
        assert torch.equal(got, ops.process_logits(x, **some)) or torch.isnan(got).any()
    if dtype == torch.float32:
        y = x.contiguous()
        want = ops.process_logits(y, **kw)
        assert ops.process_logits(y, **kw, out=y) is not None
        torch.testing.assert_close(y, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 5, 31, 8190, 8191, 8193, 16383])
def test_logits_of_rows_that_start_anywhere(vocab, dtype):
    gen = torch.Generator(DEV).manual_seed(vocab)
    rows = 5
    x = (3 * torch.randn(rows, vocab, generator=gen, device=DEV)).to(dtype)
    tokens = torch.randint(-2, vocab + 3, (rows, 300), generator=gen, device=DEV).to(torch.int32)
    ids = torch.randint(-2, vocab + 3, (rows * 600,), generator=gen, device=DEV).to(torch.int32)  # more than threads
    kw = dict(tokens=tokens, token_lens=ints([300, 0, 7, 299, 1]).to(DEV), prompt_lens=ints([100, 0, 3, 299, 0]).to(DEV),
              repetition=torch.rand(rows, generator=gen, device=DEV) + 0.5, presence=torch.rand(rows, generator=gen, device=DEV),
              frequency=torch.rand(rows, generator=gen, device=DEV),
              bias=(ints([0, 600, 1200, 1200, 2400, 3000]).to(DEV), ids, torch.randn(rows * 600, generator=gen, device=DEV)),
              allowed=torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=gen, device=DEV).to(torch.int32))
    want = torch.full((rows, vocab), math.nan, device=DEV)
    ref = process_logits_reference(x.double(), *(kw[k] for k in (
        "tokens", "token_lens", "prompt_lens", "repetition", "presence", "frequency")), *kw["bias"], kw["allowed"])
    ops.process_logits(x, **kw, out=want)
    # a quotient, three sums and up to 1200 biases under 2^3, each rounded to 2^-24 of sizes under 2^13
    torch.testing.assert_close(want, ref.float(), rtol=2.0 ** -21, atol=1204 * 2.0 ** -24 * 2.0 ** 13)
    for stride, first, before in ((vocab, 1, 0), (vocab, 1, 1), (vocab + 1, 0, 0), (vocab + 2, 3, 2), (vocab + 3, 2, 3),
                                  (vocab + 4, 0, 1)):
        around = torch.full((stride * rows + first + 8,), math.nan, device=DEV, dtype=dtype)
        view = around[first:first + stride * rows].view(rows, stride)[:, :vocab]
        view.copy_(x)
        out = torch.full((before + rows * vocab + 8,), 77.0, device=DEV)
        got = ops.process_logits(view, **kw, out=out[before:before + rows * vocab].view(rows, vocab))
        assert torch.equal(got, want), (stride, first, before)
        assert (out[:before] == 77).all() and (out[before + rows * vocab:] == 77).all()


def test_logits_out_that_overlaps_is_refused():
    memory = torch.zeros(64, device=DEV)
    x = memory[:40].view(2, 20)
    with pytest.raises(ValueError, match="shares no memory"):
        ops.process_logits(x, out=memory[4:44].view(2, 20))
    with pytest.raises(ValueError, match="shares no memory"):
        ops.process_logits(memory.view(torch.bfloat16)[:40].view(2, 20), out=memory[:40].view(2, 20))
    ops.process_logits(x[:, :10], out=memory[40:60].view(2, 10))


def stale(shape, dtype):
    """Leaves a freed block of NaN of this size behind: what a kernel does not write shows."""
    torch.full(shape, math.nan, dtype=dtype, device=DEV)


@pytest.mark.parametrize("heads,kv", [(8, 2), (3, 1), (20, 20), (24, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_hint_below_the_real_number_of_new_tokens(heads, kv, dtype):
    """``max_new`` chooses a kernel and changes no result, whatever it says."""
    counts, lens = [3, 1, 9, 40, 0, 2], [300, 1, 9, 5000, 7, 129]
    st = filled(lens, kv, 32, seed=heads)
    for hint in (1, 2, 9):
        stale((sum(counts), heads, DIM), dtype)
        check_attention(st, list(range(6)), counts, heads, dtype, max_new=hint, kernel=1)


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("many", [2, 40])
def test_rows_before_the_first_sequence_are_zero(kernel, many):
    counts = [3, 30] * (many // 2)
    st = filled([50, 30] * (many // 2), 2, 32)
    q = torch.randn(4 + sum(counts) + 2, 8, DIM, device=DEV).bfloat16()
    cu = [4 + sum(counts[:i]) for i in range(many + 1)]
    want = attend(q[4:-2], st, list(range(many)), [c - 4 for c in cu], kernel=kernel)
    stale(q.shape, q.dtype)
    got = attend(q, st, list(range(many)), cu, kernel=kernel)
    check_kernel_status(DEV)
    assert not got[:4].any() and not got[-2:].any() and torch.equal(got[4:-2], want)


def test_append_of_rows_before_the_first_sequence():
    st = filled([50, 30], 2, 32)
    x = torch.randn(39, 4, DIM, device=DEV).bfloat16()
    stale(x.shape, x.dtype)
    got = append_both(st, x, x[:, :2], x[:, 2:], [0, 1], [4, 7, 37])
    assert not got[:4].any() and not got[37:].any() and got[4].any()


@pytest.mark.parametrize("cu,bad", [([-3, 2, 4], [0, 1]), ([0, 2, 9], [2, 3, 4]), ([-5, -2, 3], [0, 1, 2]), ([0, 3, 1], [])])
def test_bounds_that_leave_the_rows_are_reported(cu, bad):
    """A sequence whose rows begin before the first or end after the last one is skipped: its rows are zeros."""
    st = filled([60, 70], 2, 32)
    q = torch.randn(5, 8, DIM, device=DEV).bfloat16()
    for kernel in (1, 2):
        stale(q.shape, q.dtype)
        out = attend(q, st, [0, 1], cu, kernel=kernel)
        assert torch.isfinite(out).all() and not out[bad].any()
        assert kernel_status(DEV)["kv_cache"] == 3
    cos, sin = (t.to(DEV) for t in tables(128, DIM))
    before = st["pages"].clone(), st["scales"].clone()
    stale(q.shape, q.dtype)
    out = ops.cache_append(q, q[:, :2], q[:, :2], cos, sin, st["pages"], st["scales"], st["table"], st["lens"],
                           ints([0, 1]).to(DEV), ints(cu).to(DEV))
    assert torch.isfinite(out).all() and not out[bad].any()
    assert kernel_status(DEV)["kv_cache"] == 3
    held = [i for i in range(2) if cu[i] < 0 or cu[i + 1] > 5]  # the sequences that are skipped
    for i in held:
        rows = st["table"][i, :3].long()
        rows = rows[rows >= 0]
        assert torch.equal(st["pages"].view(torch.uint8)[rows], before[0].view(torch.uint8)[rows])


@pytest.mark.parametrize("many", [1, 5, 33, 160, 161, 1024, 1025, 2100])
def test_the_line_of_sequences(many):
    """Shares of whole units over few and many sequences, beyond one launch's too; both widths of row tiles."""
    lens = [1 + (i * 331) % 200 for i in range(many)]
    lens[0] = 9000 if many < 40 else 700
    st = filled(lens, 2, 64, seed=many)
    order = [(i * 17) % many if many % 17 else i for i in range(many)]
    check_attention(st, order, [1] * many, 8, max_new=1, kernel=1)
    counts = [min(lens[s], 1 + s % 6) for s in order]
    check_attention(st, order, counts, 8, kernel=1)


@pytest.mark.parametrize("offsets", [[2 ** 31 - 1, 2 ** 31 - 1, 2], [-5, 2, 2 ** 31 - 1], [2 ** 31 - 300, 0, -2 ** 31], [3, 2, 1]])
def test_bias_offsets_outside_the_list(offsets):
    x = torch.randn(2, 100, device=DEV)
    ids, values = ints([4, 4, 9]).to(DEV), torch.tensor([1.0, 2.0, 5.0], device=DEV)
    want = x.clone()
    for row in range(2):
        for i in range(max(offsets[row], 0), min(offsets[row + 1], 3)):
            want[row, ids[i].item()] += values[i]
    got = ops.process_logits(x, bias=(ints(offsets).to(DEV), ids, values))
    torch.testing.assert_close(got, want, rtol=0, atol=3 * 2.0 ** -24 * 2.0 ** 4)  # three sums under 2^4
    host = ops.process_logits(x.cpu(), bias=(ints(offsets), ids.cpu(), values.cpu()))
    torch.testing.assert_close(host, want.cpu(), rtol=0, atol=3 * 2.0 ** -24 * 2.0 ** 4)


def test_forks_of_a_negative_length():
    """Reported, read as no tokens: nothing outside the table is looked at."""
    st = {k: t.to(DEV) for k, t in pool(8, 1, 16, DIM, 3, 4, layers=2).items()}
    book = (st["table"], st["lens"], st["refs"])
    ops.cache_reserve(*book, [0, 1, 2], [20, 40, 17], 16)
    st["lens"][0] = -20
    before = [t.clone() for t in (st["pages"].view(torch.uint8), st["scales"])]
    held = st["table"][:2].clone()
    assert ops.cache_fork(st["pages"], st["scales"], *book, [0, 1], [3, 2]).item() == 0
    assert kernel_status(DEV)["kv_cache"] == 3
    assert st["lens"].tolist() == [-20, 40, 40, 0] and st["table"][3].tolist() == [-1] * 3
    assert torch.equal(st["table"][:2], held) and torch.equal(st["table"][2, :2], held[1, :2])
    assert st["refs"].sum().item() == 2 + 3 + 3
    fresh = st["table"][2, 2].long()
    assert torch.equal(st["pages"].view(torch.uint8)[:, fresh], before[0][:, held[1, 2].long()])
    keep = torch.arange(8, device=DEV) != fresh
    assert torch.equal(st["pages"].view(torch.uint8)[:, keep], before[0][:, keep]) and torch.equal(st["scales"][:, keep], before[1][:, keep])


@pytest.mark.parametrize("slots,each", [(4096, 600000), (4000, 600000), (2, 524288), (1, 524287)])
def test_reserving_more_pages_than_32_bits_count(slots, each):
    """The sum of a batch's needs may pass 2^31 and 2^32: they lack then, and nothing changes."""
    table = torch.full((slots, 600000), -1, dtype=torch.int32, device=DEV)
    lens, refs = torch.zeros(slots, dtype=torch.int32, device=DEV), torch.zeros(100, dtype=torch.int32, device=DEV)
    refs[::4] = 1
    lack = ops.cache_reserve(table, lens, refs, list(range(slots)), [each * 16] * slots, 16).item()
    assert lack == min(slots * each - 75, 2 ** 31 - 1)
    assert not lens.any() and refs.sum().item() == 25 and (table[0] == -1).all() and (table[-1] == -1).all()


def test_copies_of_more_layers_than_a_grid_has_rows():
    layers = 65535 + 3
    pages = torch.zeros(layers, 2, 2, 1, 16, DIM, dtype=torch.uint8, device=DEV)
    pages[:, 0] = torch.arange(layers, device=DEV).remainder(120).to(torch.uint8)[:, None, None, None, None]
    scales = torch.arange(layers, device=DEV, dtype=torch.float32)[:, None, None, None, None].repeat(1, 2, 2, 1, 1)
    scales[:, 1] = 0
    ops.cache_copy(pages.view(torch.float8_e4m3fn), scales, ints([0]).to(DEV), ints([1]).to(DEV))
    assert torch.equal(pages[:, 1], pages[:, 0]) and torch.equal(scales[:, 1], scales[:, 0])


def test_graphs_leave_little_memory_behind():
    """Counters that outlive a graph do not come from its own pool, of which each would hold a segment."""
    st = filled([600, 130], 2, 64)
    q = torch.randn(2, 8, DIM, device=DEV).bfloat16()
    args = (st["pages"], st["scales"], st["table"], st["lens"], ints([0, 1]).to(DEV), ints([0, 1, 2]).to(DEV))
    want = ops.cache_attention(q, *args)

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.cache_attention(q, *args)
            again = ops.cache_attention(out, *args)
        for _ in range(2):
            graph.replay()
            assert torch.equal(out, want) and torch.equal(again, ops.cache_attention(want, *args))
        graph.reset()

    capture()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_reserved()
    for _ in range(6):
        capture()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    assert torch.cuda.memory_reserved() - before <= 2 * 2 ** 20


def test_streams_and_graphs_side_by_side():
    """Workspaces are a stream's or a graph's own: what runs at once does not mix."""
    sizes = ([9000, 40, 3000], [700] * 20, [20000])
    sets = [filled(lens, 2, 64, seed=i) for i, lens in enumerate(sizes)]
    calls = []
    for st, lens in zip(sets, sizes):
        n = len(lens)
        q = torch.randn(n, 8, DIM, device=DEV, generator=torch.Generator(DEV).manual_seed(n)).bfloat16()
        args = (q, st["pages"], st["scales"], st["table"], st["lens"], ints(list(range(n))).to(DEV), ints(list(range(n + 1))).to(DEV))
        calls.append((lambda a=args: ops.cache_attention(*a, max_new=1)))
    want = [call() for call in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = calls[0]()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        torch.cuda.synchronize()
        got = [[] for _ in calls]
        for _ in range(10):
            graph.replay()
            for stream, call, out in zip(streams, calls, got):
                with torch.cuda.stream(stream):
                    out.append(call())
        torch.cuda.synchronize()
        assert torch.equal(captured, want[0])
        for outs, w in zip(got, want):
            assert all(torch.equal(o, w) for o in outs)
    check_kernel_status(DEV)


@pytest.mark.parametrize("kernel", [1, 2])
def test_attention_of_several_tokens_in_a_graph(kernel):
    st = filled([600, 700], 2, 64)
    q = torch.randn(100, 8, DIM, device=DEV).bfloat16()
    cu, seqs = ints([0, 40, 90]).to(DEV), ints([0, 1]).to(DEV)
    call = lambda: ext().cache_attention(q, st["pages"], st["scales"], st["table"], st["lens"], seqs, cu, None,  # noqa: E731
                                         DIM ** -0.5, 0, kernel)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens, bounds in (([600, 700], [0, 40, 90]), ([64, 99], [0, 1, 100]), ([500, 3], [0, 97, 100])):
        st["lens"].copy_(ints(lens))
        cu.copy_(ints(bounds))
        q.copy_(torch.randn(100, 8, DIM))
        graph.replay()
        assert torch.equal(out, call())
    check_kernel_status(DEV)


def test_prompts_do_not_depend_on_the_run():
    counts = [700, 33, 2000]
    st = filled(counts, 4, 64)
    q, first = check_attention(st, [0, 1, 2], counts, 16, prefix=[700, 0, 1000], kernel=2)
    for _ in range(5):
        assert torch.equal(attend(q, st, [0, 1, 2], [0, 700, 733, 2733], [700, 0, 1000], kernel=2), first)


def test_compaction_into_a_pool_that_is_too_small():
    st = {k: t.to(DEV) for k, t in pool(12, 1, 16, DIM, 4, 3, layers=2).items()}
    book = (st["table"], st["lens"], st["refs"])
    ops.cache_reserve(*book, [0, 1, 2], [40, 17, 33], 16)
    ops.cache_free(*book, [1])

    def other(pages):
        return (torch.zeros(2, pages, 2, 1, 16, DIM, device=DEV).to(torch.float8_e4m3fn), torch.zeros(2, pages, 2, 1, 1, device=DEV),
                torch.full_like(st["table"], 77), ints([9] * pages).to(DEV))

    small, fits = other(5), other(6)
    assert ops.cache_compact(st["pages"], st["scales"], st["table"], st["refs"], small).item() == 1
    assert not small[0].view(torch.uint8).any() and not small[1].any() and (small[2] == 77).all() and (small[3] == 9).all()
    assert ops.cache_compact(st["pages"], st["scales"], st["table"], st["refs"], fits).item() == 0
    assert fits[2].tolist() == [[0, 1, 2, -1], [-1] * 4, [5, 3, 4, -1]] and fits[3].tolist() == [1] * 6
    check_kernel_status(DEV)
