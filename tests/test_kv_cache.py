"""The 8-bit paged key/value cache and the logits operators, PyTorch formulations (CPU): against plain
64-bit formulas, a step-by-step model of the page bookkeeping, and their refusals."""
import math
import random

import pytest
import torch

from mimir_b200 import ops
from mimir_b200.ops.kv_cache import BLOCK


def tables(positions, dim, base=10000.0):
    angle = torch.outer(torch.arange(positions, dtype=torch.float32),
                        base ** (-torch.arange(0, dim, 2, dtype=torch.float32) / dim))
    angle = torch.cat((angle, angle), -1)
    return angle.cos(), angle.sin()


def pool(pages, kv, page, dim, width, slots, seed=0, layers=None):
    gen = torch.Generator().manual_seed(seed)
    lead = () if layers is None else (layers,)
    x = torch.randn(*lead, pages, 2, kv, page, dim, generator=gen)
    scales = torch.ldexp(torch.ones(*lead, pages, 2, kv, page // BLOCK),
                         torch.randint(-9, -3, (*lead, pages, 2, kv, page // BLOCK), generator=gen))
    return dict(pages=(x * 64).to(torch.float8_e4m3fn), scales=scales,
                table=torch.full((slots, width), -1, dtype=torch.int32), lens=torch.zeros(slots, dtype=torch.int32),
                refs=torch.zeros(pages, dtype=torch.int32))


def ints(values):
    return torch.tensor(values, dtype=torch.int32)


def nearest_e4m3(x):
    """The e4m3 values nearest to ``x`` (float64, |x| <= 448), ties to even."""
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x.abs().clamp_min(2.0 ** -6)).exponent - 4)
    return torch.round(x / step) * step


@pytest.mark.parametrize("dim", [8, 128])
def test_append_then_attention_equals_the_formula(dim):
    """Token by token and in one go, the cache holds what the formula says, to one e4m3 rounding of the block's
    scale, and attention over it equals 64-bit attention over the held values."""
    heads, kv, page, n = 4, 2, 16, 37
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, h, dim, generator=gen) for h in (heads, kv, kv))
    k, v = (x * torch.exp(torch.randn(n, 1, 1, generator=gen)) for x in (k, v))
    cos, sin = tables(64, dim)
    at, half = torch.arange(n), dim // 2
    kd = k.double()
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    turned = kd * c + torch.cat((-kd[..., half:], kd[..., :half]), -1) * s
    for steps in ([n], [1] * n, [5, 11, 1, 20]):
        st = pool(8, kv, page, dim, 4, 2)
        done, outs = 0, []
        for count in steps:
            assert ops.cache_reserve(st["table"], st["lens"], st["refs"], [1], [count], page).item() == 0
            cu = ints([0, count])
            rows = slice(done, done + count)
            qr = ops.cache_append(q[rows], k[rows], v[rows], cos, sin, st["pages"], st["scales"], st["table"],
                                  st["lens"], ints([1]), cu)
            outs.append(ops.cache_attention(qr, st["pages"], st["scales"], st["table"], st["lens"], ints([1]), cu))
            done += count
        from mimir_b200.ops.kv_cache import cache_values
        held = cache_values(st["pages"], st["scales"], st["table"], 1, n).double()
        for b in range(0, n, BLOCK):
            for which, x in ((0, turned), (1, v.double())):
                block = x[b:b + BLOCK]
                amax = block.abs().amax((0, 2))
                scale = torch.tensor([next(2.0 ** e for e in range(-32, 99) if a <= 448 * 2.0 ** e) for a in amax.tolist()])
                # one rounding (half a step of the value, or of the smallest normal), fp32 products, and
                # a second rounding of at most as much for tokens written under a smaller scale
                err = (held[which, :, b:b + BLOCK].transpose(0, 1) - block).abs()
                bound = 2 * torch.maximum(block.abs() * 2.0 ** -4, (scale * 2.0 ** -10)[None, :, None]) * 1.001
                assert bool((err <= bound).all())
        if steps == [n]:
            s64 = torch.einsum("tkgd,kjd->kgtj", qr.double().unflatten(1, (kv, -1)), held[0]) * dim ** -0.5
            s64 = s64.masked_fill(at[None] > at[:, None], -math.inf)
            ref = torch.einsum("kgtj,kjd->tkgd", torch.softmax(s64, -1), held[1]).flatten(1, 2)
            torch.testing.assert_close(outs[0].double(), ref, atol=2e-5, rtol=2e-5)


def test_bytes_are_the_nearest_ones():
    dim, kv = 8, 1
    gen = torch.Generator().manual_seed(9)
    v = torch.randn(16, kv, dim, generator=gen) * torch.exp(3 * torch.randn(16, 1, dim, generator=gen))
    st = pool(2, kv, 16, dim, 1, 1)
    ops.cache_reserve(st["table"], st["lens"], st["refs"], [0], [16], 16)
    cos, sin = tables(16, dim)
    ops.cache_append(v, v, v, cos, sin, st["pages"], st["scales"], st["table"], st["lens"], ints([0]), ints([0, 16]))
    scale = st["scales"][0, 1, 0, 0].double()
    assert v.abs().max() <= 448 * scale and v.abs().max() > 224 * scale
    assert torch.equal(st["pages"][0, 1, 0].double() * scale, nearest_e4m3(v[:, 0].double() / scale) * scale)


def test_values_that_are_not_finite_poison_their_block_only():
    dim, cos_sin = 8, tables(64, 8)
    st = pool(4, 1, 16, dim, 4, 1)
    x = torch.randn(40, 1, dim, generator=torch.Generator().manual_seed(1))
    v = x.clone()
    v[20, 0, 3] = math.inf
    ops.cache_reserve(st["table"], st["lens"], st["refs"], [0], [40], 16)
    q = ops.cache_append(x, x, v, *cos_sin, st["pages"], st["scales"], st["table"], st["lens"], ints([0]), ints([0, 40]))
    page = st["table"][0, 1].item()
    assert torch.isnan(st["scales"]).sum() == 1 and torch.isnan(st["scales"][page, 1, 0, 0])
    assert not torch.isnan(st["pages"].float()).any()
    out = ops.cache_attention(q, st["pages"], st["scales"], st["table"], st["lens"], ints([0]), ints([0, 40]))
    assert torch.isfinite(out[:16]).all()  # rows before the block do not see it


def test_prefix_rows_see_the_prefix():
    dim = 8
    st = pool(3, 1, 16, dim, 2, 1)
    st["table"][0] = ints([2, 0])
    st["lens"][0] = 20
    q = torch.randn(6, 2, dim, generator=torch.Generator().manual_seed(2))  # positions 14 .. 19
    got = ops.cache_attention(q, st["pages"], st["scales"], st["table"], st["lens"], ints([0]), ints([0, 6]), ints([17]))
    from mimir_b200.ops.kv_cache import cache_values
    k, v = cache_values(st["pages"], st["scales"], st["table"], 0, 20).double()[:, 0]
    for t, keys in enumerate([17, 17, 17, 18, 19, 20]):
        for h in range(2):
            p = torch.softmax(k[:keys] @ q[t, h].double() * dim ** -0.5, 0)
            torch.testing.assert_close(got[t, h].double(), p @ v[:keys], atol=2e-5, rtol=2e-5)


class Model:
    """The page bookkeeping, one page at a time."""

    def __init__(self, slots, width, pages, page):
        self.rows, self.lens, self.page, self.width = [[] for _ in range(slots)], [0] * slots, page, width
        self.refs, self.data = [0] * pages, list(range(pages))

    def take(self, count):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        return free[:count] if len(free) >= count else None

    def reserve(self, seqs, counts):
        need = [-(-(self.lens[s] + c) // self.page) - len(self.rows[s]) for s, c in zip(seqs, counts)]
        if any(-(-(self.lens[s] + c) // self.page) > self.width for s, c in zip(seqs, counts)):
            return -1
        got = self.take(sum(need))
        if got is None:
            return sum(need) - self.refs.count(0)
        for s, c, n in zip(seqs, counts, need):
            for _ in range(n):
                p = got.pop(0)
                self.rows[s].append(p)
                self.refs[p] = 1
            self.lens[s] += c
        return 0

    def free(self, seqs):
        for s in seqs:
            for p in self.rows[s]:
                self.refs[p] -= 1
            self.rows[s], self.lens[s] = [], 0

    def fork(self, src, dst):
        self.free(dst)
        for a, b in zip(src, dst):
            self.rows[b], self.lens[b] = self.rows[a][:self.lens[a] // self.page], self.lens[a]
            for p in self.rows[b]:
                self.refs[p] += 1
        parts = [(a, b) for a, b in zip(src, dst) if self.lens[a] % self.page]
        got = self.take(len(parts))
        if got is None:
            lack = len(parts) - self.refs.count(0)
            self.free(dst)
            return lack
        for (a, b), p in zip(parts, got):
            self.rows[b].append(p)
            self.refs[p] = 1
            self.data[p] = self.data[self.rows[a][len(self.rows[b]) - 1]]
        return 0

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p in range(len(live)) if not self.refs[p]]
        to = {p: p if p < len(live) else holes.pop(0) for p in live}
        refs, data = [0] * len(self.refs), list(self.data)
        for p, o in to.items():
            refs[o], data[o] = self.refs[p], self.data[p]
        self.refs, self.data = refs, data
        self.rows = [[to[p] for p in row] for row in self.rows]


def drive_pages(device, slots, width, pages, page, steps, seed, layers=2, kv=1, dim=128):
    """Random page operations on ``device`` against :class:`Model`, checked after every one."""
    rng = random.Random(seed)
    st = {k: t.to(device) for k, t in pool(pages, kv, page, dim, width, slots, seed, layers).items()}
    first_pages, first_scales = st["pages"].clone(), st["scales"].clone()
    model, book = Model(slots, width, pages, page), (st["table"], st["lens"], st["refs"])
    seen = set()
    for _ in range(steps):
        do = rng.choice(["reserve"] * 4 + ["free", "fork", "fork", "compact"])
        seen.add(do)
        some = rng.sample(range(slots), rng.randint(1, slots // 2))
        if do == "reserve":
            counts = [rng.choice([0, 1, 1, page, rng.randint(1, page * width // 2)]) for _ in some]
            assert ops.cache_reserve(*book, some, counts, page).item() == model.reserve(some, counts)
        elif do == "free":
            ops.cache_free(*book, some)
            model.free(some)
        elif do == "fork":
            src = [rng.choice(some) for _ in range(slots)]
            dst = [s for s in range(slots) if s not in some][:rng.randint(1, slots)]
            src = src[:len(dst)]
            assert ops.cache_fork(st["pages"], st["scales"], *book, src, dst).item() == model.fork(src, dst)
        else:
            assert ops.cache_compact(st["pages"], st["scales"], st["table"], st["refs"]).item() == 0
            model.compact()
        assert st["table"].tolist() == [row + [-1] * (width - len(row)) for row in model.rows]
        assert st["lens"].tolist() == model.lens and st["refs"].tolist() == model.refs
        live = [p for p, r in enumerate(model.refs) if r]
        came = [model.data[p] for p in live]
        assert torch.equal(st["pages"].view(torch.uint8)[:, live], first_pages.view(torch.uint8)[:, came])
        assert torch.equal(st["scales"][:, live], first_scales[:, came])
    assert seen == {"reserve", "free", "fork", "compact"}


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_page_operations_follow_the_model(seed):
    drive_pages("cpu", slots=6, width=5, pages=20, page=16, steps=60, seed=seed, dim=8)


def test_compaction_into_another_pool():
    st = pool(12, 1, 16, 8, 4, 3, layers=2)
    book = (st["table"], st["lens"], st["refs"])
    ops.cache_reserve(*book, [0, 1, 2], [40, 17, 33], 16)
    ops.cache_free(*book, [1])
    out = (torch.zeros(2, 6, 2, 1, 16, 8).to(torch.float8_e4m3fn), torch.zeros(2, 6, 2, 1, 1),
           torch.zeros_like(st["table"]), ints([9] * 6))
    small = tuple(t[:, :5].contiguous() if i < 2 else t[:5].clone() if i == 3 else t for i, t in enumerate(out))
    assert ops.cache_compact(st["pages"], st["scales"], st["table"], st["refs"], small).item() == 1
    assert ops.cache_compact(st["pages"], st["scales"], st["table"], st["refs"], out).item() == 0
    assert out[2].tolist() == [[0, 1, 2, -1], [-1] * 4, [5, 3, 4, -1]]
    assert out[3].tolist() == [1] * 6
    for slot in (0, 2):
        for j in range(3):
            a, b = st["table"][slot, j].long(), out[2][slot, j].long()
            assert torch.equal(st["pages"].view(torch.uint8)[:, a], out[0].view(torch.uint8)[:, b])


def test_refusals():
    st = pool(4, 2, 16, 8, 3, 2, layers=1)
    book = (st["table"], st["lens"], st["refs"])
    pages, scales = st["pages"][0], st["scales"][0]
    x, (cos, sin), cu = torch.randn(1, 2, 8), tables(48, 8), ints([0, 1])
    with pytest.raises(ValueError, match="page_size"):
        ops.cache_reserve(*book, [0], [1], 24)
    with pytest.raises(ValueError, match="name each slot once"):
        ops.cache_reserve(*book, [0, 0], [1, 1], 16)
    with pytest.raises(ValueError, match="slots of the page table"):
        ops.cache_free(*book, [2])
    with pytest.raises(ValueError, match="both source and destination"):
        ops.cache_fork(st["pages"], st["scales"], *book, [0], [0])
    with pytest.raises(ValueError, match="int32"):
        ops.cache_reserve(st["table"].long(), st["lens"], st["refs"], [0], [1], 16)
    with pytest.raises(ValueError, match="divisible"):
        ops.cache_attention(torch.randn(1, 3, 8), pages, scales, st["table"], st["lens"], ints([0]), cu)
    with pytest.raises(ValueError, match="one more entry"):
        ops.cache_attention(torch.randn(1, 2, 8), pages, scales, st["table"], st["lens"], ints([0]), ints([0, 1, 1]))
    with pytest.raises(ValueError, match="scales"):
        ops.cache_attention(torch.randn(1, 2, 8), pages, scales[..., :0], st["table"], st["lens"], ints([0]), cu)
    with pytest.raises(ValueError, match="float8"):
        ops.cache_append(x, x, x, cos, sin, pages.float(), scales, st["table"], st["lens"], ints([0]), cu)
    with pytest.raises(ValueError, match="no room"):
        ops.cache_append(x, x, x, cos, sin, pages, scales, st["table"], st["lens"], ints([0]), cu)
    with pytest.raises(ValueError, match="one type"):
        ops.cache_append(x, x, x.bfloat16(), cos, sin, pages, scales, st["table"], st["lens"], ints([0]), cu)
    with pytest.raises(ValueError, match="need tokens"):
        ops.process_logits(torch.randn(2, 7), repetition=torch.ones(2))
    with pytest.raises(ValueError, match="ceil"):
        ops.process_logits(torch.randn(2, 33), allowed=torch.zeros(2, 1, dtype=torch.int32))


def test_logits_rules_one_by_one():
    x = torch.tensor([[2.0, -2.0, 1.0, 0.5, math.nan, 3.0]])
    out = ops.process_logits(x, tokens=ints([[0, 1, 1, 3, -1, 6, 2]]), token_lens=ints([6]), prompt_lens=ints([2]),
                             repetition=torch.tensor([2.0]), presence=torch.tensor([0.25]), frequency=torch.tensor([0.5]),
                             bias=(ints([0, 3]), ints([5, 5, 9]), torch.tensor([1.0, 2.0, 50.0])), allowed=ints([[0b101111]]))
    # 0: prompt only; 1: prompt and generated once; 3: generated; 2: after the row's end; 4: not allowed; 5: two biases
    assert out.tolist() == [[1.0, -4.0 - 0.5 - 0.25, 1.0, 0.25 - 0.5 - 0.25, -math.inf, 6.0]]
    assert torch.equal(ops.process_logits(x[:, :4]), x[:, :4])
    assert torch.isinf(ops.process_logits(x, allowed=ints([[0]]))).all()
    y = x.clone()
    assert ops.process_logits(y, allowed=ints([[0]]), out=y) is y and torch.isinf(y).all()


@pytest.mark.parametrize("cu", [[-1, 2], [0, 4], [2, 1]])
def test_bounds_that_leave_the_rows_are_refused(cu):
    st = pool(4, 2, 16, 8, 3, 2)
    ops.cache_reserve(st["table"], st["lens"], st["refs"], [0], [20], 16)
    x, rest = torch.randn(3, 2, 8), (st["pages"], st["scales"], st["table"], st["lens"], ints([0]), ints(cu))
    with pytest.raises(ValueError, match="cu_new must rise"):
        ops.cache_append(x, x, x, *tables(48, 8), *rest)
    with pytest.raises(ValueError, match="cu_new must rise"):
        ops.cache_attention(x, *rest)
