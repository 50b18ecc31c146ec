"""The cache in 8 bits and its attention against the definitions in 64 bits.

Written numbers and numbers read back are the definition's bits.  Attention: with u half a step of the output's type, w what a weight is rounded
by (2^-11 as one fp16 term, 2^-22 as two), A the largest sum of |scale q k| of a row's tokens and B its sum of p |v| over the denominator,

    |error| <= u |o| + B (w + 2 e + 2^-20) + T V s,   e = A (2^-22 + (D terms / 16 + 8) 2^-23)

e bounds a score's error: queries of fp32 rows have 22 bits, the tensor core cuts a sum off once per 16 channels and term by up to 2^-23 of it, and the scale, the page's
power and the exponent's argument are rounded; the error of a weight relative to the others is at most twice that.  2^-20: the exponentials (2^-22 each) and the sums of
weights and outputs.

T V s, T tokens and V their largest value: small weights.  A weight is fp16 2^(t - R + 7), t = x + e - E with x its score in powers of two, 2^e its page's step and 2^E the largest
page's.  Below 2^-14 fp16 has steps of 2^-24, so it is off by up to 2^-25 whatever its size.  R is the t of a token that was seen, and e <= E, so the denominator, which has that token's
2^(x - R + 7) = 2^(t - R + 7 + E - e), is at least 2^7.  A code is at most c = 448 (127), so a token adds at most 2^-25 c 2^E / 2^7; and c 2^E < 2 V, as E is the smallest exponent for
V.  That is s = 2^-31.  (Few rows count from 2^14, not 2^7, and the two terms of fp32 rows leave 2^-25 too: 2^-38.)"""

import math

import pytest
import torch

from dia_tts_prune_b200 import lm_ops

pytestmark = pytest.mark.gpu

LARGEST = {"e4m3": 448.0, "int8": 127.0}
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cumulative(counts):
    return ints([sum(counts[:i]) for i in range(len(counts) + 1)])


def nearest(v, fmt):
    if fmt == "int8":
        return torch.round(v)
    _, x = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (x - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def two(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


class Exact:
    """Pages of values in 64 bits, written token by token as the definition says; a page that stands for NaNs is all NaN."""

    def __init__(self, pages, heads, dim, page, fmt):
        self.v = torch.zeros(pages, heads, page, dim, dtype=torch.float64)
        self.e = torch.full((pages, heads), -100)
        self.page, self.fmt = page, fmt

    def append(self, x, table, past, counts):
        """x [rows, heads, dim] in 64 bits"""
        at = 0
        for i, n in enumerate(counts):
            done = 0
            while done < n:
                pos = past[i] + done
                place, slot = pos % self.page, pos // self.page
                m = min(n - done, self.page - place)
                rows = x[at + done:at + done + m].transpose(0, 1)
                done += m
                if past[i] < 0 or slot >= len(table[i]) or not 0 <= table[i][slot] < len(self.v):
                    continue
                p = table[i][slot]
                most = rows.abs().amax((1, 2))
                bad = ~torch.isfinite(most) | (torch.isnan(self.v[p, :, 0, 0]) if place else False)
                need = torch.full(most.shape, -100)
                for h in range(len(most)):
                    if not bad[h]:
                        while most[h] > LARGEST[self.fmt] * 2.0 ** int(need[h]):
                            need[h] += 1
                e = torch.maximum(self.e[p], need) if place else need
                self.e[p] = e
                unit = two(e)[:, None, None]
                self.v[p, :, :place] = nearest(self.v[p, :, :place] / unit, self.fmt) * unit
                self.v[p, :, place:place + m] = nearest(rows / unit, self.fmt) * unit
                self.v[p][bad] = math.nan
            at += n

    def read(self, table, past, counts):
        out = []
        for i, n in enumerate(counts):
            for j in range(n):
                pos = past[i] + j
                slot = pos // self.page
                there = past[i] >= 0 and slot < len(table[i]) and 0 <= table[i][slot] < len(self.v)
                out.append(self.v[table[i][slot], :, pos % self.page] if there else torch.zeros_like(self.v[0, :, 0]))
        return torch.stack(out) if out else self.v.new_zeros(0, self.v.shape[1], self.v.shape[3])


def exact_attention(q, k, v, there, past, scale, window, sinks):
    """One sequence in 64 bits: q [n, heads, dim], k, v [tokens, kv heads, dim], there [tokens].  (output, A, B)"""
    n, H, D = q.shape
    G, T = k.shape[1], k.shape[0]
    k, v = (x.repeat_interleave(H // G, 1).transpose(0, 1) for x in (k, v))                  # [heads, tokens, dim]
    q = q.transpose(0, 1)
    behind = (past + torch.arange(n, device=q.device))[:, None] - torch.arange(T, device=q.device)
    ok = (behind >= 0) & (behind < (window or 1 << 40)) & there
    z = torch.where(ok, scale * (q @ k.transpose(1, 2)), -math.inf)
    zs = z if sinks is None else torch.cat([z, sinks.double()[:, None, None].expand(H, n, 1)], 2)
    p = torch.softmax(zs, -1)[..., :T]
    p = torch.where(ok, p, 0.0) if sinks is not None else torch.where(ok.any(-1, keepdim=True), p, 0.0)
    v = torch.where(ok.any(0)[:, None], v, 0.0)                                              # (nobody sees those)
    k = torch.where(there[:, None], k, 0.0)
    A = torch.where(ok, scale * (q.abs() @ k.abs().transpose(1, 2)), 0.0).amax(-1, keepdim=True) if T else q.new_zeros(H, n, 1)
    return tuple(x.transpose(0, 1) for x in (p @ v, A, p @ v.abs()))


HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def check_attention(got, q, cache, table, past, counts, scale=None, window=None, sinks=None, lists=None):
    """Against 64 bits on the numbers that the cache reads back."""
    D, dtype = q.shape[2], q.dtype
    scale = D ** -0.5 if scale is None else scale
    terms, at = (2 if dtype == torch.float32 else 1), 0
    for i, n in enumerate(counts):
        if not n:
            continue
        total = past[i] + n
        k, v = cache.read(table[i:i + 1], ints([0]), ints([0, total]), total)
        pages = torch.tensor(lists[i], device=DEV)[torch.arange(total, device=DEV) // cache.page_size]
        there = (pages >= 0) & (pages < cache.pages)
        for r in range(0, n, 256):                                # (in pieces: long prompts have many scores)
            m = min(256, n - r)
            o, A, B = exact_attention(q[at + r:at + r + m].double(), k.double(), v.double(), there, past[i] + r, scale, window, sinks)
            e = A * (2.0 ** -22 + (D * terms / 16 + 8) * 2.0 ** -23)
            small = total * float(v.nan_to_num().abs().max()) * 2.0 ** (-38 if terms == 2 else -31)
            bound = HALF[dtype] * o.abs() + small + B * ((2.0 ** -22 if terms == 2 else 2.0 ** -11) + 2 * e + 2.0 ** -20) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
            err = (got[at + r:at + r + m].double() - o).abs()
            assert torch.equal(torch.isnan(err), torch.isnan(o)), "NaN in other places"
            worst = torch.where(torch.isnan(err), 0.0, err - bound).max()
            assert worst <= 0, (i, r, float(worst), float(err.nan_to_num().max()))
        at += n
    assert not got[at:].any()


def tables(counts, past, page, pages, generator, width=None):
    """Lists of pages of every sequence, in an order of no order, and the table on the device."""
    order = torch.randperm(pages, generator=generator).tolist()
    lists = [[order.pop() for _ in range(-(-(p + n) // page) if p >= 0 else 0)] for n, p in zip(counts, past)]
    width = width or max(1, max(map(len, lists)))
    lists = [row + [-1] * (width - len(row)) for row in lists]
    return lists, ints(lists)


def rows_of(g, shape, dtype, loud=0.05):
    x = torch.randn(shape, generator=g)
    x = x * torch.where(torch.rand(shape[-1], generator=g) < loud, 8.0, 1.0) * torch.exp(0.5 * torch.randn(shape[0], 1, 1, generator=g))
    return x.to(dtype)


# ---- written and read -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,dim,page,dtype", [(1, 1, 16, torch.float32), (3, 80, 32, torch.bfloat16), (2, 128, 16, torch.float16), (4, 64, 64, torch.bfloat16), (2, 72, 16, torch.float32),
                                                  (1, 13, 128, torch.float16), (2, 256, 128, torch.bfloat16), (8, 128, 16, torch.bfloat16), (2, 200, 32, torch.float32)])
def test_numbers_written_step_by_step(fmt, heads, dim, page, dtype):
    g = torch.Generator().manual_seed(dim + page)
    steps = [[5, 0, 1, 40, 17], [1, 1, 1, 1, 1], [0, 100, 0, 1, 16], [3, 0, 300, 0, 15], [1, 1, 1, 1, 1]]
    total = [sum(s[i] for s in steps) for i in range(5)]
    lists, table = tables(total, [0] * 5, page, 60, g)
    cache = lm_ops.Kv8(60, heads, dim, page_size=page, format=fmt)
    want = [Exact(60, heads, dim, page, fmt) for _ in range(2)]
    past = [0] * 5
    for s, counts in enumerate(steps):
        x = rows_of(g, (sum(counts), 2 * heads, dim), dtype) * 1.5 ** (3 * s)         # (later ones are larger: steps have to grow)
        k, v = x[:, :heads].contiguous(), x[:, heads:].contiguous()
        if s == 1:
            k[2], v[0, 0] = 0, 0                                                      # tokens of zeros
        cache.append(k.to(DEV), v.to(DEV), table, ints(past), cumulative(counts))
        for w, y in zip(want, (k, v)):
            w.append(y.double(), lists, past, counts)
        past = [p + n for p, n in zip(past, counts)]
        got = cache.read(table, ints([0] * 5), cumulative(past), sum(past))
        for y, w in zip(got, want):
            assert torch.equal(y.double().cpu(), w.read(lists, [0] * 5, past))
    stride = (dim + 15) // 16 * 16
    assert cache.keys.shape == (60, heads, page, stride) and not cache.keys[..., dim:].any() and not cache.values[..., dim:].any()
    # stretches that begin anywhere, in every type
    starts, counts = [2, 0, 17, 40, 30], [3, 7, 200, 1, 0]
    for t in (torch.float32, torch.bfloat16, torch.float16):
        got = cache.read(table, ints(starts), cumulative(counts), sum(counts) + 3, t)
        for y, w in zip(got, want):
            expect = w.read(lists, starts, counts).float().to(t)
            assert y.dtype == t and torch.equal(y[:-3].cpu(), expect) and not y[-3:].any()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_borders_of_steps_and_numbers(fmt):
    """Largest magnitudes at and beside the borders of exponents; the smallest and largest floats; every code and half way between two."""
    top = LARGEST[fmt]
    border = torch.tensor([top * 2.0 ** e * f for e in (-130, -101, -100, -99, -20, 0, 1, 30, 100) for f in (1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -24)])
    border = torch.cat([border, torch.tensor([0.0, 2.0 ** -149, 2.0 ** -126, torch.finfo(torch.float32).max])])
    rows = torch.zeros(len(border) * 16, 1, 8)
    g = torch.Generator().manual_seed(3)
    rows.view(-1, 16, 8)[:] = (2 * torch.rand(len(border), 16, 8, generator=g) - 1) * border[:, None, None]
    rows.view(-1, 16, 8)[:, 5, 3] = border
    rows.view(-1, 16, 8)[:, 6, 3] = -border / 3
    # one page each; then a page of halves
    halves = torch.cat([(torch.arange(128).float() - 64) * f for f in (0.5, 2.0 ** -10, 3.5, 0.25)])
    last = torch.zeros(64, 1, 8)
    last.view(-1)[:] = halves.clamp(-top, top)
    last.view(-1, 16, 8)[:, 0, 0] = top
    rows = torch.cat([rows, last])
    n, pages = len(rows), len(rows) // 16
    cache = lm_ops.Kv8(pages, 1, 8, format=fmt)
    lists = [list(range(pages))]
    cache.append(rows.to(DEV), -rows.to(DEV), ints(lists), ints([0]), ints([0, n]))
    want = Exact(pages, 1, 8, 16, fmt)
    want.append(rows.double(), lists, [0], [n])
    k, v = cache.read(ints(lists), ints([0]), ints([0, n]), n)
    # (float32's largest number goes to 2^128, which float32 reads as infinity)
    assert torch.equal(k.cpu(), want.read(lists, [0], [n]).float()) and torch.equal(v, -k)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_numbers_that_are_not_finite(fmt):
    cache = lm_ops.Kv8(6, 2, 24, page_size=16, format=fmt)
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(40, 2, 24, generator=g), torch.randn(40, 2, 24, generator=g)
    k[3, 0, 5], v[20, 1, 0], v[21, 0, 23] = math.inf, math.nan, -math.inf
    lists, table = [[4, 0, 2]], ints([[4, 0, 2]])
    want = [Exact(6, 2, 24, 16, fmt) for _ in range(2)]
    past = 0
    for n in (2, 5, 15, 10, 8):                                    # (a page that has begun gets one; a page with one goes on)
        cache.append(k[past:past + n].to(DEV), v[past:past + n].to(DEV), table, ints([past]), ints([0, n]))
        for w, y in zip(want, (k, v)):
            w.append(y[past:past + n].double(), lists, [past], [n])
        past += n
        for y, w in zip(cache.read(table, ints([0]), ints([0, past]), past), want):
            assert torch.equal(y.double().cpu().nan_to_num(123.0), w.read(lists, [0], [past]).nan_to_num(123.0))
    assert not ((cache.keys & 127) == 127).any() or fmt == "int8"   # (codes stay finite whatever the scale is)
    # the first token of a page starts it anew
    cache.append(v[:16].to(DEV), v[:16].to(DEV), table, ints([0]), ints([0, 16]))
    assert not cache.read(table, ints([0]), ints([0, 16]), 16)[0].isnan().any()


def test_tokens_that_are_not_there():
    """Pages outside the pool, places beyond the table, a negative past, rows of no sequence: nothing is written beside what is there."""
    cache = lm_ops.Kv8(8, 2, 40, page_size=16)
    for t in (cache.keys, cache.values):
        t.fill_(56)
    for t in (cache.key_scales, cache.value_scales):
        t.fill_(2.0)
    before = [t.clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales)]
    lists = [[1, 8, 3], [-1, 2, 1 << 30], [4, 5, 6], [0, 7, -(1 << 31)]]
    past, counts = [0, 10, -5, 40], [48, 38, 20, 30]
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn(sum(counts) + 9, 2, 40, generator=g), torch.randn(sum(counts) + 9, 2, 40, generator=g)
    first = ints([5, 53, 91, 111, 141])                            # five rows in front of the first sequence, four behind the last
    cache.append(k.to(DEV), v.to(DEV), ints(lists), ints(past), first)
    want = [Exact(8, 2, 40, 16, "e4m3") for _ in range(2)]
    for w, y in zip(want, (k, v)):
        w.append(y[5:].double(), lists, past, counts)
    got = cache.read(ints(lists), ints(past), first, len(k))
    for y, w in zip(got, want):
        expect = w.read(lists, past, counts)
        assert torch.equal(y[5:141].double().cpu(), expect) and not y[:5].any() and not y[141:].any()
    for p in (0, 4, 5, 6, 7):
        for t, b in zip((cache.keys, cache.values, cache.key_scales, cache.value_scales), before):
            assert torch.equal(t[p], b[p])
    # attention of the same rows sees what is there, and nothing of the sequence with a negative past
    q = torch.randn(len(k), 4, 40, generator=g).to(DEV)
    out = lm_ops.attention_kv8(q, cache, ints(lists), ints(past), first)
    assert not out[:5].any() and not out[141:].any() and not out[91:111].any() and torch.isfinite(out).all()
    check_attention(out[5:53], q[5:53], cache, ints(lists[:1]), [0], [48], lists=lists[:1])
    wide = [row + [-1] for row in lists]                           # (places beyond the table, in words that the check can read)
    check_attention(out[53:91], q[53:91], cache, ints(wide[1:2]), [10], [38], lists=wide[1:2])


def test_strides_of_rows_and_heads():
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(70, 12, 48, generator=g).to(DEV)              # 8 query, 2 key and 2 value heads
    lists, table = tables([70], [0], 16, 9, g)
    past, first = ints([0]), ints([0, 70])
    a, b = (lm_ops.Kv8(9, 2, 48) for _ in range(2))
    a.append(qkv[:, 8:10], qkv[:, 10:], table, past, first)
    b.append(qkv[:, 8:10].contiguous(), qkv[:, 10:].contiguous(), table, past, first)
    assert torch.equal(a.keys, b.keys) and torch.equal(a.values, b.values) and torch.equal(a.key_scales, b.key_scales)
    want = lm_ops.attention_kv8(qkv[:, :8].contiguous(), a, table, past, first)
    heads_first = qkv[:, :8].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(70, 8, 49, device=DEV)                       # rows that are not 16-byte aligned
    wide[..., 1:] = qkv[:, :8]
    apart = qkv[:, :8].transpose(1, 2).contiguous().transpose(1, 2)  # channels apart
    for q in (qkv[:, :8], heads_first, wide[..., 1:], apart):
        assert torch.equal(lm_ops.attention_kv8(q, a, table, past, first), want)
    c = lm_ops.Kv8(9, 2, 48)
    w = torch.zeros(70, 4, 49, device=DEV)
    w[..., 1:] = qkv[:, 8:]
    c.append(w[:, :2, 1:], w[:, 2:, 1:], table, past, first)
    assert torch.equal(a.keys, c.keys) and torch.equal(a.values, c.values)
    # a table with pages apart in a larger one; one key head for all rows (a broadcast view)
    big = torch.full((3, 40), -7, dtype=torch.int32, device=DEV)
    big[1:2, 3:3 + table.shape[1]] = table
    assert torch.equal(lm_ops.attention_kv8(qkv[:, :8], a, big[1:2, 3:3 + table.shape[1]], past, first), want)
    one = qkv[:1, :1].expand(70, 2, 48)
    a.append(one, one, table, past, first)
    assert torch.equal(a.read(table, past, first, 70)[0][0, 0], a.read(table, past, first, 70)[0][69, 1])


# ---- attention -------------------------------------------------------------------------------------------------------------------

def filled(g, fmt, heads, dim, page, past, counts, spread=0.5):
    lists, table = tables(counts, past, page, sum(-(-(p + n) // page) for p, n in zip(past, counts)) + 2, g)
    cache = lm_ops.Kv8(sum(-(-(p + n) // page) for p, n in zip(past, counts)) + 2, heads, dim, page_size=page, format=fmt)
    total = [p + n for p, n in zip(past, counts)]
    x = torch.randn(sum(total), 2 * heads, dim, generator=g) * torch.exp(spread * torch.randn(sum(total), 1, 1, generator=g))
    x = x.to(DEV)
    cache.append(x[:, :heads], x[:, heads:], table, ints([0] * len(past)), cumulative(total))
    return lists, table, cache


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("fmt,heads,group,dim,page,past,counts,window,sinks", [
    ("e4m3", 4, 4, 128, 16, [1024], [1], None, False),
    ("int8", 2, 4, 128, 64, [0, 1, 15, 16, 17, 4000, 31, 300], [1] * 8, None, False),
    ("e4m3", 1, 1, 64, 16, [0], [1], None, False),
    ("e4m3", 2, 16, 64, 32, [700, 3], [1, 1], None, True),
    ("int8", 3, 2, 80, 32, [5, 0, 200, 77], [1, 130, 3, 17], 50, True),
    ("e4m3", 1, 48, 96, 16, [500, 0], [2, 9], 100, False),
    ("int8", 2, 3, 13, 16, [90], [40], None, False),
    ("e4m3", 8, 1, 128, 128, [0, 1000], [257, 1], 1, False),
    ("int8", 1, 8, 256, 16, [300, 9], [1, 33], None, True),
    ("e4m3", 2, 2, 200, 64, [100], [70], 64, False),
    ("int8", 2, 5, 1, 16, [50], [3], None, False),
    ("e4m3", 2, 8, 128, 16, [0], [513], None, False),
    ("int8", 1, 4, 64, 16, [2000, 0, 0], [0, 300, 0], 128, False),
    ("e4m3", 1, 7, 72, 16, [20000], [1], None, False),
    ("e4m3", 1, 2, 128, 16, [30000, 10], [2, 1], 25000, False),
])
def test_attention(fmt, heads, group, dim, page, past, counts, window, sinks, dtype):
    g = torch.Generator().manual_seed(dim * page + len(past))
    lists, table, cache = filled(g, fmt, heads, dim, page, past, counts)
    q = (1.5 * torch.randn(sum(counts), heads * group, dim, generator=g)).to(dtype).to(DEV)
    s = (torch.randn(heads * group, generator=g) + 1).to(DEV) if sinks else None
    first = cumulative(counts)
    got = lm_ops.attention_kv8(q, cache, table, ints(past), first, window=window, sinks=s)
    assert got.dtype == dtype and got.shape == q.shape
    check_attention(got, q, cache, table, past, counts, window=window, sinks=s, lists=lists)
    assert torch.equal(got, lm_ops.attention_kv8(q, cache, table, ints(past), first, window=window, sinks=s))
    if all(n == 1 for n in counts):
        assert torch.equal(got, lm_ops.attention_kv8(q, cache, table, ints(past), window=window, sinks=s))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts", [[1], [200]])
def test_sizes_of_values_scores_and_queries(counts, dtype):
    """Values of a page 2^40 times another's (seen alone by some rows), scores of hundreds, queries of any size, sinks far above and below."""
    g = torch.Generator().manual_seed(7)
    past = [96]
    n = counts[0]
    lists, table = tables(counts, past, 16, 30, g)
    cache = lm_ops.Kv8(30, 2, 64)
    k, v = torch.randn(96 + n, 2, 64, generator=g), torch.randn(96 + n, 2, 64, generator=g)
    v[16:32] *= 2.0 ** 30
    v[48:64] *= 2.0 ** -30
    v[64:80] = 0
    cache.append(k.to(DEV), v.to(DEV), table, ints([0]), ints([0, 96 + n]))
    q = torch.randn(n, 8, 64, generator=g)
    q[:, 0] = 30 * k[20, 0]                                        # a row whose weights lie on the large page, the small one, the page of zeros
    q[:, 1] = 30 * k[50, 0]
    q[:, 2] = 30 * k[70, 0]
    q[:, 3] *= 2.0 ** -40
    q[:, 4] *= 40
    q[:, 5] = 0
    q[:, 6] = torch.where(torch.arange(64) == 5, 2.0 ** 20, q[:, 6])
    q = q.to(dtype).to(DEV)
    for s in (None, torch.tensor([0.0, 300, -300, 1, 2, 3, 1e30, -math.inf], device=DEV)):
        got = lm_ops.attention_kv8(q, cache, table, ints(past), ints([0, n]), sinks=s)
        check_attention(got, q, cache, table, past, counts, sinks=s, lists=lists)
    got = lm_ops.attention_kv8(q, cache, table, ints(past), ints([0, n]), scale=3.0)
    check_attention(got, q, cache, table, past, counts, scale=3.0, lists=lists)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_of_nans_that_nobody_sees(dtype):
    """A page of NaNs changes the rows that see it, and no other: behind a row, beyond its window, in pages of other sequences."""
    g = torch.Generator().manual_seed(8)
    past, counts = [40, 0], [150, 20]
    lists, table = tables([190, 20], [0, 0], 16, 20, g)
    cache = lm_ops.Kv8(20, 2, 64)
    k, v = torch.randn(210, 2, 64, generator=g), torch.randn(210, 2, 64, generator=g)
    k[100, 1, 3] = math.nan                                        # page 6 of the first sequence (tokens 96 to 111), keys of head 1
    v[130, 0, 9] = math.inf                                        # page 8 (128 to 143), values of head 0
    cache.append(k.to(DEV), v.to(DEV), table, ints([0, 0]), ints([0, 190, 210]))
    q = torch.randn(170, 4, 64, generator=g).to(dtype).to(DEV)
    out = lm_ops.attention_kv8(q, cache, table, ints(past), ints([0, 150, 170]), window=30)
    nan = out.isnan().all(-1)
    assert torch.equal(nan, out.isnan().any(-1))
    pos = torch.arange(40, 190, device=DEV)
    sees = lambda a, b: (pos >= a) & (pos - 29 <= b)                # noqa: E731  (rows that see some of tokens a to b)
    assert torch.equal(nan[:150, 2], sees(96, 111)) and torch.equal(nan[:150, 3], sees(96, 111))
    assert torch.equal(nan[:150, 0], sees(128, 143)) and torch.equal(nan[:150, 1], sees(128, 143))
    assert not nan[150:].any()
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[96:112, 1], clean_v[128:144, 0] = 0, 0
    cache.append(clean_k.to(DEV), clean_v.to(DEV), table, ints([0, 0]), ints([0, 190, 210]))
    clean = lm_ops.attention_kv8(q, cache, table, ints(past), ints([0, 150, 170]), window=30)
    assert torch.equal(out[~nan], clean[~nan])
    # a query that is not finite is its own affair
    q[3, 1, 0], q[160, 2, 63] = math.nan, math.inf
    bad = lm_ops.attention_kv8(q, cache, table, ints(past), ints([0, 150, 170]), window=30)
    hit = torch.zeros_like(nan)
    hit[3, 1] = hit[160, 2] = True
    assert bad[hit].isnan().all() and torch.equal(bad[~hit], clean[~hit])


def test_many_sequences_and_empty_ones():
    g = torch.Generator().manual_seed(9)
    n = 700
    past = [int(x) for x in torch.randint(0, 60, (n,), generator=g)]
    counts = [int(x) for x in torch.randint(0, 3, (n,), generator=g)]
    lists, table, cache = filled(g, "e4m3", 1, 64, 16, past, counts)
    q = torch.randn(sum(counts) + 5, 3, 64, generator=g).bfloat16().to(DEV)
    got = lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts))
    check_attention(got, q, cache, table, past, counts, lists=lists)


def test_nothing_to_do():
    cache = lm_ops.Kv8(4, 2, 64)
    table, none = ints([[0, 1]]), torch.empty(0, 2, 64, device=DEV)
    cache.append(none, none, table, ints([0]), ints([0, 0]))
    assert lm_ops.attention_kv8(torch.empty(0, 4, 64, device=DEV), cache, table, ints([0]), ints([0, 0])).shape == (0, 4, 64)
    q = torch.randn(3, 4, 64, device=DEV)
    empty = torch.empty(0, 2, dtype=torch.int32, device=DEV)
    assert not lm_ops.attention_kv8(q, cache, empty, ints([]), ints([0])).any()
    assert not lm_ops.attention_kv8(q, cache, table, ints([0]), ints([0, 0])).any()
    k, v = cache.read(empty, ints([]), ints([0]), 5)
    assert k.shape == (5, 2, 64) and not k.any() and not v.any()


# ---- as it is used ---------------------------------------------------------------------------------------------------------------

def test_prompt_and_decoding_steps_in_a_captured_graph():
    """Prompts in one step, then decoding steps that a graph replays: what it reads of lengths and rows is the step's, and its bits are the calls'."""
    g = torch.Generator().manual_seed(10)
    H, G, D, prompts = 8, 2, 128, [100, 7, 33]
    lists, table = tables([n + 40 for n in prompts], [0] * 3, 16, 40, g)
    cache, twin = lm_ops.Kv8(40, G, D), lm_ops.Kv8(40, G, D)
    x = torch.randn(sum(prompts), H + 2 * G, D, generator=g).bfloat16().to(DEV)
    first = cumulative(prompts)
    for c in (cache, twin):
        c.append(x[:, H:H + G], x[:, H + G:], table, ints([0] * 3), first)
    out = lm_ops.attention_kv8(x[:, :H], cache, table, ints([0] * 3), first)
    check_attention(out, x[:, :H], cache, table, [0] * 3, prompts, lists=lists)
    step, past = torch.zeros(3, H + 2 * G, D, dtype=torch.bfloat16, device=DEV), ints(prompts)

    def go(c):
        c.append(step[:, H:H + G], step[:, H + G:], table, past)
        return lm_ops.attention_kv8(step[:, :H], c, table, past)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(twin)
    torch.cuda.current_stream().wait_stream(side)
    for t in ("keys", "values", "key_scales", "value_scales"):
        getattr(twin, t).copy_(getattr(cache, t))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = go(twin)
    for i in range(30):
        step.copy_(torch.randn(step.shape, generator=g) * (1 + i / 4))
        past.copy_(ints([n + i for n in prompts]))
        graph.replay()
        want = go(cache)
        assert torch.equal(got, want)
    check_attention(want, step[:, :H], cache, table, [n + 29 for n in prompts], [1] * 3, lists=lists)
    assert torch.equal(cache.keys, twin.keys) and torch.equal(cache.value_scales, twin.value_scales)


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(11)
    lists, table, cache = filled(g, "e4m3", 2, 128, 16, [6000, 100], [1, 1])
    q = torch.randn(2, 8, 128, generator=g).to(DEV)
    past = ints([6000, 100])
    want = lm_ops.attention_kv8(q, cache, table, past)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            got.append(lm_ops.attention_kv8(q, cache, table, past))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GB of codes: the last pages are written, read and seen where they are."""
    pages = (1 << 32) // (8 * 128 * 128) + 40                       # of 128 tokens, 8 heads of 128
    cache = lm_ops.Kv8(pages, 8, 128, page_size=128)
    g = torch.Generator().manual_seed(12)
    lists = [[pages - 1, 3, pages - 2], [pages - 30, pages // 2 + 1, 0]]
    table = ints(lists)
    x = torch.randn(600, 16, 128, generator=g).to(DEV)
    first = ints([0, 300, 600])
    cache.append(x[:, :8], x[:, 8:], table, ints([0, 0]), first)
    k, v = cache.read(table, ints([0, 0]), first, 600)
    small = lm_ops.Kv8(6, 8, 128, page_size=128)
    again = ints([[0, 1, 2], [3, 4, 5]])
    small.append(x[:, :8], x[:, 8:], again, ints([0, 0]), first)
    ks, vs = small.read(again, ints([0, 0]), first, 600)
    assert torch.equal(k, ks) and torch.equal(v, vs) and cache.keys[pages - 2].any()
    q = torch.randn(600, 16, 128, generator=g).bfloat16().to(DEV)
    assert torch.equal(lm_ops.attention_kv8(q, cache, table, ints([0, 0]), first), lm_ops.attention_kv8(q, small, again, ints([0, 0]), first))


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    cache = lm_ops.Kv8(4, 2, 64, device="cuda:1")
    x = torch.randn(20, 4, 64, device="cuda:1")
    table, past, first = (ints(y).to("cuda:1") for y in ([[0, 1]], [0], [0, 20]))
    cache.append(x[:, :2], x[:, 2:], table, past, first)
    assert torch.isfinite(lm_ops.attention_kv8(x, cache, table, past, first)).all()


# ---- where one way of doing it ends and another begins ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,group,dim,page,past,counts,window,width", [
    ("e4m3", 4, 128, 16, [0], [16], None, None),                    # 64 pairs of token and head
    ("e4m3", 4, 128, 16, [5], [17], None, None),
    ("int8", 4, 64, 32, [70, 3, 0, 2000], [16, 17, 64, 65], None, None),
    ("e4m3", 1, 64, 16, [0, 0, 0, 0, 300], [64, 65, 256, 257, 1], None, None),
    ("int8", 8, 128, 64, [5000, 9000], [33, 9], None, None),       # keys in chunks, and a sequence of few rows beside
    ("e4m3", 8, 112, 128, [40000], [70], None, None),
    ("e4m3", 2, 128, 16, [6000, 0, 64, 1], [129, 3, 200, 128], 777, None),
    ("int8", 1, 80, 16, [127, 128, 129], [129, 128, 127], None, None),
    ("e4m3", 4, 128, 16, [500, 600], [1, 2], None, 128),            # tables of 2048 tokens and of more
    ("e4m3", 4, 128, 16, [500, 600], [1, 2], None, 129),
    ("int8", 2, 64, 128, [2000, 17, 0], [1, 1, 1], None, 40),
])
def test_borders_between_ways(fmt, group, dim, page, past, counts, window, width, dtype):
    """Scores of many sizes: every row has tokens of its own anywhere in reach that take most of its weight."""
    g = torch.Generator().manual_seed(sum(counts) + dim)
    total = [p + n for p, n in zip(past, counts)]
    pages = sum(-(-t // page) for t in total) + 2
    lists, table = tables(counts, past, page, pages, g, width)
    cache = lm_ops.Kv8(pages, 2, dim, page_size=page, format=fmt)
    k, v = torch.randn(sum(total), 2, dim, generator=g), torch.randn(sum(total), 2, dim, generator=g)
    v *= torch.exp2(torch.randint(-3, 4, (sum(total), 1, 1), generator=g).double()).float()
    q = torch.randn(sum(counts), 2 * group, dim, generator=g)
    at = row = 0
    for p, n in zip(past, counts):
        for i in range(n):
            low = max(0, p + i + 1 - (window or 1 << 40))
            own = torch.randint(low, p + i + 1, (2 * group,), generator=g)
            q[row + i] += k[at + own, torch.arange(2 * group) // group] * torch.randint(0, 3, (2 * group, 1), generator=g)
        at, row = at + p + n, row + n
    cache.append(k.to(DEV), v.to(DEV), table, ints([0] * len(past)), cumulative(total))
    q = q.to(dtype).to(DEV)
    got = lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts), window=window)
    check_attention(got, q, cache, table, past, counts, window=window, lists=lists)
    assert torch.equal(got, lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts), window=window))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("step", [0, 1, 2])
def test_long_sequences_among_many(step, dtype):
    """Runs of work that share a tile, tens of them, beside runs that have many tiles: every border falls elsewhere."""
    g = torch.Generator().manual_seed(17 + step)
    past = [5] * 90 + [23000 + 1500 * i + 333 * step for i in range(12)] + [int(x) for x in torch.randint(0, 200, (230,), generator=g)]
    counts = [1] * len(past)
    lists, table, cache = filled(g, "e4m3", 1, 64, 16, past, counts)
    q = torch.randn(len(past), 2, 64, generator=g).to(dtype).to(DEV)
    got = lm_ops.attention_kv8(q, cache, table, ints(past))
    check_attention(got, q, cache, table, past, counts, lists=lists)
    few = lm_ops.attention_kv8(q[90:93], cache, table[90:93], ints(past[90:93]))               # (a part of a tile for every CTA)
    check_attention(few, q[90:93], cache, table[90:93], past[90:93], [1] * 3, lists=lists[90:93])


def test_rows_behind_the_last_sequence_and_between_none():
    """Rows in front of the first sequence's, behind the last one's, and of sequences that have none: zeros, whichever way the others go."""
    g = torch.Generator().manual_seed(13)
    lists, table, cache = filled(g, "e4m3", 2, 64, 16, [30, 0, 10, 50], [20, 0, 90, 1])
    q = torch.randn(130, 8, 64, generator=g).bfloat16().to(DEV)
    past = ints([30, 0, 10, 50])
    want = lm_ops.attention_kv8(q[7:118], cache, table, past, cumulative([20, 0, 90, 1]))
    check_attention(want, q[7:118], cache, table, [30, 0, 10, 50], [20, 0, 90, 1], lists=lists)
    got = lm_ops.attention_kv8(q, cache, table, past, ints([7, 27, 27, 117, 118]))
    assert not got[:7].any() and not got[118:].any() and torch.equal(got[7:118], want)
    one = lm_ops.attention_kv8(q, cache, table[2:3], past[2:3], ints([27, 117]))             # (a step of one sequence)
    assert not one[:27].any() and not one[117:].any()
    check_attention(one[27:117], q[27:117], cache, table[2:3], [10], [90], lists=lists[2:3])
    none = lm_ops.attention_kv8(q, cache, table, ints([-1, -5, -2 ** 31, -1]), ints([7, 27, 27, 117, 118]))
    assert not none.any()


def test_positions_far_beyond_the_table():
    """Lengths that no table holds, up to the largest there are: what is there is seen, the rest is not."""
    g = torch.Generator().manual_seed(14)
    cache = lm_ops.Kv8(4, 1, 64)
    table = ints([[0, 1, 2, 3]])
    x = torch.randn(64, 2, 64, generator=g).to(DEV)
    cache.append(x[:, :1], x[:, 1:], table, ints([0]), ints([0, 64]))
    keys = cache.keys.clone()
    for rows in (1, 90):
        q = torch.randn(rows, 4, 64, generator=g).bfloat16().to(DEV)
        want = lm_ops.attention_kv8(q, cache, table, ints([63]), ints([0, rows]))
        for past in (64, 100, 5000, 2 ** 30, 2 ** 31 - 1):
            got = lm_ops.attention_kv8(q, cache, table, ints([past]), ints([0, rows]))
            assert torch.isfinite(got).all() and (got.float() - want.float()).abs().max() < 2.0 ** -5
            assert not lm_ops.attention_kv8(q, cache, table, ints([past]), ints([0, rows]), window=1)[1:].any()
            y = torch.randn(rows, 2, 64, generator=g).to(DEV)
            cache.append(y[:, :1], y[:, 1:], table, ints([past]), ints([0, rows]))
            assert torch.equal(cache.keys, keys) and not cache.read(table, ints([past]), ints([0, rows]), rows)[0].any()


def test_a_mixed_step_in_a_captured_graph():
    """Prompts beside decoding sequences; which is which, and how long, is read anew by every replay.  Two graphs in turn share nothing."""
    g = torch.Generator().manual_seed(15)
    lists, table, cache = filled(g, "int8", 2, 128, 16, [3000, 300, 2500, 80], [64] * 4)
    q = torch.randn(128, 8, 128, generator=g).bfloat16().to(DEV)
    past, first = ints([0] * 4), ints([0] * 5)
    steps = [([2990, 300, 7, 0], [1, 64, 1, 62]), ([0, 299, 2500, 80], [60, 1, 60, 1]), ([3000, 0, 1, 5], [0, 0, 64, 0]), ([2999, 17, 2000, 3], [1, 1, 1, 1])]
    lm_ops.attention_kv8(q, cache, table, past, first)
    graphs = []
    for window in (None, 500):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lm_ops.attention_kv8(q, cache, table, past, first, window=window)
        graphs.append((graph, out, window))
    for p, n in steps + steps[::-1]:
        past.copy_(ints(p))
        first.copy_(cumulative(n))
        for graph, out, window in graphs:
            graph.replay()
        for graph, out, window in graphs:
            assert torch.equal(out, lm_ops.attention_kv8(q, cache, table, past, first, window=window))
            check_attention(out, q, cache, table, p, n, window=window, lists=lists)


@pytest.mark.parametrize("past,counts", [([300], [200]), ([9000], [40]), ([20, 900], [100, 1])])
def test_a_wait_that_ran_out_shows(past, counts):
    """With no looks at any barrier every wait ends at once: results of many rows are NaN, the next call reports it, the one behind is whole again."""
    import ctypes as C

    from dia_tts_prune_b200 import _lm_lib
    g = torch.Generator().manual_seed(16)
    lists, table, cache = filled(g, "e4m3", 2, 128, 16, past, counts)
    q = torch.randn(sum(counts), 8, 128, generator=g).bfloat16().to(DEV)
    call = lambda: lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts))          # noqa: E731
    polls = getattr(_lm_lib.load(), "_ZN3dia15gemm_pair_pollsEv")
    polls.restype = C.POINTER(C.c_uint)
    want, kept = call(), polls()[0]
    polls()[0] = 0
    try:
        got = call()
    finally:
        polls()[0] = kept
    torch.cuda.synchronize()
    assert got[:counts[0]].isnan().all() and torch.equal(got[counts[0]:], want[counts[0]:])
    with pytest.raises(RuntimeError):
        call()
    for _ in range(3):
        assert torch.equal(call(), want)
