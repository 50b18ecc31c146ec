"""What no row sees changes nothing, whatever it is: beside queries of any size, behind a sequence's last token, in front of its window.

Bounds are those of the attention over the cache in 8 bits (test_kv8_gpu.py); everything else here is equal or not."""

import math

import pytest
import torch

from dia_tts_prune_b200 import lm_ops
from test_kv8_gpu import DEV, HALF, check_attention, cumulative, ints, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,past", [(100, 0), (12, 40)])        # (in tiles of 256 pairs, of 16)
def test_queries_that_are_not_finite_and_see_nothing(rows, past, dtype):
    """A row that sees nothing is zeros whatever its query; one that sees something is NaN."""
    g = torch.Generator().manual_seed(rows)
    cache = lm_ops.Kv8(12, 2, 64)
    x = torch.randn(past + rows, 4, 64, generator=g).to(DEV)
    lists = [[7, 3, -1, 12, -5, 1, 0]]                             # tokens 32 to 79 are on no page of the pool
    table = ints(lists)
    cache.append(x[:, :2], x[:, 2:], table, ints([0]), ints([0, past + rows]))
    q = torch.randn(rows, 8, 64, generator=g).to(dtype).to(DEV)
    for sinks in (None, torch.randn(8, generator=g).to(DEV)):
        clean = lm_ops.attention_kv8(q, cache, table, ints([past]), ints([0, rows]), window=16, sinks=sinks)
        check_attention(clean, q, cache, table, [past], [rows], window=16, sinks=sinks, lists=lists)
        pos = past + torch.arange(rows, device=DEV)
        blind = (pos >= 47) & (pos <= 79)
        assert blind.any() and not blind.all() and not clean[blind].any()
        for bad in (math.nan, math.inf, -math.inf):
            for r in (int(blind.nonzero()[0]), int(blind.nonzero()[-1]), int((~blind).nonzero()[0]), int((~blind).nonzero()[-1])):
                broken = q.clone()
                broken[r, 1, 5], broken[r, 6, 63] = bad, bad
                got = lm_ops.attention_kv8(broken, cache, table, ints([past]), ints([0, rows]), window=16, sinks=sinks)
                want = clean.clone()
                if not blind[r]:
                    want[r, 1], want[r, 6] = math.nan, math.nan
                assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0)), (bad, r)
    none = torch.full_like(q, math.nan)                            # nothing of the sequence is there at all
    for t, p in ((ints([[-1] * 7]), past), (table, -1)):
        assert not lm_ops.attention_kv8(none, cache, t, ints([p]), ints([0, rows])).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,dim,page,past,counts,window", [
    ("e4m3", 128, 16, [0], [100], None),
    ("int8", 64, 32, [300, 0], [90, 70], 40),
    ("e4m3", 80, 16, [5000, 3], [33, 1], None),
    ("int8", 128, 16, [100], [200], 16),
    ("e4m3", 96, 128, [400], [129], 200),
])
@pytest.mark.parametrize("scale", [None, 2.0 ** -7, 2.0 ** -126])
def test_small_queries_beside_pages_of_zeros(fmt, dim, page, past, counts, window, scale, dtype):
    """Keys of zeros, pages that were never written, and pages that are reserved behind the last token: their steps are 2^-100 or none at all."""
    g = torch.Generator().manual_seed(dim + page)
    total = [p + n for p, n in zip(past, counts)]
    slots = [-(-t // page) + 9 for t in total]
    pages = sum(slots)
    order = torch.randperm(pages, generator=g).tolist()
    lists = [[order.pop() for _ in range(max(slots))] if i == 0 else [order.pop() for _ in range(min(len(order), max(slots)))] for i in range(len(total))]
    lists = [row + [-1] * (max(slots) - len(row)) for row in lists]
    table = ints(lists)
    cache = lm_ops.Kv8(pages, 2, dim, page_size=page, format=fmt)
    k, v = torch.randn(sum(total), 2, dim, generator=g), torch.randn(sum(total), 2, dim, generator=g)
    at = 0
    for n in total:
        slot = torch.arange(n) // page
        k[at:at + n][slot % 3 == 1] = 0
        at += n
    cache.append(k.to(DEV), v.to(DEV), table, ints([0] * len(total)), cumulative(total))
    for row, n in zip(lists, total):
        for p in row[3:-(-n // page):4]:                           # (given to the sequence, and not written)
            for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales):
                t[p] = 0
    shape = torch.randn(sum(counts), 8, dim, generator=g)
    for size in (1.0, 2.0 ** -4, 2.0 ** -8, 2.0 ** -14, 2.0 ** -24, 2.0 ** -35, 2.0 ** -40, 0.0):
        q = (size * shape).to(dtype).to(DEV)
        got = lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts), scale=scale, window=window)
        check_attention(got, q, cache, table, past, counts, scale=scale, window=window, lists=lists)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fmt,page,past,counts,window", [
    ("e4m3", 16, [0], [100], None),
    ("int8", 32, [40, 7], [100, 200], None),
    ("e4m3", 16, [200], [90], 30),                                 # pages in front of the window, in the first row's 128 tokens
    ("e4m3", 64, [6000, 130], [33, 70], 3000),                     # keys in chunks
    ("int8", 16, [129, 300], [1, 3], 50),                          # few rows
])
def test_unused_places_of_a_table(fmt, page, past, counts, window, dtype):
    """Behind the page of a sequence's last token, and in front of the page of the first token that anyone sees, a table may name any page: no bit changes."""
    g = torch.Generator().manual_seed(page + len(past))
    total = [p + n for p, n in zip(past, counts)]
    need = [-(-t // page) for t in total]
    width, used = max(need) + 9, sum(need)
    cache = lm_ops.Kv8(used + 3, 2, 64, page_size=page, format=fmt)
    for t, fill in ((cache.keys, 120 if fmt == "e4m3" else 127), (cache.values, 120 if fmt == "e4m3" else 127), (cache.key_scales, 2.0 ** 100), (cache.value_scales, 2.0 ** 100)):
        t[used:] = fill                                            # three pages of others, of very large numbers, one of which stands for NaNs
    cache.value_scales[used + 1] = cache.key_scales[used + 2] = math.nan
    order = torch.randperm(used, generator=g).tolist()
    lists = []
    for n in need:
        lists.append([order.pop() for _ in range(n)] + [-1] * (width - n))
    x = torch.randn(sum(total), 4, 64, generator=g) * 2.0 ** -20   # (its pages' steps are 2^80 below the others')
    cache.append(x[:, :2].to(DEV) * 2.0 ** 20, x[:, 2:].to(DEV), ints(lists), ints([0] * len(total)), cumulative(total))
    q = torch.randn(sum(counts), 8, 64, generator=g).to(dtype).to(DEV)
    first = cumulative(counts)
    want = lm_ops.attention_kv8(q, cache, ints(lists), ints(past), first, window=window)
    if dtype != torch.float16:                                     # (which has no such small numbers)
        check_attention(want, q, cache, ints(lists), past, counts, window=window, lists=lists)
    for other in (used, used + 1, used + 2, 0):
        changed = [list(row) for row in lists]
        for row, p, n in zip(changed, past, need):
            row[n:] = [other] * (width - n)
            front = max(0, p + 1 - window) // page if window else 0
            row[:front] = [other] * front
        got = lm_ops.attention_kv8(q, cache, ints(changed), ints(past), first, window=window)
        assert torch.equal(got, want), other


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("past,counts", [([50], [1]), ([0], [100]), ([9000], [20])])
def test_sinks_of_any_size(past, counts, dtype):
    """Up to the largest and down to the lowest number of float32, which times log2(e) are none; the infinities: nothing in the denominator, and no number."""
    g = torch.Generator().manual_seed(counts[0])
    top = torch.finfo(torch.float32).max
    lists = [list(range(-(-(past[0] + counts[0]) // 16)))]
    table = ints(lists)
    cache = lm_ops.Kv8(len(lists[0]), 2, 64)
    x = torch.randn(past[0] + counts[0], 4, 64, generator=g).to(DEV)
    cache.append(x[:, :2], x[:, 2:], table, ints([0]), cumulative([len(x)]))
    q = torch.randn(counts[0], 8, 64, generator=g).to(dtype).to(DEV)
    sinks = torch.tensor([top, 0.7 * top, 0.69 * top, 2.0 ** 100, -top, -0.69 * top, -math.inf, 0.0], device=DEV)
    got = lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts), sinks=sinks)
    check_attention(got, q, cache, table, past, counts, sinks=sinks, lists=lists)
    assert not got[:, :4].any()
    bare = lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts))
    assert torch.equal(got[:, 4:7], bare[:, 4:7])
    for bad in (math.inf, math.nan):
        sinks[3] = bad
        again = lm_ops.attention_kv8(q, cache, table, ints(past), cumulative(counts), sinks=sinks)
        assert again[:, 3].isnan().all() and torch.equal(again[:, 4:], got[:, 4:])
    # rows that see nothing have nothing to give, whatever the sink
    assert not lm_ops.attention_kv8(q, cache, ints([[-1]]), ints(past), cumulative(counts), sinks=torch.full((8,), top, device=DEV)).any()


@pytest.mark.parametrize("order", [[0, 10, 5, 12], [0, 5, 3, 8], [7, 3, 12, 0], [12, 0, 0, 0], [-4, 9, 2, 40], [5, 1 << 30, -(1 << 31), 12]])
@pytest.mark.parametrize("sequences", [3, 1500])
@pytest.mark.parametrize("rows", [12, 2000])
def test_rows_of_sequences_in_no_order(order, sequences, rows):
    """`first` that decreases somewhere: which rows are whose is not said, but every call ends, and pages that the table does not name stay what they are."""
    g = torch.Generator().manual_seed(rows)
    cache = lm_ops.Kv8(2 * sequences + 8, 2, 64)
    for t in (cache.keys, cache.values):
        t.fill_(56)
    for t in (cache.key_scales, cache.value_scales):
        t.fill_(2.0)
    before = [t.clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales)]
    table = torch.arange(2 * sequences, dtype=torch.int32, device=DEV).view(sequences, 2)
    past = ints([5, 0, 20] + [1] * (sequences - 3))
    first = ints([v * rows // 12 if abs(v) < 100 else v for v in order] + [rows - 3] * (sequences - 3))
    x = torch.randn(rows, 4, 64, generator=g).to(DEV)
    cache.append(x[:, :2], x[:, 2:], table, past, first)
    torch.cuda.synchronize()
    for t, b in zip((cache.keys, cache.values, cache.key_scales, cache.value_scales), before):
        assert torch.equal(t[2 * sequences:], b[2 * sequences:])
    assert torch.isfinite(cache.key_scales).all() and torch.isfinite(cache.value_scales).all()
    assert all(torch.isfinite(y).all() for y in cache.read(table, past, first, rows))
    for dtype in (torch.bfloat16, torch.float32):
        q = torch.randn(rows, 8, 64, generator=g).to(dtype).to(DEV)
        lm_ops.attention_kv8(q, cache, table, past, first)
    torch.cuda.synchronize()
    # and a step in order behind it is what it should be
    twin = lm_ops.Kv8(2 * sequences + 8, 2, 64)
    first = ints([0, 4, 8] + [12] * (sequences - 2))
    for c in (cache, twin):
        c.append(x[:12, :2], x[:12, 2:], table, ints([0] * sequences), first)
    q = torch.randn(12, 8, 64, generator=g).to(DEV)
    got, want = (lm_ops.attention_kv8(q, c, table, ints([0] * sequences), first) for c in (cache, twin))
    assert torch.equal(got, want)


def test_rows_counted_many_times():
    """`first` that goes up and down 2049 times: what its sequences' rows come to passes 32 bits, and the call ends all the same."""
    sequences, rows = 4098, 1 << 16
    cache = lm_ops.Kv8(4, 1, 1)
    q = torch.zeros(rows, 4096, 1, dtype=torch.bfloat16, device=DEV)   # 2^20 tiles of 256 pairs
    table = torch.full((sequences, 1), -1, dtype=torch.int32, device=DEV)
    past = torch.zeros(sequences, dtype=torch.int32, device=DEV)
    first = torch.zeros(sequences + 1, dtype=torch.int32, device=DEV)
    first[1::2] = rows
    lm_ops.attention_kv8(q, cache, table, past, first)
    torch.cuda.synchronize()
    first[2:] = rows                                               # (the first sequence's, once)
    assert not lm_ops.attention_kv8(q, cache, table, past, first).any()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -12])
@pytest.mark.parametrize("past,count", [(0, 1), (30, 2), (700, 1)])
def test_float32_rows_keep_their_bits(fmt, size, past, count):
    """Pages of values of many powers: what the references of a row's weights are rounded by does not show in it."""
    g = torch.Generator().manual_seed(past + count)
    n = 100
    counts, pasts = [count] * n, [max(0, past - i) for i in range(n)]
    total = [p + c for p, c in zip(pasts, counts)]
    pages = sum(-(-t // 16) for t in total)
    lists, table = tables(counts, pasts, 16, pages, g)
    cache = lm_ops.Kv8(pages, 2, 64, format=fmt)
    k, v = torch.randn(sum(total), 2, 64, generator=g), torch.randn(sum(total), 2, 64, generator=g)
    v *= torch.exp2(torch.randint(-30, 31, (len(v) // 16 + 1, 1, 1), generator=g).float())[torch.arange(len(v)) // 16]
    cache.append(k.to(DEV), v.to(DEV), table, ints([0] * n), cumulative(total))
    q = (size * torch.randn(sum(counts), 16, 64, generator=g)).to(DEV)
    got = lm_ops.attention_kv8(q, cache, table, ints(pasts), cumulative(counts))
    check_attention(got, q, cache, table, pasts, counts, lists=lists)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("past,count", [(0, 1), (333, 3), (5000, 1), (0, 200), (3000, 100)])
def test_rows_with_one_large_weight(past, count, fmt, dtype):
    """A row whose weight lies on one token (the others have less than 2^-60 of it) is that token's values, which 8 significant bits and a power of two give every type exactly."""
    g = torch.Generator().manual_seed(past + count)
    n = past + count
    lists, table = tables([count], [past], 16, -(-n // 16), g)
    cache = lm_ops.Kv8(-(-n // 16), 2, 64, format=fmt)
    k, v = torch.randn(n, 2, 64, generator=g), torch.randn(n, 2, 64, generator=g)
    k /= k.norm(dim=-1, keepdim=True)
    cache.append(k.to(DEV), v.to(DEV), table, ints([0]), ints([0, n]))
    own = (torch.rand(count, 8, generator=g) * (past + 1 + torch.arange(count))[:, None]).long()
    head = (torch.arange(8) // 4).expand(count, 8)
    q = (4096 * k[own, head]).to(dtype).to(DEV)
    read_k, read_v = (y.double() for y in cache.read(table, ints([0]), ints([0, n]), n))
    z = torch.einsum("rhd,thd->rht", q.double(), read_k.repeat_interleave(4, 1)) / 8
    t = torch.arange(n, device=DEV)
    z = z.masked_fill(t > past + torch.arange(count, device=DEV)[:, None, None], -math.inf)
    best = z.argmax(-1)
    top = z.topk(min(2, n), -1).values
    alone = top[..., 0] - top[..., -1] > 60 * math.log(2) if n > 1 else torch.ones(count, 8, dtype=torch.bool, device=DEV)
    alone |= (past + torch.arange(count, device=DEV) == 0)[:, None]
    assert alone.float().mean() > 0.9
    got = lm_ops.attention_kv8(q, cache, table, ints([past]), ints([0, count]))
    want = read_v[best, head.to(DEV)]
    assert torch.equal(want, want.to(dtype).double()) and torch.equal(got[alone].double(), want[alone])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_the_largest_weight_of_few_rows_is_not_rounded(fmt, dtype):
    """Where pages' values have one power, a row's largest weight is 2^14 in fp16: what weights are rounded by (2^-11) counts for the others alone.  The rest of the bound is
    check_attention's, of scores and sums."""
    g = torch.Generator().manual_seed(31)
    n = 100
    past = [15 + i // 2 for i in range(n)]
    total = [p + 1 for p in past]
    lists, table = tables([1] * n, past, 16, sum(-(-t // 16) for t in total), g)
    cache = lm_ops.Kv8(sum(-(-t // 16) for t in total), 1, 64, format=fmt)
    k, v = torch.randn(sum(total), 1, 64, generator=g), torch.randn(sum(total), 1, 64, generator=g).clamp(-5, 5)
    k /= k.norm(dim=-1, keepdim=True)
    q, at = torch.empty(n, 4, 64), 0
    for i, t in enumerate(total):
        v[at:at + t:16, 0, 63] = 6                                 # (in every page)
        q[i] = 60 * k[at + torch.randint(0, t, (4,), generator=g), 0]
        at += t
    cache.append(k.to(DEV), v.to(DEV), table, ints([0] * n), cumulative(total))
    q = q.to(dtype).to(DEV)
    got = lm_ops.attention_kv8(q, cache, table, ints(past))
    assert cache.value_scales[[p for row in lists for p in row if p >= 0]].unique().numel() == 1
    large = 0
    for i, t in enumerate(total):
        k1, v1 = (y.double()[:, 0] for y in cache.read(table[i:i + 1], ints([0]), ints([0, t]), t))
        z = q[i].double() @ k1.T / 8
        p = torch.softmax(z, -1)
        large += int((p.amax(-1) > 0.5).sum())
        rest = p.scatter(1, p.argmax(-1, keepdim=True), 0.0)
        A = (q[i].double().abs() @ k1.abs().T / 8).amax(-1, keepdim=True)
        e = A * (2.0 ** -22 + (64 / 16 + 8) * 2.0 ** -23)
        o, B = p @ v1, p @ v1.abs()
        bound = HALF[dtype] * o.abs() + 2.0 ** -11 * (rest @ v1.abs()) + B * (2 * e + 2.0 ** -20) + t * 6 * 2.0 ** -37 + 2.0 ** -25
        assert ((got[i].double() - o).abs() <= bound).all(), i
    assert large > 200
