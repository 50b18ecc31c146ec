"""What the operators for a cache in 8 bits are measured on.

A served model writes the keys and values of its tokens into pages, 8 bits a number with one power of two for the tokens of a page and head,
reads them back, and attends to them: one token per request, or a portion of a prompt.

Kinds of a case
  write    a step's keys and values are appended behind what their sequences hold, and the pages that changed are read back
  read     keys and values of whole sequences as numbers again (a prefix handed to another program, a check of what 8 bits cost)
  attend   grouped-query attention of a step's rows over the cache, causal, with a window and a sink where the case says so

``rows`` and ``past`` are the new tokens of every sequence and the tokens that it holds before them, ``heads`` query heads over ``kv_heads``,
``page`` tokens of a page, ``format`` of a number (E4M3 or two's complement), ``dtype`` of the rows that come in and go out.  Lists are texts.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
LOWEST = -100                                                     # of a page's exponents


def _ints(text):
    return [int(t) for t in str(text).split(",")]


def _same(n, count):
    return ",".join([str(n)] * count)


def _ragged(count, longest):
    """Lengths of running requests: most of them well below the longest."""
    return ",".join(str(max(1, round(longest * (0.03 + 0.97 * ((i * 37 % count) / count) ** 1.5)))) for i in range(count))


def listed():
    wide = dict(heads=16, kv_heads=4, dim=128)                    # the benchmark's language models of width 2048
    narrow = dict(heads=8, kv_heads=2, dim=128)                   # and of width 1024
    return [
        # a decoding step of eight requests: latency
        dict(name="write_token8", kind="write", **wide, page=16, format="e4m3", dtype="bfloat16", rows=_same(1, 8), past="1024,1025,1039,7,500,2000,4095,333"),
        # four prompts in one step: bytes
        dict(name="write_prompts", kind="write", heads=32, kv_heads=8, dim=128, page=16, format="e4m3", dtype="bfloat16", rows="4096,2048,1500,548", past="0,0,700,3000"),
        # odd sizes, rows as the engine has them
        dict(name="write_odd", kind="write", heads=6, kv_heads=3, dim=80, page=32, format="int8", dtype="float32", rows="201,1,77", past="13,95,0"),
        # a long prefix for another program
        dict(name="read_prefix", kind="read", **wide, page=16, format="e4m3", dtype="bfloat16", rows="65536,32768", past="0,0"),
        # the middle of some sequences, an odd size
        dict(name="read_odd", kind="read", heads=6, kv_heads=3, dim=80, page=32, format="int8", dtype="float32", rows="861,130,1", past="40,3,999"),
        # one request: latency
        dict(name="attend_token", kind="attend", **wide, page=16, format="e4m3", dtype="bfloat16", rows="1", past="1024", window=0, sinks=False),
        # eight requests whose rows are float32, as the engine's are
        dict(name="attend_token8", kind="attend", **wide, page=16, format="e4m3", dtype="float32", rows=_same(1, 8), past=_same(4096, 8), window=0, sinks=False),
        # a full server: many requests of all lengths
        dict(name="attend_token64", kind="attend", heads=32, kv_heads=8, dim=128, page=16, format="e4m3", dtype="bfloat16", rows=_same(1, 64), past=_ragged(64, 24576), window=0, sinks=False),
        # one request with a very long past: nothing to split but the past
        dict(name="attend_long", kind="attend", **narrow, page=64, format="int8", dtype="bfloat16", rows="1", past="131071", window=0, sinks=False),
        # a whole prompt
        dict(name="attend_prompt", kind="attend", **wide, page=16, format="e4m3", dtype="bfloat16", rows="4096", past="0", window=0, sinks=False),
        # a portion of a long prompt
        dict(name="attend_portion", kind="attend", heads=32, kv_heads=8, dim=128, page=32, format="e4m3", dtype="bfloat16", rows="512", past="16384", window=0, sinks=False),
        # prompt portions and decoding requests in one step, a window and a sink, another head size
        dict(name="attend_mixed", kind="attend", heads=16, kv_heads=8, dim=64, page=64, format="int8", dtype="bfloat16", rows="1,300,1,37,1,1000,1,1", past="5000,17,1023,64,1,2500,0,9999",
             window=1024, sinks=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend"])
    while True:
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = min(48, kv * rng.choice([1, 2, 3, 4, 6, 8, 16]))
        heads -= heads % kv
        case = dict(kind=kind, heads=heads, kv_heads=kv, dim=rng.choice([64, 128, 128, 96, 80, rng.randint(8, 256)]), page=rng.choice([16, 16, 32, 64, 128]),
                    format=rng.choice(["e4m3", "int8"]), dtype=rng.choice(["bfloat16", "bfloat16", "float32", "float16"]))
        sequences = _log_uniform(rng, 1, 64)
        if kind == "read":
            rows = [_log_uniform(rng, 1, 65536) for _ in range(sequences)]
            past = [rng.choice([0, _log_uniform(rng, 1, 4096)]) for _ in range(sequences)]
        else:
            most = _log_uniform(rng, 1, 4096) if rng.random() < 0.5 else 1
            rows = [_log_uniform(rng, 1, most) if rng.random() < 0.7 else 1 for _ in range(sequences)]
            longest = _log_uniform(rng, 1, 131072 if sequences < 3 else 24576)
            past = [rng.choice([0, _log_uniform(rng, 1, longest), longest]) if most > 1 else _log_uniform(rng, 1, longest) for _ in range(sequences)]
        case.update(rows=",".join(map(str, rows)), past=",".join(map(str, past)))
        tokens = sum(r + p for r, p in zip(rows, past)) if kind == "attend" else sum(rows)
        if kind == "attend":
            case.update(window=rng.choice([0, 0, _log_uniform(rng, 16, 4096)]), sinks=rng.random() < 0.4)
        if (sum(r + p for r, p in zip(rows, past)) * kv * case["dim"] <= 400000 * 8 * 128 and tokens * kv * case["dim"] <= (400000 if kind == "attend" else 98304) * 4 * 128
                and (kind != "attend" or _pairs(case) * heads * case["dim"] * (3 if case["dtype"] == "float32" else 1) <= 512 * 16384 * 32 * 128)):
            return case


def _pairs(case):
    """How many (row, token) pairs a causal row with a window sees."""
    total = 0
    for n, p in zip(_ints(case["rows"]), _ints(case["past"])):
        w = case.get("window") or (n + p)
        full = max(0, min(n, w - p))                              # rows that see all in front of them
        total += full * p + full * (full + 1) // 2 + (n - full) * w
    return total


def _seen(case):
    """Tokens of the cache that some row sees."""
    total = 0
    for n, p in zip(_ints(case["rows"]), _ints(case["past"])):
        total += n + min(p, (case.get("window") or (n + p)) - 1)
    return total


# ---- numbers in 8 bits -----------------------------------------------------------------------------------------------------

def _table(fmt, device):
    """The numbers that the 256 codes stand for, before their page's scale."""
    c = torch.arange(256, device=device)
    if fmt == "int8":
        return torch.where(c > 127, c - 256, c).float()
    e, m = (c >> 3) & 15, c & 7
    v = torch.where(e == 0, m.float() * 2.0 ** -9, (8 + m).float() * torch.exp2((e - 10).float()))
    return torch.where(c > 127, -v, v)


def _exponents(most, fmt):
    """The smallest e for which most <= LARGEST 2^e, at least LOWEST."""
    f, x = torch.frexp(most)
    bits, part = (9, 0.875) if fmt == "e4m3" else (7, 127 / 128)
    return torch.where(most > 0, x - bits + (f > part).to(x.dtype), LOWEST).clamp(min=LOWEST)


def _power(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(v, fmt):
    """Codes of numbers that are at most LARGEST, to the nearest, half way to the even one."""
    if fmt == "int8":
        return torch.round(v).to(torch.int32).bitwise_and(255).to(torch.uint8)
    return v.to(torch.float8_e4m3fn).view(torch.uint8)


def _filled(g, case, pages, loud):
    """Codes [pages, kv_heads, page, dim] and scales [pages, kv_heads] of pages full of tokens."""
    G, P, D = case["kv_heads"], case["page"], case["dim"]
    codes = torch.empty(pages, G, P, D, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, G, dtype=torch.float32, device="cuda")
    for at in torch.arange(pages).split(max(1, (1 << 27) // (G * P * D))):
        part = slice(int(at[0]), int(at[-1]) + 1)
        x = torch.randn(len(at), G, P, D, generator=g, device="cuda") * loud
        e = _exponents(x.abs().amax((2, 3)), case["format"])
        scales[part] = _power(e)
        codes[part] = _codes(x * _power(-e)[:, :, None, None], case["format"])
    return codes, scales


def _case_sizes(case):
    rows, past = _ints(case["rows"]), _ints(case["past"])
    return rows, past, [-(-(n + p) // case["page"]) for n, p in zip(rows, past)]


def _first(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, past, need = _case_sizes(case)
    H, G, D, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    pages = sum(need) + 3                                         # a pool in which some pages are free
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(rows), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    # some channels of the keys are much larger than the others, as trained models have them; tokens of values differ in size
    loud = torch.where(torch.rand(G, 1, D, generator=g, device="cuda") < 0.03, 6.0, 1.0)
    keys, key_scales = _filled(g, case, pages, loud)
    values, value_scales = _filled(g, case, pages, torch.exp(0.5 * torch.randn(G, case["page"], 1, generator=g, device="cuda")))
    state = dict(case=case, table=table, past=torch.tensor(past, dtype=torch.int32, device="cuda"), first=_first(rows), total=sum(rows), host=(rows, past))
    if case["kind"] == "write":
        # the keys and values of a step lie in one projection with its queries
        x = torch.randn(sum(rows), H + 2 * G, D, generator=g, device="cuda")
        x[:, H:H + G] *= loud[:, 0] * torch.exp(0.3 * torch.randn(sum(rows), 1, 1, generator=g, device="cuda"))
        x = x.to(dtype)
        state.update(k=x[:, H:H + G], v=x[:, H + G:])
        back = [p // case["page"] * case["page"] for p in past]   # from the start of the page that gets the first new token
        counts = [n + p - b for n, p, b in zip(rows, past, back)]
        state.update(back=torch.tensor(back, dtype=torch.int32, device="cuda"), back_first=_first(counts), back_total=sum(counts), back_host=(counts, back))
    elif case["kind"] == "attend":
        q = torch.randn(sum(rows), H, D, generator=g, device="cuda") / torch.where(loud[:, 0] > 1, 6.0, 1.0).repeat_interleave(H // G, 0)
        q *= torch.exp(0.5 * torch.randn(1, H, 1, generator=g, device="cuda"))
        state.update(q=q.to(dtype), sinks=torch.randn(H, generator=g, device="cuda") + 2 if case["sinks"] else None)
    if own:
        from dia_tts_prune_b200 import lm_ops
        cache = lm_ops.Kv8(pages, G, D, page_size=case["page"], format=case["format"], device="cuda")
        cache.keys[..., :D], cache.values[..., :D] = keys, values
        cache.key_scales.copy_(key_scales)
        cache.value_scales.copy_(value_scales)
        state["cache"] = cache
    else:
        state["cache"] = dict(k=keys, v=values, ks=key_scales, vs=value_scales)
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _places(case, table, counts, starts):
    """Page and place in it of every packed row."""
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    pos = torch.cat([torch.arange(s, s + n, device="cuda") for n, s in zip(counts, starts)])
    return table[seq, pos // case["page"]].long(), pos % case["page"]


def _plain_append(case, codes, scales, x, table, rows, past):
    fmt = case["format"]
    page, place = _places(case, table, rows, past)
    x = x.float()
    most = x.abs().amax(-1)                                       # [rows, kv_heads]
    need = torch.zeros_like(scales).index_reduce_(0, page, most, "amax")
    e = _exponents(need, fmt)
    begun = [i for i, (n, p) in enumerate(zip(rows, past)) if n and p % case["page"]]
    if begun:                                                     # pages that hold earlier tokens: their step may only grow
        old = table[begun, [past[i] // case["page"] for i in begun]].long()
        e_old = torch.frexp(scales[old])[1] - 1
        e[old] = torch.maximum(e[old], e_old)
        again = _table(fmt, "cuda")[codes[old].int()] * _power(e_old - e[old])[:, :, None, None]
        codes[old] = _codes(again, fmt)
    touched = page.unique()
    scales[touched] = _power(e[touched])
    codes[page, :, place] = _codes(x * _power(-e)[page][:, :, None], fmt)


def _plain_read(case, codes, scales, table, counts, starts, dtype):
    page, place = _places(case, table, counts, starts)
    return (_table(case["format"], "cuda")[codes[page, :, place].int()] * scales[page][:, :, None]).to(dtype)


def _plain_attention(state):
    case, cache, q = state["case"], state["cache"], state["q"]
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows, past = state["host"]
    numbers, out, at = _table(case["format"], "cuda"), torch.empty_like(q), 0
    for i, (n, p) in enumerate(zip(rows, past)):
        low = max(0, p + 1 - case["window"]) // P if case["window"] else 0
        pages = state["table"][i, low:-(-(n + p) // P)].long()
        k, v = ((numbers[cache[c][pages].int()] * cache[s][pages][:, :, None, None]).transpose(0, 1).reshape(G, -1, D) for c, s in (("k", "ks"), ("v", "vs")))
        pos_k = torch.arange(low * P, low * P + k.shape[1], device="cuda")
        for r in torch.arange(n).split(max(1, (1 << 28) // (H * k.shape[1]))):
            qr = q[at + int(r[0]):at + int(r[-1]) + 1].float().view(len(r), G, H // G, D).permute(1, 2, 0, 3)
            s = (qr.reshape(G, -1, D) @ k.transpose(1, 2)).view(G, H // G, len(r), -1) * D ** -0.5
            pos_q = p + r.to("cuda")[:, None]
            hidden = pos_k > pos_q
            if case["window"]:
                hidden = hidden | (pos_k <= pos_q - case["window"])
            s.masked_fill_(hidden, -math.inf)
            most = s.amax(-1, keepdim=True)
            if state["sinks"] is not None:
                sink = state["sinks"].view(G, H // G, 1, 1)
                most = torch.maximum(most, sink)
            s = s.sub_(most).exp_()
            total = s.sum(-1, keepdim=True)
            if state["sinks"] is not None:
                total = total + (sink - most).exp()
            o = (s.view(G, -1, s.shape[-1]) @ v).view(G, H // G, len(r), D) / total
            out[at + int(r[0]):at + int(r[-1]) + 1] = o.permute(2, 0, 1, 3).reshape(len(r), H, D).to(q.dtype)
        at += n
    return out


@torch.no_grad()
def _plain(state):
    case, cache = state["case"], state["cache"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "attend":
        return _plain_attention(state)
    counts, starts = state["host"]
    if case["kind"] == "write":
        for c, s, x in (("k", "ks", "k"), ("v", "vs", "v")):
            _plain_append(case, cache[c], cache[s], state[x], state["table"], *state["host"])
        (counts, starts), dtype = state["back_host"], torch.float32
    return tuple(_plain_read(case, cache[c], cache[s], state["table"], counts, starts, dtype) for c, s in (("k", "ks"), ("v", "vs")))


# ---- a pass --------------------------------------------------------------------------------------------------------------

def run(state):
    if not own:
        return _plain(state)
    from dia_tts_prune_b200 import lm_ops
    case, cache = state["case"], state["cache"]
    if case["kind"] == "write":
        cache.append(state["k"], state["v"], state["table"], state["past"], state["first"])
        return cache.read(state["table"], state["back"], state["back_first"], state["back_total"])
    if case["kind"] == "read":
        return cache.read(state["table"], state["past"], state["first"], state["total"], DTYPES[case["dtype"]])
    return lm_ops.attention_kv8(state["q"], cache, state["table"], state["past"], state["first"], window=case["window"] or None, sinks=state["sinks"])


def work(case):
    s, G, D = BYTES[case["dtype"]], case["kv_heads"], case["dim"]
    rows, past, need = _case_sizes(case)
    if case["kind"] == "write":                                   # rows in, 8-bit numbers and what the changed pages stand for out
        back = sum(n + p % case["page"] for n, p in zip(rows, past))
        return {"bytes": 2 * G * D * (sum(rows) * (s + 1) + back * 4), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": 2 * G * D * sum(rows) * (1 + s) + 8 * G * sum(rows) / case["page"], "flops": 0}
    H = case["heads"]
    return {"bytes": _seen(case) * G * (2 * D + 8 / case["page"]) + 2 * sum(rows) * H * D * s, "flops": 4 * _pairs(case) * H * D}


# ---- the same from the definitions in 64 bits ----------------------------------------------------------------------------

def _two(e):
    """2^e in float64, for whole e (a power function may be a rounding off)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _number(codes, fmt):
    c = codes.to(torch.int64)
    if fmt == "int8":
        return (c - 256 * (c >= 128)).double()
    sign, field, fraction = 1 - 2 * (c >= 128).double(), (c % 128) // 8, (c % 8).double()
    normal = (1 + fraction / 8) * _two(field - 7)
    return sign * torch.where(field > 0, normal, fraction / 8 * 2.0 ** -6)


def _nearest(v, fmt):
    """v to the nearest number of the format (half way: the even one), in 64 bits."""
    if fmt == "int8":
        return torch.round(v)
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = _two(exponent - 3)
    return torch.round(v / step) * step


def _exact_pages(case, codes, scales, x, table, rows, past):
    """Values [kv_heads, tokens, dim] of the changed pages' tokens of every sequence, packed."""
    fmt, P, out, at = case["format"], case["page"], [], 0
    for i, (n, p) in enumerate(zip(rows, past)):
        begin = p // P
        pages = table[i, begin:-(-(n + p) // P)].long()
        held = p - begin * P
        old = _number(codes[pages[:1], :, :held], fmt)[0] * scales[pages[0]].double()[:, None, None]
        new = x[at:at + n].double().transpose(0, 1)
        tokens = torch.cat([old, new], 1)
        pad = torch.nn.functional.pad(tokens, (0, 0, 0, len(pages) * P - tokens.shape[1])).view(tokens.shape[0], len(pages), P, -1)
        fresh = pad.clone()
        fresh[:, 0, :held] = 0
        most = fresh.abs().amax((2, 3))
        # the smallest power of two that is enough
        unit = _two(torch.ceil(torch.log2((most / LARGEST[fmt]).clamp(min=2.0 ** LOWEST))))
        unit = torch.where(most > LARGEST[fmt] * unit, 2 * unit, torch.where((most <= LARGEST[fmt] * unit / 2) & (unit > 2.0 ** LOWEST), unit / 2, unit))
        if held:
            unit[:, 0] = torch.maximum(unit[:, 0], scales[pages[0]].double())
        got = _nearest(pad / unit[:, :, None, None], fmt) * unit[:, :, None, None]
        out.append(got.reshape(tokens.shape[0], len(pages) * P, -1)[:, :held + n])
        at += n
    return torch.cat(out, 1).transpose(0, 1).contiguous()


@torch.no_grad()
def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    cache, table, fmt, P = state["cache"], state["table"], case["format"], case["page"]
    rows, past = state["host"]
    if case["kind"] == "write":
        return tuple(_exact_pages(case, cache[c], cache[s], state[x], table, rows, past) for c, s, x in (("k", "ks", "k"), ("v", "vs", "v")))
    kinds = (("k", "ks"), ("v", "vs"))
    if case["kind"] == "read":
        got = [[], []]
        for i, (n, p) in enumerate(zip(rows, past)):
            pages = table[i, p // P:-(-(n + p) // P)].long()
            for j, (c, s) in enumerate(kinds):
                v = _number(cache[c][pages], fmt) * cache[s][pages].double()[:, :, None, None]
                got[j].append(v.transpose(1, 2).reshape(len(pages) * P, case["kv_heads"], -1)[p % P:p % P + n])
        return tuple(torch.cat(v) for v in got)
    H, D, share = case["heads"], case["dim"], case["heads"] // case["kv_heads"]
    out, at = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (n, p) in enumerate(zip(rows, past)):
        pages = table[i, :-(-(n + p) // P)].long()
        j = torch.arange(n + p, device="cuda")
        for head in range(case["kv_heads"]):
            k, v = ((_number(cache[c][pages, head], fmt) * cache[s][pages, head].double()[:, None, None]).reshape(-1, D)[:n + p] for c, s in kinds)
            for h in range(head * share, (head + 1) * share):
                for r in torch.arange(n, device="cuda").split(max(1, (1 << 26) // (n + p))):
                    z = state["q"][at + r, h].double() @ k.T / math.sqrt(D)
                    behind = (p + r)[:, None] - j
                    ok = behind >= 0
                    if case["window"]:
                        ok &= behind < case["window"]
                    z = torch.where(ok, z, -math.inf)
                    if state["sinks"] is not None:
                        z = torch.cat([z, state["sinks"][h].double().expand(len(r), 1)], 1)
                    out[at + r, h] = torch.softmax(z, -1)[:, :n + p] @ v
        at += n
    return out
