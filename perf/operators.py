"""What the operators for 4-bit weights and for scoring texts are measured on.

A language model's matrix is laid out in microscaled 4-bit numbers, its product gives logits or activations, and the loss of a
text under a head (and the loss's gradient) says what a change of the weights costs.

Kinds of a case
  quantize   rows in MXFP4 (blocks of 32 along a row share a power of two, elements are E2M1) and the values they stand for
  linear     the product of rows with a matrix that is kept in MXFP4; the rows are brought to MXFP4 on the way
  loss       every token's cross entropy under a head, the logits never in memory
  gradient   the mean of that loss over the tokens that count, and its gradients by the rows and by the head (a training step)

``rows`` are tokens (matrix rows for ``quantize``), ``width`` the model's width, ``out`` output channels or the vocabulary.
``dtype`` is the rows' type; heads and matrices are bfloat16 as everywhere in the framework, before they are laid out.
"""

from __future__ import annotations

import math

import torch

own = False

IGNORE = -100
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}


def listed():
    return [
        # a head of the benchmark's wider language model, laid out when the model is loaded
        dict(name="quantize_head", kind="quantize", rows=32768, width=2048, dtype="bfloat16"),
        # activations of an odd prompt portion whose width is no multiple of a block
        dict(name="quantize_odd", kind="quantize", rows=861, width=1000, dtype="float32"),
        # one decoded token through a square projection: latency
        dict(name="linear_token", kind="linear", rows=1, width=2048, out=2048, dtype="bfloat16"),
        # the head for eight running requests: the weights' bytes
        dict(name="linear_decode8_head", kind="linear", rows=8, width=2048, out=32768, dtype="float32"),
        # a prompt portion of odd length through an odd shape
        dict(name="linear_odd", kind="linear", rows=333, width=2000, out=1028, dtype="bfloat16"),
        # long prompts through a wide feed-forward
        dict(name="linear_prompt", kind="linear", rows=4096, width=4096, out=16384, dtype="bfloat16"),
        # one token scored (speculative checks, choice tasks): latency and the head's bytes
        dict(name="loss_token", kind="loss", rows=1, width=1024, out=16384, dtype="bfloat16", scale=1.0, ignored=0.0),
        # a text scored under a served model: float32 rows as the engine gives them, an odd vocabulary
        dict(name="loss_text", kind="loss", rows=700, width=2048, out=40007, dtype="float32", scale=0.25, ignored=0.0),
        # a long batch under a large vocabulary
        dict(name="loss_long", kind="loss", rows=4096, width=4096, out=131072, dtype="bfloat16", scale=1.0, ignored=0.1),
        # a training step on a short batch with padding
        dict(name="gradient_short", kind="gradient", rows=129, width=1000, out=16385, dtype="bfloat16", scale=1.0, ignored=0.3),
        # a training step of the benchmark's wider model
        dict(name="gradient_long", kind="gradient", rows=8192, width=2048, out=32768, dtype="bfloat16", scale=1.0, ignored=0.05),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _flops(case):
    per = 2.0 * case["rows"] * case["width"] * case.get("out", 1)
    return {"quantize": 0.0, "linear": per, "loss": per, "gradient": 3 * per}[case["kind"]]


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "loss", "gradient"])
    while True:
        case = dict(kind=kind, rows=_log_uniform(rng, 1, 8192 if kind == "gradient" else 4096), width=_log_uniform(rng, 32, 4096))
        if rng.random() < 0.5:                                    # widths of models are round, half of the time
            case["width"] = max(64, case["width"] // 64 * 64)
        if kind == "quantize":
            case.update(rows=_log_uniform(rng, 1, 32768), dtype=rng.choice(["bfloat16", "float16", "float32"]))
            if case["rows"] * case["width"] <= 32768 * 2048:
                return case
            continue
        case.update(out=_log_uniform(rng, 64, {"linear": 32768, "loss": 131072, "gradient": 65536}[kind]),
                    dtype=rng.choice(["bfloat16", "float32"]) if kind != "gradient" else "bfloat16")
        most = {"linear": 2.0 * 4096 * 4096 * 16384, "loss": 2.0 * 4096 * 4096 * 131072, "gradient": 6.0 * 8192 * 2048 * 32768}[kind]
        if kind in ("loss", "gradient"):
            case.update(scale=rng.choice([1.0, 0.25, 0.0625 * rng.randint(8, 24)]), ignored=rng.choice([0.0, 0.1, 0.5]))
        cost = _flops(case) * (3 if kind == "loss" and case["dtype"] == "float32" else 1)
        if cost <= most:
            return case


def _rows(g, case):
    """Rows behind a norm: about unit scale, a few channels much larger than the others, as trained models have them."""
    x = torch.randn(case["rows"], case["width"], generator=g, device="cuda")
    loud = torch.rand(case["width"], generator=g, device="cuda") < 0.02
    return x * torch.where(loud, 8.0, 1.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    if kind == "quantize":
        x = torch.randn(case["rows"], case["width"], generator=g, device="cuda") * 0.02
        x *= torch.exp(torch.randn(case["rows"], 1, generator=g, device="cuda"))
        if case["rows"] > 4:
            x[case["rows"] // 2].zero_()                          # a pruned row
        return dict(case=case, x=x.to(dtype))
    w = (torch.randn(case["out"], case["width"], generator=g, device="cuda") / math.sqrt(case["width"])).to(torch.bfloat16)
    x = _rows(g, case)
    if kind == "linear":
        if case["rows"] > 4:
            x[-1].zero_()                                         # a padding row
        state = dict(case=case, x=x.to(dtype))
        if own:
            from dia_tts_prune_b200 import lm_ops
            state["w"] = lm_ops.quantize_mxfp4(w)                 # what a program keeps of the matrix
        else:
            codes, exponents = _to_mxfp4(w)
            state["w"] = _values(codes, exponents, case["width"])
        return state
    t = torch.randint(0, case["out"], (case["rows"],), generator=g, device="cuda")
    # a model that has learnt something: rows lean towards their target, some of them far
    lean = 8.0 * torch.rand(case["rows"], 1, generator=g, device="cuda") ** 2
    x = x + lean * w[t].float() / case["scale"]
    t = torch.where(torch.rand(case["rows"], generator=g, device="cuda") < case["ignored"], IGNORE, t)
    x = x.to(dtype)
    if kind == "gradient":
        x, w = x.requires_grad_(True), w.requires_grad_(True)
    return dict(case=case, x=x, w=w, t=t)


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _power(e):
    """2^e in float32, for whole -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _to_mxfp4(x):
    """Codes 0 .. 15 (sign, then the index of the magnitude) and exponents (128 for a block that is not finite) of rows."""
    rows, width = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -width % 32)).view(rows, -1, 32)
    most = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(most)
    exponent = torch.frexp(most)[1] - 3                           # floor(log2(most)) - 2
    exponent = torch.where(most == 0, -127, exponent.clamp(-127, 125))
    half = torch.div(exponent, 2, rounding_mode="floor")
    scaled = x * _power(-half) * _power(half - exponent)          # times 2^-exponent, in two steps of normal numbers
    mag = scaled.abs()
    code = torch.zeros_like(mag, dtype=torch.uint8)
    # borders half way between two magnitudes go to the even code
    for border, above in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)):
        code += (mag > border) if above else (mag >= border)
    code += 8 * torch.signbit(scaled).to(torch.uint8)
    return torch.where(bad, 0, code), torch.where(bad, 128, exponent)


def _values(code, exponent, width):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
    v = table[(code & 7).long()]
    v = torch.where(code >= 8, -v, v)
    half = torch.div(exponent, 2, rounding_mode="floor")
    v = v * _power(half) * _power(exponent - half)
    v = torch.where(exponent == 128, math.nan, v)
    return v.reshape(v.shape[0], -1)[:, :width].contiguous()


def _plain_loss(x, w, t, scale):
    """Losses of the tokens and what their gradients need: float32 logits in place of probabilities, rows that count."""
    z = (x.float() @ w.float().T).mul_(scale)
    counts = t != IGNORE
    at = torch.where(counts, t, 0)[:, None]
    most = z.amax(-1, keepdim=True)
    hit = z.gather(1, at) - most
    p = z.sub_(most).exp_()
    total = p.sum(-1, keepdim=True)
    loss = torch.where(counts, (total.log() - hit)[:, 0], 0.0)
    return loss, p, total, counts, at


@torch.no_grad()
def _plain(state):
    case = state["case"]
    if case["kind"] == "quantize":
        return _values(*_to_mxfp4(state["x"]), case["width"])
    if case["kind"] == "linear":
        a = _values(*_to_mxfp4(state["x"]), case["width"])
        return (a @ state["w"].T).to(state["x"].dtype)
    x, w = state["x"], state["w"]
    loss, p, total, counts, at = _plain_loss(x, w, state["t"], case["scale"])
    if case["kind"] == "loss":
        return loss
    n = counts.sum().clamp(min=1)
    p.div_(total)
    p.scatter_add_(1, at, torch.full_like(p[:, :1], -1.0))
    p.mul_((counts.float() * case["scale"] / n)[:, None])
    dx, dw = p @ w.float(), p.T @ x.float()
    return loss.sum() / n, dx.to(x.dtype), dw.to(w.dtype)


# ---- a pass --------------------------------------------------------------------------------------------------------------

def run(state):
    if not own:
        return _plain(state)
    from dia_tts_prune_b200 import lm_ops
    case = state["case"]
    if case["kind"] == "quantize":
        return lm_ops.quantize_mxfp4(state["x"]).dequantize()
    if case["kind"] == "linear":
        return lm_ops.linear_mxfp4(state["x"], state["w"])
    if case["kind"] == "loss":
        return lm_ops.linear_cross_entropy(state["x"], state["w"], state["t"], scale=case["scale"], reduction="none")
    loss = lm_ops.linear_cross_entropy(state["x"], state["w"], state["t"], scale=case["scale"], reduction="mean")
    dx, dw = torch.autograd.grad(loss, (state["x"], state["w"]))
    return loss.detach(), dx, dw


def work(case):
    M, K, s = case["rows"], case["width"], BYTES[case["dtype"]]
    if case["kind"] == "quantize":                                # rows in, 4-bit numbers and float32 values out
        return {"bytes": M * K * (s + 4.25 / 8 + 4), "flops": 0}
    N = case["out"]
    if case["kind"] == "linear":
        return {"bytes": M * K * s + N * K * 4.25 / 8 + M * N * s, "flops": 2 * M * N * K}
    if case["kind"] == "loss":
        return {"bytes": M * K * s + N * K * 2 + M * 12, "flops": 2 * M * N * K}
    return {"bytes": 2 * M * K * s + 2 * N * K * 2 + M * 8 + 4, "flops": 6 * M * N * K}


# ---- the same from the definitions in 64 bits ----------------------------------------------------------------------------

def _exact_mxfp4(x):
    rows, width = x.shape
    out = torch.zeros(rows, -(-width // 32) * 32, dtype=torch.float64, device=x.device)
    out[:, :width] = x.double()
    blocks = out.view(rows, -1, 32)
    most = blocks.abs().amax(-1, keepdim=True)
    # floor(log2(most)) - 2 out of the number itself: float32 numbers are normal in float64, whose exponent stands in bits 52 ..
    shared = (most.clamp(min=2.0 ** -149).view(torch.int64) >> 52) - 1023 - 2
    unit = ((shared.clamp(-127, 125) + 1023) << 52).view(torch.float64)
    magnitudes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    r = blocks.abs() / unit
    lower = torch.searchsorted(magnitudes, r.clamp(max=6), right=True) - 1
    upper = (lower + 1).clamp(max=7)
    to_lower, to_upper = r - magnitudes[lower], magnitudes[upper] - r
    up = (to_upper < to_lower) | ((to_upper == to_lower) & (lower % 2 == 1))
    v = torch.where(up, magnitudes[upper], magnitudes[lower]) * unit * torch.sign(blocks)
    v = torch.where(torch.isfinite(most), v, math.nan)
    return v.reshape(rows, -1)[:, :width]


@torch.no_grad()
def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    x = state["x"].detach()
    if case["kind"] == "quantize":
        return _exact_mxfp4(x)
    if case["kind"] == "linear":
        return _exact_mxfp4(x) @ state["w"].double().T
    w, t = state["w"].detach().double(), state["t"]
    keep = t != IGNORE
    n = max(int(keep.sum()), 1)
    losses = torch.zeros(case["rows"], dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(w) if case["kind"] == "gradient" else None
    for r in torch.arange(case["rows"], device=x.device).split(1024):
        h = x[r].double()
        logp = torch.log_softmax(case["scale"] * (h @ w.T), -1)
        target = torch.where(keep[r], t[r], 0)
        losses[r] = -logp[torch.arange(len(r), device=x.device), target] * keep[r]
        if dw is not None:
            p = logp.exp()
            p[torch.arange(len(r), device=x.device), target] -= 1
            p *= (keep[r].double() * case["scale"] / n)[:, None]
            dx[r] = p @ w
            dw += p.T @ h
    return losses if dw is None else (losses.sum() / n, dx, dw)
