"""Scoring texts under served models, heads in 4 bits, and the operators one behind the other: captured, on other streams, twice at once."""

import json
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def model(design="pubopel", dtype="float32", **kw):
    from dia_tts_prune_b200 import lm_config as CFG
    from dia_tts_prune_b200 import synthetic as SY
    from dia_tts_prune_b200.lm_model import CausalLM
    if design == "pubopel":
        cfg = SY.pubopel_config(width=96, layers=2, heads=4, kv_heads=2, dim=24, experts=4, top=2, expert_ff=40, shared_ff=56, vocab=301, window=20, keep_first=3)
        w, c = SY.pubopel_weights(cfg, 3), CFG.PubopelConfig.model_validate(cfg)
    elif design == "fipadra":
        cfg = SY.fipadra_config(width=64, kinds=["delta", "retention"], heads=4, dim=16, vdim=16, vocab=301, ff=96, logit_scale=0.5)
        w, c = SY.fipadra_weights(cfg, 3), CFG.FipadraConfig.model_validate(cfg)
    else:
        cfg = SY.kupelix_config(width=64, kinds=["attention", "hgrn2"], heads=4, kv_heads=2, dim=16, vdim=16, vocab=301, ff=96)
        w, c = SY.kupelix_weights(cfg, 3), CFG.KupelixConfig.model_validate(cfg)
    return CausalLM(c, w, dtype=dtype, device="cuda:0", **{**dict(max_tokens=256, max_sequences=3, page_size=8, max_rows=64), **kw})


def texts(lengths, seed=0, vocab=301):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def rows_of(m, sequences):
    """Per sequence the rows in front of the head, as the engine gives them."""
    out = []
    for s in sequences:
        seq = m.state.open("x")
        out.append(m.engine.step([(seq, s[:-1], list(range(len(s) - 1)))], hidden=True))
        m.state.close("x")
    return out


def expected(hidden, head, sequence):
    """log-probabilities in 64 bits and how far off float32 sums of exact products may be: a loss moves by twice a logit (2^-22 of the
    magnitudes at each of K / 16 steps of three terms, see the losses' own tests) and by 2^-18 for exponentials and logarithms."""
    h, w, t = hidden.double().cpu(), head.double().cpu(), torch.tensor(sequence[1:])
    logp = torch.log_softmax(h @ w.T, 1).gather(1, t[:, None])[:, 0]
    return logp, 2 * (3 * h.shape[1] / 16 + 6) * 2.0 ** -22 * (h.abs() @ w.abs().T).amax(1) + 2.0 ** -18


@pytest.mark.parametrize("design", ["pubopel", "kupelix", "fipadra"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_of_served_models(design, dtype):
    m = model(design, dtype)
    sequences = texts((40, 2, 150, 1, 3, 0, 64, 90))              # more than there are slots, longer than a step, nothing to score
    got = m.score(sequences)
    assert [len(g) for g in got] == [39, 1, 149, 0, 2, 0, 63, 89]
    assert m.state.free_slots == 3 and m.state.free_pages == m.state.n_pages and not m.state.sequences
    head = m.engine.head
    for s, g in zip(sequences, got):
        if len(s) < 2:
            continue
        hidden, = rows_of(m, [s])
        # a sequence of its own and the same one beside others go through kernels for other numbers of rows: hidden differs by their roundings,
        # which float32 rows show as 2^-12 of the largest logit at most; bfloat16 products by the steps of bfloat16
        want, off = expected(hidden if dtype == "float32" else hidden.bfloat16(), head, s)
        slack = (2.0 ** -12 if dtype == "float32" else 2.0 ** -4) * (hidden.double().cpu() @ head.double().cpu().T).abs().amax(1)
        assert ((torch.tensor(g, dtype=torch.float64) - want).abs() <= off + slack).all()
        assert all(x <= 0 for x in g)


@pytest.mark.parametrize("design", ["pubopel", "kupelix", "fipadra"])
def test_hidden_rows_are_what_the_head_multiplies(design):
    m = model(design)
    for n in (1, 2, 40, 64):
        s = texts((n,), seed=n)[0]
        a, b = m.state.open("a"), m.state.open("b")
        want = sorted({0, n // 2, n - 1})
        logits = m.engine.step([(a, s, want)])
        hidden = m.engine.step([(b, s, want)], hidden=True)
        assert hidden.shape == (len(want), m.engine.width)
        ref = hidden.double() @ m.engine.head.double().T
        # (the rows of the two steps may come from a captured and an uncaptured pass of the same kernels; logits are float32 sums)
        assert ((logits.double() - ref).abs() <= 2.0 ** -16 * (hidden.double().abs() @ m.engine.head.double().abs().T)).all()
        m.state.close("a"), m.state.close("b")
    with pytest.raises(ValueError):
        m.engine.step([], keep_layers=True, hidden=True)


def test_scores_refuse_and_leave_nothing():
    from dia_tts_prune_b200.lm_state import OutOfPages
    m = model()
    for bad in ([1, 301], [-1, 2]):
        with pytest.raises(ValueError):
            m.score([[1, 2, 3], bad])
    with pytest.raises(OutOfPages):
        m.score(texts((300,)))
    assert m.state.free_slots == 3 and m.state.free_pages == m.state.n_pages and not m.state.sequences
    assert m.score([]) == []


@pytest.mark.parametrize("design", ["pubopel", "fipadra"])
def test_heads_in_4_bits(design):
    """Logits are the product of the rounded rows and the rounded head (exact products, float32 sums); scores are their log-softmax; decoding
    picks the largest; and the whole head's bytes shrink by 3.76."""
    from dia_tts_prune_b200 import lm_ops
    m, plain = model(design, head_format="mxfp4"), model(design)
    head = m.engine.head.dequantize()
    assert torch.equal(head, lm_ops.quantize_mxfp4(plain.engine.head).dequantize())
    for n, wants in ((1, [0]), (40, [39]), (64, list(range(64)))):
        s = texts((n,), seed=n)[0]
        a = m.state.open("a")
        logits = m.engine.step([(a, s, wants)])
        m.state.close("a")
        a = m.state.open("a")
        hidden = m.engine.step([(a, s, wants)], hidden=True)
        m.state.close("a")
        rows = lm_ops.quantize_mxfp4(hidden).dequantize()
        ref, most = rows.double() @ head.double().T, rows.double().abs() @ head.double().abs().T
        # one step of 4 bits where the two passes' rows round to neighbours: a row may differ in a few elements by half its block's largest
        close = (logits.double() - ref).abs() <= (hidden.shape[1] / 64 + 2) * 2.0 ** -22 * most
        assert close.float().mean() > 0.9 and ((logits.double() - ref).abs() <= 0.25 * most).all()
    got = m.score(texts((50, 33)))
    for s, g in zip(texts((50, 33)), got):
        hidden, = rows_of(m, [s])
        want, off = expected(lm_ops.quantize_mxfp4(hidden).dequantize(), head, s)
        assert ((torch.tensor(g, dtype=torch.float64) - want).abs() <= off + 0.25).all()
    out = m.generate(texts((5, 9)), max_new_tokens=6)
    assert [len(o) for o in out] == [6, 6] and all(0 <= t < 301 for o in out for t in o)
    assert m.generate(texts((5, 9)), max_new_tokens=6) == out


def test_score_command(tmp_path, capsys):
    from dia_tts_prune_b200 import synthetic as SY
    from dia_tts_prune_b200.__main__ import main
    from dia_tts_prune_b200.checkpoint import save_safetensors
    cfg = SY.pubopel_config(width=64, layers=1, heads=2, kv_heads=1, dim=32, experts=2, top=1, expert_ff=16, shared_ff=None, vocab=50)
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    save_safetensors(tmp_path / "model.safetensors", SY.pubopel_weights(cfg, 1))
    for fmt in ("bfloat16", "mxfp4"):
        assert main(["score", "--model", str(tmp_path), "--tokens", "1 2 3 4", "--tokens", "7", "--head-format", fmt]) == 0
        a, b = (json.loads(line) for line in capsys.readouterr().out.strip().splitlines())
        assert a["tokens"] == 3 == len(a["logprobs"]) and abs(math.exp(-a["logprob"] / 3) - a["perplexity"]) < 1e-6
        assert b == {"tokens": 0, "logprob": 0.0, "perplexity": None, "logprobs": []}


# ---- the operators one behind the other ------------------------------------------------------------------------------------------------

def chain(x, w4, head, t):
    """A matrix in 4 bits, then the head's loss and both gradients."""
    from dia_tts_prune_b200 import lm_ops
    y = lm_ops.linear_mxfp4(x, w4).requires_grad_(True)
    head = head.detach().requires_grad_(True)
    loss = lm_ops.linear_cross_entropy(y, head, t)
    return (loss.detach(), *torch.autograd.grad(loss, (y, head)), lm_ops.linear_cross_entropy(y.detach()[:5].float(), head.detach(), t[:5], reduction="none"),
            lm_ops.linear_mxfp4(x[:3], w4))


def inputs(m, seed):
    from dia_tts_prune_b200 import lm_ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, 192, generator=g, device="cuda").bfloat16()
    w4 = lm_ops.quantize_mxfp4(torch.randn(256, 192, generator=g, device="cuda") / 14)
    head = (torch.randn(1111, 256, generator=g, device="cuda") / 16).bfloat16()
    return x, w4, head, torch.randint(0, 1111, (m,), generator=g, device="cuda")


def test_the_chain_is_reproducible_and_captured():
    """The same bits every time, from a captured graph too, whose inputs may change between replays; two graphs share nothing."""
    a, b = inputs(300, 1), inputs(300, 2)
    want = [chain(*i) for i in (a, b)]
    for i, w in ((a, want[0]), (b, want[1])):
        assert all(torch.equal(u, v) for u, v in zip(chain(*i), w))
    graphs = []
    for i in (a, b):
        x, w4, head, t = i[0].clone(), i[1], i[2].clone(), i[3].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                chain(x, w4, head, t)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(x, w4, head, t)
        graphs.append((g, out, x, head, t))
    for _ in range(3):
        for g, *_ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (g, out, *_), w in zip(graphs, want):
        assert all(torch.equal(u, v) for u, v in zip(out, w))
    g, out, x, head, t = graphs[0]
    x.copy_(b[0]), t.copy_(b[3])
    g.replay()
    for u, v in zip(out, chain(b[0], a[1], a[2], b[3])):
        assert torch.equal(u, v)


def test_two_streams_at_once():
    a, b = inputs(150, 3), inputs(170, 4)
    want = [chain(*i) for i in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for k, i in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                got[k].append(chain(*i))
    torch.cuda.synchronize()
    for k in (0, 1):
        for out in got[k]:
            assert all(torch.equal(u, v) for u, v in zip(out, want[k]))


def test_a_matrix_laid_out_right_before_its_product():
    """Products ask for their weights before their predecessor has ended: not before one that writes them has."""
    from dia_tts_prune_b200 import lm_ops
    g = torch.Generator(device="cuda").manual_seed(5)
    ws = [torch.randn(4096, 1024, generator=g, device="cuda") for _ in range(3)]
    for m in (1, 40):
        x = torch.randn(m, 1024, generator=g, device="cuda").bfloat16()
        want = []
        for w in ws:
            q = lm_ops.quantize_mxfp4(w)
            torch.cuda.synchronize()
            want.append(lm_ops.linear_mxfp4(x, q))
        torch.cuda.synchronize()
        for _ in range(5):
            got = []
            for w in ws:
                lm_ops.linear_mxfp4(x, q)
                q = lm_ops.quantize_mxfp4(w)                       # (its memory is an earlier one's)
                got.append(lm_ops.linear_mxfp4(x, q))
            assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_results_do_not_alias_what_the_gradient_needs():
    """A loss changed in place before its backward pass; hidden changed in place is noticed."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    x, _, head, t = inputs(64, 6)
    h = torch.randn(64, 256, device="cuda").bfloat16().requires_grad_(True)
    head.requires_grad_(True)
    want = torch.autograd.grad(linear_cross_entropy(h, head, t) * 0.5, (h, head))
    loss = linear_cross_entropy(h, head, t)
    loss *= 0.5
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(loss, (h, head)), want))
    each = linear_cross_entropy(h, head, t, reduction="none")
    each.mul_(0.0)
    assert not torch.autograd.grad(each.sum(), h)[0].any()
    k = h.detach().clone().requires_grad_(True)
    loss = linear_cross_entropy(k, head, t)
    with torch.no_grad():
        k.add_(1)
    with pytest.raises(RuntimeError, match="in-?place"):
        loss.backward()
    loss = linear_cross_entropy(h, head, t)
    loss.backward(retain_graph=True)
    once = h.grad.clone()
    loss.backward()
    assert torch.equal(h.grad, once * 2) and h.grad.dtype == head.grad.dtype == torch.bfloat16


def test_a_wait_that_ran_out_shows():
    """With no looks at any barrier every wait ends at once: results are NaN, the next call reports it, the one behind is whole again."""
    import ctypes as C

    from dia_tts_prune_b200 import _lm_lib, lm_ops
    x, w4, head, t = inputs(300, 7)
    polls = getattr(_lm_lib.load(), "_ZN3dia15gemm_pair_pollsEv")
    polls.restype = C.POINTER(C.c_uint)
    y = lm_ops.linear_mxfp4(x, w4)
    calls = [lambda: lm_ops.linear_mxfp4(x, w4), lambda: lm_ops.linear_mxfp4(x[:2], w4), lambda: lm_ops.linear_cross_entropy(y, head, t, reduction="none"),
             lambda: lm_ops.linear_cross_entropy(y[:2], head, t[:2], reduction="none")]
    leaf = y.clone().requires_grad_(True)
    loss = lm_ops.linear_cross_entropy(leaf, head, t)
    kept = polls()[0]
    for call in calls:
        want = call()
        polls()[0] = 0
        try:
            got = call()
        finally:
            polls()[0] = kept
        torch.cuda.synchronize()
        assert got.isnan().all()
        with pytest.raises(RuntimeError):
            call()
        assert torch.equal(call(), want)
    torch.autograd.grad(loss, leaf, retain_graph=True)


def test_a_head_that_the_kernel_in_front_writes():
    """Kernels start before their predecessor has ended; what it writes may be the head of the next loss (a product's result, a gradient)."""
    from dia_tts_prune_b200 import lm_ops
    g = torch.Generator(device="cuda").manual_seed(8)
    w4 = lm_ops.quantize_mxfp4(torch.randn(4096, 512, generator=g, device="cuda") / 22)
    xs = [torch.randn(12, 512, generator=g, device="cuda").bfloat16() for _ in range(3)]
    h, t = torch.randn(3, 4096, generator=g, device="cuda").bfloat16(), torch.tensor([0, 5, 11], device="cuda")
    want = []
    for x in xs:
        y = lm_ops.linear_mxfp4(x, w4)
        torch.cuda.synchronize()
        want.append(lm_ops.linear_cross_entropy(h, y, t, reduction="none"))
    torch.cuda.synchronize()
    for _ in range(10):
        got = [lm_ops.linear_cross_entropy(h, lm_ops.linear_mxfp4(x, w4), t, reduction="none") for x in xs]
        assert all(torch.equal(u, v) for u, v in zip(got, want))
    rows = torch.randn(200, 512, generator=g, device="cuda").bfloat16()
    head = (torch.randn(3000, 512, generator=g, device="cuda") / 22).bfloat16().requires_grad_(True)
    targets = torch.randint(0, 3000, (200,), generator=g, device="cuda")

    def loss_under_a_gradient(wait):
        dw, = torch.autograd.grad(lm_ops.linear_cross_entropy(rows, head, targets), head)
        if wait:
            torch.cuda.synchronize()
        return lm_ops.linear_cross_entropy(rows[:3] * 100, dw, targets[:3], reduction="none")

    want = loss_under_a_gradient(True)
    for _ in range(10):
        assert torch.equal(loss_under_a_gradient(False), want)


@pytest.mark.parametrize("m,n,k", [(300, 512, 2000), (2048, 16384, 1024), (2100, 12290, 72), (3, 4096, 8192), (1, 130, 40)])
def test_products_whose_waits_ran_out_leave_in_order(m, n, k):
    """No looks at any barrier, with copies on their way that are asked for ahead of the first wait: tiles of one SM, of pairs, few rows.  Results
    are NaN, the next call reports it, and what runs on the SMs behind it is whole."""
    import ctypes as C

    from dia_tts_prune_b200 import _lm_lib, lm_ops
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w4 = torch.randn(m, k, generator=g, device="cuda").bfloat16(), lm_ops.quantize_mxfp4(torch.randn(n, k, generator=g, device="cuda"))
    polls = getattr(_lm_lib.load(), "_ZN3dia15gemm_pair_pollsEv")
    polls.restype = C.POINTER(C.c_uint)
    want, kept = lm_ops.linear_mxfp4(x, w4), polls()[0]
    polls()[0] = 0
    try:
        got = lm_ops.linear_mxfp4(x, w4)
    finally:
        polls()[0] = kept
    behind = want.float() * 2                                      # (another kernel on the SMs that were given up)
    torch.cuda.synchronize()
    assert got.isnan().all() and torch.equal(behind, want.float() + want.float())
    with pytest.raises(RuntimeError):
        lm_ops.linear_mxfp4(x, w4)
    for _ in range(3):
        assert torch.equal(lm_ops.linear_mxfp4(x, w4), want)


def test_gradients_whose_waits_ran_out_leave_in_order():
    import ctypes as C

    from dia_tts_prune_b200 import _lm_lib, lm_ops
    g = torch.Generator(device="cuda").manual_seed(3)
    h, w = torch.randn(300, 512, generator=g, device="cuda").bfloat16().requires_grad_(True), (torch.randn(3000, 512, generator=g, device="cuda") / 22).bfloat16().requires_grad_(True)
    t = torch.randint(0, 3000, (300,), generator=g, device="cuda")
    polls = getattr(_lm_lib.load(), "_ZN3dia15gemm_pair_pollsEv")
    polls.restype = C.POINTER(C.c_uint)
    out = torch.empty(1, device="cuda")
    for rows in (300, 100):                                        # (pairs of SMs, one SM per tile)
        loss = lm_ops.linear_cross_entropy(h[:rows], w, t[:rows])
        want = torch.autograd.grad(loss, (h, w), retain_graph=True)
        # the launches go by the limit of the thread that makes them: the C entry, from this one
        lib, st = _lm_lib.load(), torch.cuda.current_stream().cuda_stream
        kept = torch.empty(2 * rows + 1, device="cuda")
        need = lib.lm_b200_op_loss_work_bytes(h.data_ptr(), 1, 512, w.data_ptr(), 512, rows, 3000, 512)
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        assert lib.lm_b200_op_loss(h.data_ptr(), 1, 512, w.data_ptr(), 512, t.data_ptr(), 1, -100, rows, 3000, 512, 1.0, 2, out.data_ptr(), kept.data_ptr(), work.data_ptr(), need, st) == 0
        need = lib.lm_b200_op_loss_grad_work_bytes(h.data_ptr(), 512, w.data_ptr(), 512, rows, 3000, 512, 1, 1)
        work, one = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.ones((), device="cuda")
        dh, dw = torch.zeros_like(h[:rows]), torch.zeros_like(w)

        def backward():
            return lib.lm_b200_op_loss_grad(h.data_ptr(), 512, w.data_ptr(), 512, t.data_ptr(), 1, -100, rows, 3000, 512, 1.0, kept.data_ptr(), one.data_ptr(), 0,
                                            kept.data_ptr() + 8 * rows, dh.data_ptr(), dw.data_ptr(), work.data_ptr(), need, st)

        torch.cuda.synchronize()
        limit = polls()[0]
        polls()[0] = 0
        try:
            assert backward() == 0
        finally:
            polls()[0] = limit
        torch.cuda.synchronize()
        assert dh.isnan().all() and dw.isnan().all()
        assert backward() != 0                                     # (says that a wait ran out)
        assert backward() == 0
        assert torch.equal(dh, want[0][:rows]) and torch.equal(dw, want[1])


def test_weights_that_the_kernel_in_front_writes():
    """``lm_engine.linear`` takes bfloat16 weights where they are: a 4-bit product's result, the gradient of a loss by its head alone, whose kernels
    let their successor start before they have written it."""
    from dia_tts_prune_b200 import lm_engine, lm_ops
    g = torch.Generator(device="cuda").manual_seed(12)
    w4 = lm_ops.quantize_mxfp4(torch.randn(2048, 512, generator=g, device="cuda") / 22)
    xs = [torch.randn(16, 512, generator=g, device="cuda").bfloat16() for _ in range(4)]
    a, wide = torch.randn(2, 2048, generator=g, device="cuda"), torch.randn(3000, 2048, generator=g, device="cuda")   # (a few rows; many rows and few outputs)
    rows = torch.randn(200, 512, generator=g, device="cuda").bfloat16()
    heads = [(torch.randn(3000, 512, generator=g, device="cuda") / 22).bfloat16().requires_grad_(True) for _ in range(3)]
    targets, b = torch.randint(0, 3000, (200,), generator=g, device="cuda"), torch.randn(2, 512, generator=g, device="cuda")

    def product(x, act, wait):
        y = lm_ops.linear_mxfp4(x, w4)
        if wait:
            torch.cuda.synchronize()
        return lm_engine.linear(act, y)

    def gradient(head, wait):
        dw, = torch.autograd.grad(lm_ops.linear_cross_entropy(rows, head, targets), head)
        if wait:
            torch.cuda.synchronize()
        return lm_engine.linear(b, dw)

    for act in (a, wide):
        want = [product(x, act, True) for x in xs]
        torch.cuda.synchronize()
        for _ in range(20):
            assert all(torch.equal(u, v) for u, v in zip([product(x, act, False) for x in xs], want))
    want = [gradient(h, True) for h in heads]
    torch.cuda.synchronize()
    for _ in range(20):
        assert all(torch.equal(u, v) for u, v in zip([gradient(h, False) for h in heads], want))


def test_rows_that_the_kernel_in_front_writes():
    """Products of few rows, losses and gradients read what the kernel in front has just written, over and over in the same memory."""
    from dia_tts_prune_b200 import lm_ops
    g = torch.Generator(device="cuda").manual_seed(14)
    ws = [lm_ops.quantize_mxfp4(torch.randn(1024, 1024, generator=g, device="cuda") / 32) for _ in range(6)]
    head, t = (torch.randn(2000, 1024, generator=g, device="cuda") / 32).bfloat16(), torch.randint(0, 2000, (16,), generator=g, device="cuda")
    xs = [torch.randn(16, 1024, generator=g, device="cuda").to(d) for d in (torch.bfloat16, torch.float32) for _ in range(3)]

    def through(x, wait):
        for w in ws:
            x = lm_ops.linear_mxfp4(x, w)
            if wait:
                torch.cuda.synchronize()
        losses = lm_ops.linear_cross_entropy(x, head, t, reduction="none")
        if x.dtype == torch.float32:
            return x, losses
        a = x.detach().requires_grad_(True)
        return x, losses, torch.autograd.grad(lm_ops.linear_cross_entropy(a, head, t), a)[0]

    want = [through(x, True) for x in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, ref in zip(xs, want):
            assert all(torch.equal(u, v) for u, v in zip(through(x, False), ref))


def exact_logprobs(hidden, engine, targets):
    """log-probabilities in 64 bits of the rows as the engine multiplies them (as they are, in bfloat16, in 4 bits), and the losses' own bound (see
    test_loss_gpu.py): sums of 16 products lose 2^-22 of the magnitudes a step, exponentials and logarithms 2^-20."""
    from dia_tts_prune_b200 import lm_ops
    head, terms = engine.head, 1
    if isinstance(head, lm_ops.Mxfp4):
        rows, head = lm_ops.quantize_mxfp4(hidden).dequantize(), head.dequantize()
    elif engine.precision == "float32":
        rows, terms = hidden, 3
    else:
        rows = hidden.bfloat16()
    h, w, t = rows.double().cpu(), head.double().cpu(), targets.cpu().long()
    z = h @ w.T
    loss = -torch.log_softmax(z, 1).gather(1, t[:, None])[:, 0]
    dz = (h.shape[1] / 16 + 2) * terms * 2.0 ** -22 * (h.abs() @ w.abs().T).amax(1)
    return -loss, 2 * dz + 2.0 ** -20 + 2.0 ** -22 * (z.abs().amax(1) + loss)


@pytest.mark.parametrize("design", ["pubopel", "kupelix", "fipadra"])
@pytest.mark.parametrize("dtype,head_format", [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float32", "mxfp4"), ("bfloat16", "mxfp4")])
def test_scores_are_the_losses_of_the_rows_that_were_scored(design, dtype, head_format, monkeypatch):
    """The scores against the rows and targets of the same step, at the losses' own bound; every row's target is the token behind it."""
    m = model(design, dtype, head_format=head_format)
    sequences, seen, plain = texts((40, 2, 150, 1, 3, 0, 64, 90), seed=5), [], m.engine.token_losses

    def record(hidden, targets):
        seen.append((hidden.clone(), targets.clone()))
        return plain(hidden, targets)

    monkeypatch.setattr(m.engine, "token_losses", record)
    got = m.score(sequences)
    assert len(seen) > 1
    hidden, targets = torch.cat([h for h, _ in seen]), torch.cat([t for _, t in seen])
    assert targets.tolist() == [t for s in sequences for t in s[1:]]
    want, off = exact_logprobs(hidden, m.engine, targets)
    assert ((torch.tensor([x for g in got for x in g], dtype=torch.float64) - want).abs() <= off).all()
    # rows in their order: the same texts one at a time go through kernels for other numbers of rows, whose bfloat16 products differ by some 2^-8
    # of a row; other rows are far away
    alone = torch.cat([h for s in sequences if len(s) > 1 for h in rows_of(m, [s])]).double()
    near = torch.cdist(alone, hidden.double())
    same = torch.tensor([[a == b for b in targets.tolist()] for a in targets.tolist()])
    assert (near.diagonal() <= 0.1 * alone.norm(dim=1)).all()
    apart = near.cpu() + torch.where(same, 1e9, 0.0)
    assert (apart.amin(1) > near.diagonal().cpu()).float().mean() > 0.99


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("design", ["pubopel", "kupelix", "fipadra"])
def test_logits_of_a_head_in_4_bits_are_its_product(design, dtype):
    """Every logit of a step against the product of the same rows with the same head in 64 bits, at the product's own bound (64 exact products
    at a time, 2^-22 of the magnitudes a step, see test_mxfp4_gpu.py); and the product called by itself has the step's bits."""
    from dia_tts_prune_b200 import lm_ops
    m = model(design, dtype, head_format="mxfp4", step_graphs=False)
    head = m.engine.head.dequantize().double()
    for n, wants in ((1, [0]), (40, [39]), (40, [3, 17]), (64, list(range(64)))):
        s, out = texts((n,), seed=n)[0], []
        for hidden in (False, True):
            a = m.state.open("a")
            out.append(m.engine.step([(a, s, wants)], hidden=hidden))
            m.state.close("a")
        logits, hidden = out
        rows = lm_ops.quantize_mxfp4(hidden).dequantize().double()
        bound = (hidden.shape[1] / 64 + 2) * 2.0 ** -22 * (rows.abs() @ head.abs().T) + 2.0 ** -24 * (rows @ head.T).abs()
        assert ((logits.double() - rows @ head.T).abs() <= bound).all()
        assert torch.equal(logits, lm_ops.linear_mxfp4(hidden, m.engine.head))


@pytest.mark.parametrize("design", ["pubopel", "kupelix", "fipadra"])
def test_captured_steps_of_a_head_in_4_bits(design):
    """Steps of a few rows are captured with the head's product inside: the bits of steps that are not, as the sequences go on."""
    a, b = (model(design, "bfloat16", head_format="mxfp4", step_graphs=g) for g in (True, False))
    prompts = texts((5, 9, 2), seed=8)
    open_ = [[m.state.open(f"s{i}") for i in range(3)] for m in (a, b)]
    for _ in range(2):                                             # (captured once, replayed afterwards)
        for k in (1, 2, 3):
            out = [m.engine.step([(seq, p, [len(p) - 1]) for seq, p in zip(seqs[:k], prompts)]) for m, seqs in zip((a, b), open_)]
            assert torch.equal(*out)
            for _ in range(3):
                tokens = out[0].argmax(1).tolist()
                out = [m.engine.step([(seq, [t], [0]) for seq, t in zip(seqs[:k], tokens)]) for m, seqs in zip((a, b), open_)]
                assert torch.equal(*out)


def test_a_thread_that_has_not_used_the_device():
    """Its first call is an operator's, with memory that torch has at hand."""
    import threading

    from dia_tts_prune_b200 import lm_ops
    x, w4, head, t = inputs(300, 9)
    y = lm_ops.linear_mxfp4(x, w4)
    calls = [lambda: lm_ops.linear_mxfp4(x[:2], w4), lambda: lm_ops.linear_mxfp4(x, w4), lambda: lm_ops.linear_cross_entropy(y, head, t, reduction="none"),
             lambda: lm_ops.linear_cross_entropy(y[:3], head, t[:3], reduction="none"), lambda: lm_ops.quantize_mxfp4(y).dequantize()]
    for call in calls:
        call()                                                     # (its workspace is at hand afterwards)
        want, got = call(), []
        thread = threading.Thread(target=lambda: got.append(call()))
        thread.start()
        thread.join()
        assert torch.equal(got[0], want)


def test_the_first_backward_pass_of_a_program():
    """By the rows alone: its thread has not used the device, and nothing else is launched in front.  (P and the result are rounded to bfloat16, 2^-8
    each, and what the gradient sums are a target's row and a mean of many: next to no cancellation.)"""
    import subprocess
    import sys
    program = """
import torch
from dia_tts_prune_b200.lm_ops import linear_cross_entropy
h = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_(True)
w, t = torch.randn(300, 64, device="cuda").bfloat16(), torch.arange(40, device="cuda")
linear_cross_entropy(h, w, t).backward()
p = torch.softmax(h.detach().double() @ w.double().T, 1)
p[torch.arange(40), t] -= 1
want = p @ w.double() / 40
assert ((h.grad.double() - want).norm() <= 2.0 ** -7 * want.norm())
"""
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
