"""The cross entropy of rows under a head and its gradient (csrc/lm_loss.cu) against the definition in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def operands(m, v, k, seed, dtype=torch.bfloat16, ignored=0.2, lean=6.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(v, k, generator=g) / k ** 0.5).bfloat16()
    t = torch.randint(0, v, (m,), generator=g)
    h = torch.randn(m, k, generator=g) + lean * torch.rand(m, 1, generator=g) * w[t].float()
    t[torch.rand(m, generator=g) < ignored] = -100
    return h.to(dtype).cuda(), w.cuda(), t.cuda()


class Exact:
    """Losses, probabilities and gradients in 64 bits, and how far off the kernels' may be.

    A logit is a sum of exact products; the tensor core adds 16 at a time to a float32 sum and cuts off, at most 2^-22 of the magnitudes
    so far at each of K / 16 steps (float32 rows: three times as many, and 2^-22 of each product beyond their three terms): ``dz``.  A loss
    moves by twice the largest of them, by 2^-20 for the exponentials and logarithms and by a few roundings of its parts."""

    def __init__(self, h, w, t, scale=1.0):
        self.h, self.w, t = h.detach().double().cpu(), w.detach().double().cpu(), t.cpu().long()
        self.keep, self.scale, k = t != -100, scale, h.shape[1]
        z = scale * self.h @ self.w.T
        self.steps = (k / 16 + 2) * (3 if h.dtype == torch.float32 else 1) * 2.0 ** -22
        self.dz = self.steps * scale * (self.h.abs() @ self.w.abs().T).amax(1)
        logp, at = torch.log_softmax(z, 1), torch.where(self.keep, t, 0)[:, None]
        self.loss = torch.where(self.keep, -logp.gather(1, at)[:, 0], 0.0)
        self.loss_off = torch.where(self.keep, 2 * self.dz + 2.0 ** -20 + 2.0 ** -22 * (z.abs().amax(1) + self.loss), 0.0)
        self.p, self.onehot = logp.exp(), torch.zeros_like(z).scatter_(1, at, 1.0)

    def gradient(self, g, own=False):
        """(by rows, by the head) and their bounds: P is off by 2^-8 of itself (bfloat16) and by its probability's 4 dz + 2^-18; the sums of V
        (or M) products lose as the logits do, in pieces; and the results are bfloat16.  own: rows with factors of their own take them into
        h for the head's gradient, which is rounded once more (2^-8, and 2^-8 of that of P)."""
        g = (g.double().cpu() * self.keep * self.scale)[:, None]
        P = (self.p - self.onehot) * g
        dP = 2.0 ** -8 * P.abs() + (self.p * g).abs() * (4 * self.dz[:, None] + 2.0 ** -18) + P.abs() * 2.0 ** -18
        out = []
        for a, da, b in ((P, dP, self.w), (P.T, dP.T + (1.01 * 2.0 ** -8 * P.T.abs() if own else 0), self.h)):
            want, lost = a @ b, (a.shape[1] / 16 + 2) * 2.0 ** -22
            out.append((want, 1.01 * (da @ b.abs()) + lost * (a.abs() @ b.abs()) + 2.0 ** -8 * want.abs() + 2.0 ** -133))
        return out


def within(got, want, bound):
    off = (got.detach().double().cpu() - want).abs() - bound
    assert not off.isnan().any() and off.max() <= 0, float(off.max())


SIZES = [(1, 1, 1), (1, 2, 8), (1, 256, 64), (2, 257, 65), (3, 300, 52), (16, 50000, 136), (17, 700, 1100), (32, 129, 2048), (33, 520, 64), (127, 64, 128), (129, 1000, 100), (256, 511, 72), (257, 1025, 200), (5, 20000, 64),
         (300, 9000, 96), (40, 640, 2048), (700, 300, 1001),
         (16400, 4500, 40)]                                        # two pieces of the vocabulary


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,v,k", SIZES)
def test_losses(m, v, k, dtype):
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(m, v, k, m + v, dtype)
    for scale in (1.0, 0.25):
        e = Exact(h, w, t, scale)
        within(linear_cross_entropy(h, w, t, scale=scale, reduction="none"), e.loss, e.loss_off)
        n = max(int(e.keep.sum()), 1)
        for reduction, by in (("sum", 1), ("mean", n)):
            got = linear_cross_entropy(h, w, t.int(), scale=scale, reduction=reduction)
            within(got, e.loss.sum() / by, e.loss_off.sum() / by + 2.0 ** -23 * e.loss.sum() / by)


@pytest.mark.parametrize("m,v,k", SIZES)
def test_gradients(m, v, k):
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(m, v, k, 2 * m + v)
    h.requires_grad_(True), w.requires_grad_(True)
    e = Exact(h, w, t, 0.5)
    loss = linear_cross_entropy(h, w, t, scale=0.5)
    dh, dw = torch.autograd.grad(loss, (h, w))
    n = max(int(e.keep.sum()), 1)
    (want_h, off_h), (want_w, off_w) = e.gradient(torch.full((m,), 1.0 / n))
    assert dh.dtype == dw.dtype == torch.bfloat16
    within(dh, want_h, off_h)
    within(dw, want_w, off_w)
    # every token's own factor, through an expanded and a strided gradient, one input at a time
    g = torch.randn(m, generator=torch.Generator().manual_seed(m)).cuda()
    (want_h, off_h), (want_w, off_w) = e.gradient(g, own=True)
    loss = linear_cross_entropy(h, w.detach(), t, scale=0.5, reduction="none")
    within(torch.autograd.grad(loss, h, torch.stack([g, g], 1)[:, 0])[0], want_h, off_h)
    loss = linear_cross_entropy(h.detach(), w, t, scale=0.5, reduction="none")
    within(torch.autograd.grad(loss, w, g)[0], want_w, off_w)
    loss = linear_cross_entropy(h, w, t, scale=0.5, reduction="none")
    (want_h, off_h), _ = e.gradient(torch.ones(m))
    within(torch.autograd.grad(loss.sum(), h)[0], want_h, off_h)


def test_gradient_against_differences():
    """Central differences of the loss in 64 bits along random directions, and the gradient's own product with them: the two differ by the
    gradient's bound (see Exact) times the direction and by the third derivative's step^2 / 6 < 1e-6 of a loss whose logits move by less than one."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(33, 700, 48, 5)
    h.requires_grad_(True), w.requires_grad_(True)
    dh, dw = torch.autograd.grad(linear_cross_entropy(h, w, t, reduction="sum"), (h, w))
    e = Exact(h, w, t)
    (_, off_h), (_, off_w) = e.gradient(torch.ones(33))

    def loss(a, b):
        return torch.nn.functional.cross_entropy(a @ b.T, t.cpu(), reduction="sum")

    g = torch.Generator().manual_seed(0)
    for _ in range(4):
        u, s = torch.randn(e.h.shape, generator=g).double(), 1e-4
        slope = (loss(e.h + s * u, e.w) - loss(e.h - s * u, e.w)) / (2 * s)
        assert abs(slope - (dh.double().cpu() * u).sum()) <= (off_h * u.abs()).sum() + 1e-4
        u = torch.randn(e.w.shape, generator=g).double()
        slope = (loss(e.h, e.w + s * u) - loss(e.h, e.w - s * u)) / (2 * s)
        assert abs(slope - (dw.double().cpu() * u).sum()) <= (off_w * u.abs()).sum() + 1e-4


def test_rows_that_do_not_count_and_bad_targets():
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(40, 500, 64, 7, ignored=0.0)
    t[3], t[17], t[39] = -100, -100, -100
    clean = h.clone()
    h[3], h[17, 5], h[39, 0] = math.nan, math.inf, -math.inf
    clean[[3, 17, 39]] = 0
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(a, b, t)
    dh, dw = torch.autograd.grad(loss, (a, b))
    a0, b0 = clean.requires_grad_(True), w.clone().requires_grad_(True)
    loss0 = linear_cross_entropy(a0, b0, t)
    dh0, dw0 = torch.autograd.grad(loss0, (a0, b0))
    assert loss.isfinite() and torch.equal(loss, loss0) and torch.equal(dh, dh0) and torch.equal(dw, dw0) and not dh[[3, 17, 39]].any()
    # nothing counts: zero, with gradients of zeros
    none = torch.full_like(t, -100)
    loss = linear_cross_entropy(a, b, none)
    dh, dw = torch.autograd.grad(loss, (a, b))
    assert loss == 0 and not dh.any() and not dw.any()
    assert linear_cross_entropy(a, b, none, reduction="sum") == 0 and not linear_cross_entropy(a, b, none, reduction="none").any()
    # a target outside the vocabulary shows, in its row alone
    bad = t.clone()
    bad[5], bad[6] = 500, -1
    rows = linear_cross_entropy(a0, b0, bad, reduction="none")
    assert rows.isnan().nonzero()[:, 0].tolist() == [5, 6]
    dh, = torch.autograd.grad(rows[:5].sum() + rows[7:].sum(), a0)
    assert torch.equal(dh[0], torch.autograd.grad(linear_cross_entropy(a0, b0, t, reduction="sum"), a0)[0][0])
    # another number for the rows that do not count
    assert torch.equal(linear_cross_entropy(a0, b0, torch.where(t == -100, 7, t), ignore_index=7, reduction="none")[3], rows[3])


def test_infinities_and_far_logits():
    """Logits of hundreds, a head row of minus infinities (probability zero) and a loss next to zero, which keeps its digits."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(20, 400, 64, 8, ignored=0.0)
    far = (h.float() * 64).bfloat16()
    e = Exact(far, w, t)
    within(linear_cross_entropy(far, w, t, reduction="none"), e.loss, e.loss_off)
    pos = h.abs() + 0.5
    w2 = w.clone()
    w2[11] = -math.inf
    w2[64:96] = -math.inf                                          # (a whole block of columns)
    t2 = torch.where((t == 11) | ((t >= 64) & (t < 96)), 0, t)
    kept = torch.tensor([j for j in range(400) if j != 11 and not 64 <= j < 96])
    at = torch.searchsorted(kept, t2.cpu())
    e = Exact(pos, w[kept.cuda()], at)
    within(linear_cross_entropy(pos, w2, t2, reduction="none"), e.loss, e.loss_off)
    sure, one = torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 64, dtype=torch.bfloat16, device="cuda")
    sure[0, 0], one[1, 0] = 16.0, 1.0
    got = linear_cross_entropy(sure, one, torch.tensor([1], device="cuda"), reduction="none")
    want = math.log1p(2 * math.exp(-16.0))                         # 2.25e-7; float32's sum 1 + that is off by 2^-24 (6e-8) at most
    assert abs(float(got) - want) <= 2.0 ** -23


@pytest.mark.parametrize("v", [300, 4097, 513])
def test_gradients_of_far_away_logits(v):
    """All logits of a row hundreds below (or above) zero, a vocabulary that ends inside a tile: columns that are not there have logits of
    zero, far above those, and no part in the gradients."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    for m in (3, 140, 300):
        for sign in (-1.0, 1.0):
            h, w, t = operands(m, v, 64, 31)
            h[:, 0], w[:, 0] = 32.0, 8.0 * sign                    # (256 of every logit)
            e = Exact(h, w, t)
            assert float(e.p.sum(1).sub(1).abs().max()) < 1e-9 and float((e.h @ e.w.T).mul(sign).min()) > 150
            a, b = h.requires_grad_(True), w.requires_grad_(True)
            loss = linear_cross_entropy(a, b, t, reduction="none")
            within(loss, e.loss, e.loss_off)
            got = torch.autograd.grad(loss.sum(), (a, b))
            for x, (want, bound) in zip(got, e.gradient(torch.ones(m))):
                within(x, want, bound)


def test_factors_of_rows_that_lie_far_apart():
    """Gradients of every row's loss may come with any stride."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(3, 40, 16, 5, ignored=0.0)
    g = torch.tensor([1.0, -2.0, 0.5], device="cuda")
    far = torch.empty_strided((3,), ((1 << 31) + 3,), dtype=torch.float32, device="cuda")     # (17 GB, of which three numbers are touched)
    far.copy_(g)
    out = []
    for by in (g, far, torch.stack((g, g), 1)[:, 1], g.flip(0).flip(0)):
        a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        out.append(torch.autograd.grad(linear_cross_entropy(a, b, t, reduction="none"), (a, b), by))
    for x in out[1:]:
        assert torch.equal(x[0], out[0][0]) and torch.equal(x[1], out[0][1])


def test_strides_leading_dimensions_and_empty():
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(24, 300, 104, 9)
    want = linear_cross_entropy(h, w, t, reduction="none")
    big = torch.zeros(24, 333, dtype=torch.bfloat16, device="cuda")
    big[:, 8:112] = h
    wide = torch.zeros(300, 120, dtype=torch.bfloat16, device="cuda")
    wide[:, :104] = w
    odd = torch.zeros(600, 107, dtype=torch.bfloat16, device="cuda")
    odd[::2, 1:105] = w
    for a in (big[:, 8:112], h.T.contiguous().T):
        for b in (wide[:, :104], odd[::2, 1:105], w.T.contiguous().T):
            assert torch.equal(linear_cross_entropy(a, b, t, reduction="none"), want)
            x, y = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
            p, q = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
            for got, ref in zip(torch.autograd.grad(linear_cross_entropy(x, y, t), (x, y)), torch.autograd.grad(linear_cross_entropy(p, q, t), (p, q))):
                assert torch.equal(got, ref)
    assert torch.equal(linear_cross_entropy(h.view(4, 6, 104), w, t.view(4, 6), reduction="none"), want.view(4, 6))
    assert torch.equal(linear_cross_entropy(h[0], w, t[0], reduction="none"), want[0])
    assert linear_cross_entropy(h[:0], w, t[:0], reduction="none").shape == (0,)
    assert linear_cross_entropy(h[:0], w, t[:0]) == 0
    a, b = h[:0].clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(a, b, t[:0])
    loss.backward()
    assert loss == 0 and a.grad.shape == (0, 104) and not b.grad.any()


@pytest.mark.parametrize("m,v,k", [(1, 40, 7), (33, 300, 100), (129, 257, 65), (300, 1025, 264)])
def test_nothing_is_written_beside_the_results(m, v, k):
    """Every output inside a larger buffer whose other bytes stay: losses, what the gradient needs, both gradients, the workspace."""
    from dia_tts_prune_b200 import _lm_lib
    lib, st = _lm_lib.load(), torch.cuda.current_stream().cuda_stream
    h, w, t = operands(m, v, k, 3)

    def room(nbytes, align=256):
        buf = torch.full((nbytes + 4 * align,), 77, dtype=torch.uint8, device="cuda")
        at = (buf.data_ptr() + 2 * align - 1) // align * align
        return buf, at, at - buf.data_ptr(), nbytes

    def kept(r):
        buf, _, at, n = r
        return bool((buf[:at] == 77).all() and (buf[at + n:] == 77).all())

    each, one, keep, dh, dw = room(4 * m), room(4), room(8 * m + 4), room(2 * m * k), room(2 * v * k)
    need = lib.lm_b200_op_loss_work_bytes(h.data_ptr(), 1, k, w.data_ptr(), k, m, v, k)
    work = room(need)
    for reduction, out in ((0, each), (2, one)):
        assert lib.lm_b200_op_loss(h.data_ptr(), 1, k, w.data_ptr(), k, t.data_ptr(), 1, -100, m, v, k, 1.0, reduction, out[1], keep[1], work[1], need, st) == 0
    need = lib.lm_b200_op_loss_grad_work_bytes(h.data_ptr(), k, w.data_ptr(), k, m, v, k, 1, 1)
    work2, g = room(need), torch.ones((), device="cuda")
    assert lib.lm_b200_op_loss_grad(h.data_ptr(), k, w.data_ptr(), k, t.data_ptr(), 1, -100, m, v, k, 1.0, keep[1], g.data_ptr(), 0, keep[1] + 8 * m, dh[1], dw[1],
                                    work2[1], need, st) == 0
    torch.cuda.synchronize()
    assert all(kept(r) for r in (each, one, keep, dh, dw, work, work2))


def test_offsets_past_32_bits():
    """Rows, and a head, of 2^31 numbers and some: losses and gradients of the last rows are what they are alone; the head's last rows have
    the formula's gradient."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    g = torch.Generator(device="cuda").manual_seed(2)
    rows, k, v, last = 270000, 8192, 300, 432
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w, t = (torch.randn(v, k, generator=g, device="cuda") / 90).bfloat16(), torch.randint(0, v, (rows,), generator=g, device="cuda")
    got = []
    for a, targets in ((x, t), (x[-last:], t[-last:])):
        a = a.detach().requires_grad_(True)
        loss = linear_cross_entropy(a, w, targets, reduction="none")
        got.append((loss[-last:], torch.autograd.grad(loss.sum(), a)[0][-last:]))
    # (logits alike; dh's sums over the vocabulary may be split where there are few rows: a rounding and the sums' own loss apart)
    assert torch.equal(got[0][0], got[1][0])
    z = (x[-last:].double() @ w.double().T).softmax(1)
    z[torch.arange(last), t[-last:]] -= 1
    bound = 2.0 ** -7 * got[1][1].double().abs() + 2.0 ** -18 * (z.abs() @ w.double().abs())
    assert ((got[0][1].double() - got[1][1].double()).abs() <= bound).all()
    del got, a, loss
    for m in (3, 40):
        h = (torch.randn(m, k, generator=g, device="cuda") / 30).bfloat16()
        t = torch.randint(rows - last, rows, (m,), generator=g, device="cuda")
        a, b = h.clone().requires_grad_(True), x.requires_grad_(True)
        loss = linear_cross_entropy(a, b, t, reduction="none")
        lse = torch.full((m,), -math.inf, dtype=torch.float64, device="cuda")
        for i in range(0, rows, 27000):
            lse = torch.logaddexp(lse, (h.double() @ x.detach()[i:i + 27000].double().T).logsumexp(1))
        tail = x.detach()[-last:].double()
        z = h.double() @ tail.T
        dz = (k / 16 + 2) * 2.0 ** -22 * float((h.double().abs() @ tail.abs().T).max()) * 1.5      # (of other rows too: their largest is like that)
        hit = z.gather(1, (t - (rows - last))[:, None])[:, 0]
        assert ((loss.double() - (lse - hit)).abs() <= 2 * dz + 2.0 ** -20 + 2.0 ** -22 * (z.abs().amax() + loss.double())).all()
        dw = torch.autograd.grad(loss.sum(), b)[0][-last:].double()
        P = (z - lse[:, None]).exp()
        dP = P * (4 * dz + 2.0 ** -18)
        P[torch.arange(m), t - (rows - last)] -= 1
        want = P.T @ h.double()
        bound = 1.01 * ((dP + (2.0 ** -8 + 2.0 ** -18) * P.abs()).T @ h.double().abs()) + (m / 16 + 2) * 2.0 ** -22 * (P.abs().T @ h.double().abs())
        assert ((dw - want).abs() <= bound + 2.0 ** -8 * want.abs() + 2.0 ** -133).all()


@pytest.mark.parametrize("m,v,k", [(129, 8500, 1000), (40, 8449, 64), (1, 9473, 96), (256, 14400, 512), (1000, 13313, 200), (3, 12290, 4)])
def test_every_share_of_the_rows_gradient_is_written(m, v, k):
    """The gradient by the rows is a sum of shares of the vocabulary.  These end short of a whole piece of it, so that dividing the piece and
    dividing the columns that are there give different numbers of shares; the workspace holds NaN beforehand."""
    from dia_tts_prune_b200 import _lm_lib
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    lib, st = _lm_lib.load(), torch.cuda.current_stream().cuda_stream
    h, w, t = operands(m, v, k, m + v)
    e = Exact(h, w, t, 0.5)
    n = max(int(e.keep.sum()), 1)
    (want_h, off_h), (want_w, off_w) = e.gradient(torch.full((m,), 1.0 / n))
    ld = (k + 7) // 8 * 8
    a, b = (torch.nn.functional.pad(x, (0, ld - k)) for x in (h, w))
    kept, out = torch.empty(2 * m + 1, device="cuda"), torch.empty((), device="cuda")
    need = lib.lm_b200_op_loss_work_bytes(a.data_ptr(), 1, ld, b.data_ptr(), ld, m, v, k)
    work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    assert lib.lm_b200_op_loss(a.data_ptr(), 1, ld, b.data_ptr(), ld, t.data_ptr(), 1, -100, m, v, k, 0.5, 2, out.data_ptr(), kept.data_ptr(), work.data_ptr(), need, st) == 0
    one = torch.ones((), device="cuda")
    for rows, head in ((True, True), (True, False), (False, True)):
        dh, dw = (torch.full(s, math.nan, dtype=torch.bfloat16, device="cuda") for s in ((m, k), (v, k)))
        need = lib.lm_b200_op_loss_grad_work_bytes(a.data_ptr(), ld, b.data_ptr(), ld, m, v, k, rows, head)
        work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        assert lib.lm_b200_op_loss_grad(a.data_ptr(), ld, b.data_ptr(), ld, t.data_ptr(), 1, -100, m, v, k, 0.5, kept.data_ptr(), one.data_ptr(), 0, kept.data_ptr() + 8 * m,
                                        dh.data_ptr() if rows else None, dw.data_ptr() if head else None, work.data_ptr(), need, st) == 0
        if rows:
            within(dh, want_h, off_h)
        if head:
            within(dw, want_w, off_w)
    # and as a program calls it, behind others whose workspaces it takes over
    x, y = h.requires_grad_(True), w.requires_grad_(True)
    for _ in range(3):
        torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        within(torch.autograd.grad(linear_cross_entropy(x, y, t, scale=0.5), x)[0], want_h, off_h)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("shape", [(0,), (3, 0)])
def test_losses_of_nothing_have_gradients_of_zeros(shape, reduction):
    """Whichever of the two asks for one."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    t = torch.zeros(shape, dtype=torch.long, device="cuda")
    for rows, head in ((True, True), (True, False), (False, True)):
        h = torch.zeros(*shape, 16, dtype=torch.bfloat16, device="cuda", requires_grad=rows)
        w = torch.full((40, 16), math.inf, dtype=torch.bfloat16, device="cuda", requires_grad=head)
        loss = linear_cross_entropy(h, w, t, reduction=reduction)
        assert loss.dtype == torch.float32 and loss.shape == (shape if reduction == "none" else ())
        loss.sum().backward()
        assert loss.sum() == 0
        if rows:
            assert h.grad.shape == h.shape
        if head:
            assert w.grad.shape == w.shape and not w.grad.any()
    assert not linear_cross_entropy(h.detach(), w.detach(), t, reduction=reduction).requires_grad


@pytest.mark.parametrize("m,v,k", [(40, 300, 4104), (200, 520, 8200), (129, 257, 4097), (33000, 300, 40), (70000, 513, 24), (1, 600000, 8), (257, 32900, 4700)])
def test_contractions_longer_than_an_accumulator(m, v, k):
    """Channels beyond 4096 (P), rows beyond 32768 (the head's gradient), columns of a share beyond 32768 (the rows')."""
    test_gradients(m, v, k)


def test_long_sums_of_one_sign_do_not_drift():
    """Sums whose terms have one sign, which a tensor-core accumulator cuts off at every step (16 terms, up to 2^-23 of the sum).

    Head: probabilities of one half (no logit differs), so that its second row's gradient is half the sum of 2^23 positive rows: 2^-12 for
    the 2048 steps of an accumulator, 2^-16 for 256 float32 sums of them, 2^-8 for the result's rounding, each relative.
    Rows of 2^18 channels with logits of about 40: P by one accumulator for 4096 channels (256 steps, 2^-15 of the logit) and 64 sums in
    float32 (2^-18), the log-sum by one for 1024 (64 steps, 2^-17) and 256 sums (2^-16)."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    g = torch.Generator(device="cuda").manual_seed(1)
    h = (1 + torch.rand(1 << 23, 8, generator=g, device="cuda")).bfloat16()
    w = torch.zeros(2, 8, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(linear_cross_entropy(h, w, torch.zeros(1 << 23, dtype=torch.int32, device="cuda"), reduction="sum"), w)
    want = 0.5 * h.double().sum(0)
    assert ((dw[1].double() / want - 1).abs() <= 2.0 ** -8 + 2.0 ** -12 + 2.0 ** -15).all(), (dw[1].double() / want - 1).tolist()
    assert torch.equal(dw[0], -dw[1])
    del h
    k = 1 << 18
    h = (1 + torch.rand(40, k, generator=g, device="cuda")).bfloat16()
    w = ((1 + torch.rand(64, k, generator=g, device="cuda")) * (40 / 2.25 / k)).bfloat16()
    t = torch.randint(0, 64, (40,), generator=g, device="cuda")
    e = Exact(h, w, t)
    e.dz = (2.0 ** -15 + 2.0 ** -18 + 2.0 ** -17 + 2.0 ** -16) / 4 * (e.h.abs() @ e.w.abs().T).amax(1)      # (the bound of P has it four times)
    a, b = h.requires_grad_(True), w.requires_grad_(True)
    got = torch.autograd.grad(linear_cross_entropy(a, b, t, reduction="sum"), (a, b))
    for x, (ref, bound) in zip(got, e.gradient(torch.ones(40))):
        within(x, ref, bound)


@pytest.mark.parametrize("m", [3, 50, 300])
@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** 126])
def test_the_smallest_and_largest_scale(m, scale):
    """Logits next to zero: the loss is the vocabulary's logarithm (2^-20 for exponentials and logarithms), the gradient zero times the scale or
    as small as that."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(m, 300, 72, m, ignored=0.0)
    if scale > 1:
        h.zero_()
    h.requires_grad_(True)
    loss = linear_cross_entropy(h, w, t, scale=scale, reduction="none")
    assert ((loss.double() - math.log(300)).abs() <= 2.0 ** -18).all()
    dh, = torch.autograd.grad(loss.sum(), h)
    want = (torch.full((m, 300), 1 / 300, device="cuda", dtype=torch.float64).scatter_add_(1, t[:, None], -torch.ones(m, 1, device="cuda", dtype=torch.float64)) @ w.double())
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -7 * (1 / 300 * w.double().abs().sum(0) + w.double().abs()[t])
    assert ((dh.double() / scale - want).abs() <= bound + 2.0 ** -133 / scale).all()


def test_second_derivatives_are_refused():
    """A gradient taken with its graph may be used, but not differentiated: not alone, and not beside a term that has a derivative."""
    from dia_tts_prune_b200.lm_ops import linear_cross_entropy
    h, w, t = operands(20, 300, 64, 4)
    for rows, head in ((True, True), (True, False), (False, True)):
        a, b = h.clone().requires_grad_(rows), w.clone().requires_grad_(head)
        leaves = [x for x in (a, b) if x.requires_grad]
        loss = linear_cross_entropy(a, b, t)
        want = torch.autograd.grad(loss, leaves, retain_graph=True)
        got = torch.autograd.grad(loss, leaves, create_graph=True)
        assert all(torch.equal(u, v) for u, v in zip(got, want)) and all(x.requires_grad for x in got)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(sum(x.float().square().sum() for x in got), leaves, retain_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            (loss + got[0].float().square().sum()).backward()
        # kept, but not differentiated
        loss = linear_cross_entropy(a, b, t)
        loss.backward(create_graph=True)
        assert torch.equal((a if rows else b).grad, want[0])
        a.grad = b.grad = None
