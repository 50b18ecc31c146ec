"""Rows in MXFP4 and products with them (csrc/lm_mxfp4.cu) against the definition in 64 bits."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def values(x: torch.Tensor) -> torch.Tensor:
    """What the rows stand for in MXFP4, in 64 bits: every element's nearest magnitude, of two as near the one with the even code."""
    a = x.detach().cpu().double().numpy()
    rows, width = a.shape
    a = np.concatenate([a, np.zeros((rows, -width % 32))], 1).reshape(rows, -1, 32)
    with np.errstate(invalid="ignore", divide="ignore"):
        most = np.abs(a).max(-1, keepdims=True)
        finite = np.isfinite(most)
        _, e = np.frexp(np.where(finite & (most > 0), most, 2.0 ** -126))
        unit = np.ldexp(1.0, np.maximum(e - 3, -127))
        r = np.where(finite, np.abs(a) / unit, 0)
        gap = np.abs(np.minimum(r, 6)[..., None] - MAGNITUDES)
        gap[..., 1::2] += 1e-12                                  # (halves of E2M1's steps are multiples of 0.25: far more than this)
        v = np.sign(a) * MAGNITUDES[gap.argmin(-1)] * unit
        v = np.where(finite, v, np.nan)
    return torch.from_numpy(v.reshape(rows, -1)[:, :width].copy())


def rows_of(m, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(2 * torch.randn(m, 1, generator=g))
    return x.to(dtype).cuda()


def same(got, want):
    got = got.double().cpu()
    return bool(((got == want) | (got.isnan() & want.isnan())).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (2, 31), (3, 33), (7, 128), (128, 129), (129, 256), (5, 1000), (300, 2048), (1, 8192)])
def test_values_are_the_definitions(m, k, dtype):
    from dia_tts_prune_b200 import lm_ops
    x = rows_of(m, k, m + k, dtype)
    q = lm_ops.quantize_mxfp4(x)
    assert q.shape == (m, k)
    assert same(q.dequantize(), values(x))
    assert same(q.dequantize(torch.bfloat16), values(x))          # (4 significant bits: bfloat16 holds them)


def test_borders_and_extremes():
    """All halves between two magnitudes with either sign, the smallest and largest scales, subnormal numbers, signed zeros."""
    from dia_tts_prune_b200 import lm_ops
    half = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.5, 6.0, 6.5, 7.0, 7.99])
    row = torch.cat([half, -half, torch.tensor([4.0, 0.0, -0.0, 1e-30, -1e-30, 2 ** -149, 0.2499999, 0.2500001])])
    x = torch.stack([row * 2.0 ** s for s in (0, 1, -3, 100, 125, -100, -126, -140)])
    x[4] = x[4].clamp(-3.4e38, 3.4e38)
    x = torch.cat([x, torch.zeros(1, 32), torch.full((1, 32), 2.0 ** -149), torch.full((1, 32), 3.4028234e38)])
    x = torch.cat([x, torch.randn(11, 32)], 1).cuda()
    assert same(lm_ops.quantize_mxfp4(x).dequantize(), values(x))


def test_blocks_that_are_not_finite_stand_for_nan_alone():
    from dia_tts_prune_b200 import lm_ops
    x = rows_of(130, 160, 3)
    x[0, 5], x[1, 40], x[129, 159], x[7, 96] = math.inf, math.nan, -math.inf, math.nan
    got = lm_ops.quantize_mxfp4(x).dequantize().cpu()
    assert same(got, values(x))
    assert int(got.isnan().sum()) == 4 * 32
    w = rows_of(64, 160, 4)
    y = lm_ops.linear_mxfp4(x, lm_ops.quantize_mxfp4(w)).cpu()
    assert y[[0, 1, 7, 129]].isnan().all() and y.isnan().sum() == 4 * 64
    few = lm_ops.linear_mxfp4(x[:8], lm_ops.quantize_mxfp4(w)).cpu()         # (rows that are rounded inside the product)
    assert few[[0, 1, 7]].isnan().all() and few.isnan().sum() == 3 * 64
    few = lm_ops.linear_mxfp4(w[:3], lm_ops.quantize_mxfp4(x)).cpu()
    assert few[:, [0, 1, 7, 129]].isnan().all() and few.isnan().sum() == 4 * 3
    y = lm_ops.linear_mxfp4(w, lm_ops.quantize_mxfp4(x)).cpu()
    assert y[:, [0, 1, 7, 129]].isnan().all() and y.isnan().sum() == 4 * 64


def test_strides():
    """Rows that stand apart, rows that do not start at 16 bytes, and neighbours along the other axis."""
    from dia_tts_prune_b200 import lm_ops
    big = rows_of(40, 301, 9, torch.bfloat16)
    w = lm_ops.quantize_mxfp4(rows_of(33, 100, 10))
    for x in (big[:, :100], big[::3, 1:101], big[:, 201:], rows_of(100, 40, 11).T, big[:1, :100].expand(5, 100)):
        assert same(lm_ops.quantize_mxfp4(x).dequantize(), values(x))
        assert torch.equal(lm_ops.linear_mxfp4(x, w), lm_ops.linear_mxfp4(x.contiguous().clone(), w))


def check(x, w, y, values=values):
    """Products are exact; a tensor core adds 64 of them at a time to a float32 sum and cuts off, which loses at most 2^-22 of the
    magnitudes summed so far at each of K / 64 steps (2^-23 for the sum and as much for the products that are lined up with it); and the
    result's own rounding: half a step, which is eps / 2 of a normal number and eps / 2 of the smallest normal number below that (float16:
    2^-25; a result of 3e-5 stood 2.96e-8 off).  From half a step above its largest number on a type has infinities (float16: 65520)."""
    a, b = values(x), values(w)
    want, most, t = a @ b.T, a.abs() @ b.abs().T, torch.finfo(y.dtype)
    bound = (x.shape[1] / 64 + 2) * 2.0 ** -22 * most + t.eps / 2 * (want.abs() + t.smallest_normal)
    assert y.dtype == x.dtype and y.shape == want.shape
    got = y.double().to(want.device)
    beyond = got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= t.max * (1 + t.eps / 4))
    worst = torch.where(beyond, 0.0, (got - want).abs() - bound).max()
    assert worst <= 0, float(worst)


SIZES = [(1, 1, 1), (1, 2048, 2048), (2, 5, 33), (3, 130, 256), (8, 1028, 200), (9, 64, 384), (16, 257, 4096), (17, 300, 1000), (32, 128, 128), (33, 96, 640),
         (64, 2048, 1024), (65, 129, 129), (128, 128, 128), (129, 127, 500), (257, 384, 1152), (333, 1028, 2000), (1000, 640, 520),
         (150, 71, 128), (300, 1601, 900)]                                     # rows that begin anywhere


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_against_64_bits(m, n, k, dtype):
    from dia_tts_prune_b200 import lm_ops
    x, w = rows_of(m, k, m, dtype) * 0.25, rows_of(n, k, n, torch.bfloat16) / k ** 0.5
    if m > 2:
        x[m // 2] = 0
    check(x, w, lm_ops.linear_mxfp4(x, lm_ops.quantize_mxfp4(w)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(513, 12290, 1408), (1030, 12288, 2100), (2000, 9001, 1000), (8192, 4100, 640)])
def test_long_products_on_pairs_of_sms(m, n, k, dtype):
    """Tiles that are partly filled on both sides, an odd number of pieces, rows that begin anywhere; the values are those of the tests above."""
    from dia_tts_prune_b200 import lm_ops
    x, w = rows_of(m, k, m, dtype) * 0.25, rows_of(n, k, n, torch.bfloat16) / k ** 0.5
    x[m // 2] = 0
    y = lm_ops.linear_mxfp4(x, lm_ops.quantize_mxfp4(w))
    check(x, w, y, lambda a: lm_ops.quantize_mxfp4(a).dequantize().double())
    assert torch.equal(y, lm_ops.linear_mxfp4(x, lm_ops.quantize_mxfp4(w)))


def test_many_tiles_on_every_sm_and_leading_dimensions():
    from dia_tts_prune_b200 import lm_ops
    x, w = rows_of(1030, 320, 1, torch.bfloat16) * 0.25, rows_of(8200, 320, 2, torch.bfloat16)
    q = lm_ops.quantize_mxfp4(w)
    y = lm_ops.linear_mxfp4(x.view(5, 206, 320), q)
    assert y.shape == (5, 206, 8200)
    check(x, w, y.view(1030, 8200))
    assert lm_ops.linear_mxfp4(x[0], q).shape == (8200,)
    assert lm_ops.linear_mxfp4(x[:3], q, out_dtype=torch.float32).dtype == torch.float32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,shift", [(1, 130, 40, 0), (5, 2047, 300, 1), (16, 64, 8200, 0), (40, 129, 130, 1), (200, 1001, 72, 0), (200, 1001, 72, 3), (513, 12290, 700, 1)])
def test_nothing_is_written_beside_the_results(m, n, k, shift, dtype):
    """Results, values and the 4-bit buffers inside larger ones whose other bytes stay; results may begin at any element."""
    from dia_tts_prune_b200 import _lm_lib, lm_ops
    lib, st = _lm_lib.load(), torch.cuda.current_stream().cuda_stream
    x, w = rows_of(m, k, m, dtype), rows_of(n, k, n)
    q, size, code = lm_ops.quantize_mxfp4(w), dtype.itemsize, 0 if dtype == torch.float32 else 1

    def room(nbytes, off=0):
        buf = torch.full((nbytes + 1024,), 77, dtype=torch.uint8, device="cuda")
        at = (buf.data_ptr() + 511) // 256 * 256 + off
        return buf, at, at - buf.data_ptr(), nbytes

    def kept(r):
        buf, _, at, nb = r
        return bool((buf[:at] == 77).all() and (buf[at + nb:] == 77).all())

    y, v, need = room(m * n * size, shift * size), room(m * k * size, shift * size), lib.lm_b200_op_linear_mxfp4_work_bytes(m, n, k)
    work, codes, scales = room(need), room(lib.lm_b200_mxfp4_code_bytes(m, k)), room(lib.lm_b200_mxfp4_scale_bytes(m, k))
    at = q.data.data_ptr()
    assert lib.lm_b200_op_linear_mxfp4(x.data_ptr(), code, k, at, at + q.scales_at, y[1], code, m, n, k, work[1] if need else None, need, st) == 0
    assert lib.lm_b200_op_mxfp4_quantize(x.data_ptr(), code, k, m, k, codes[1], scales[1], st) == 0
    assert lib.lm_b200_op_mxfp4_dequantize(codes[1], scales[1], m, k, v[1], code, st) == 0
    torch.cuda.synchronize()
    assert all(kept(r) for r in (y, v, work, codes, scales))
    got = y[0][y[2]:y[2] + y[3]].clone().view(dtype).view(m, n)
    assert torch.equal(got, lm_ops.linear_mxfp4(x, q))
    assert torch.equal(v[0][v[2]:v[2] + v[3]].clone().view(dtype).view(m, k), lm_ops.quantize_mxfp4(x).dequantize(dtype))


def test_offsets_past_32_bits():
    """A matrix of 2^31 numbers and some: its last rows have the values, and the products, that they have alone."""
    from dia_tts_prune_b200.lm_ops import linear_mxfp4, quantize_mxfp4
    g = torch.Generator(device="cuda").manual_seed(2)
    rows, k, last = 270000, 8192, 432                              # (270000 is 2109 blocks of 128 and 48: the last 432 rows begin a block)
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q, alone = quantize_mxfp4(x), quantize_mxfp4(x[-last:])
    assert torch.equal(q.dequantize(torch.bfloat16)[-last:], alone.dequantize(torch.bfloat16))
    for m in (2, 40, 300):
        a = torch.randn(m, k, generator=g, device="cuda").bfloat16()
        assert torch.equal(linear_mxfp4(a, q)[:, -last:], linear_mxfp4(a, alone))
    w = quantize_mxfp4(torch.randn(8200, k, generator=g, device="cuda"))
    assert torch.equal(linear_mxfp4(x, w)[-last:], linear_mxfp4(x[-last:], w))


@pytest.mark.parametrize("m,k", [(1, 1), (3, 33), (7, 128), (129, 257), (300, 2048)])
def test_values_in_float16(m, k):
    """The nearest float16 of every value: exact in its normal range, subnormal numbers below (half way: to the even one), infinities from 65520 on."""
    from dia_tts_prune_b200 import lm_ops
    x = rows_of(m, k, m + k)
    scale = 2.0 ** torch.linspace(-40, 24, m)[:, None].round().cuda()
    for y in (x, x * scale, x.half(), torch.full_like(x, 65504.0), torch.full_like(x, 2.0 ** -24), torch.full_like(x, 2.0 ** -25), torch.full_like(x, 3.0 * 2.0 ** -26)):
        want = values(y).float().half()                            # (float32 holds the values as they are)
        got = lm_ops.quantize_mxfp4(y).dequantize(torch.float16)
        assert got.dtype == torch.float16 and same(got, want.double())
    y = x.clone()
    y[0, 0] = math.nan
    assert same(lm_ops.quantize_mxfp4(y).dequantize(torch.float16), values(y).float().half().double())


def test_more_rows_than_a_grid_has_room_for():
    """65535 x 128 rows and some: rounding, values and products of the rows on either side of the border are what they are alone."""
    from dia_tts_prune_b200.lm_ops import linear_mxfp4, quantize_mxfp4
    rows, k, at = 65535 * 128 + 300, 40, 65535 * 128 - 200
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(6))
    q = quantize_mxfp4(x)
    for part in (slice(0, 300), slice(at, rows)):
        assert same(q.dequantize()[part], values(x[part]))
    w = rows_of(12, k, 3, torch.bfloat16)
    w4 = quantize_mxfp4(w)
    y = linear_mxfp4(x, w4)
    check(x[at:], w, y[at:])
    assert torch.equal(y[at:], linear_mxfp4(x[at:], w4)) and torch.equal(y[:1000], linear_mxfp4(x[:1000], w4))
    z = linear_mxfp4(w, q)                                         # (as the matrix of a product)
    assert torch.equal(z[:, at:], linear_mxfp4(w, quantize_mxfp4(x[at - 56:]))[:, 56:])      # (from a block of 128 rows on)
