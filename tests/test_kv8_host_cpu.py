"""What the cache in 8 bits and its attention refuse, and how their C entries answer what they do not take: without a GPU."""

import copy
import ctypes as C
import math

import pytest
import torch

from dia_tts_prune_b200 import _lm_lib, lm_ops


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def test_caches_that_are_refused():
    for k in (dict(format="e5m2"), dict(format=None), dict(page_size=8), dict(page_size=24), dict(page_size=256)):
        with pytest.raises(ValueError):
            lm_ops.Kv8(4, 2, 64, device="cpu", **k)
    for a in ((0, 2, 64), (4, 0, 64), (4, 2, 0), (4, 2, 257), (4, 4097, 64), (1 << 31, 2, 64), (-1, 2, 64)):
        with pytest.raises(ValueError):
            lm_ops.Kv8(*a, device="cpu")


def test_a_cache_holds_what_it_says():
    c = lm_ops.Kv8(5, 3, 72, page_size=32, format="int8", device="cpu")
    assert c.keys.shape == c.values.shape == (5, 3, 32, 80) and c.keys.dtype == torch.uint8 and c.key_scales.shape == c.value_scales.shape == (5, 3)
    assert c.nbytes == 2 * (5 * 3 * 32 * 80 + 4 * 5 * 3) and c.device.type == "cpu" and (c.pages, c.kv_heads, c.dim, c.page_size, c.format) == (5, 3, 72, 32, "int8")
    assert not c.keys.any() and not c.value_scales.any()
    # the kernels have the tensors' addresses: other tensors in their place are refused, and so are copies that would share them unseen
    for name in ("keys", "values", "key_scales", "value_scales", "pages", "dim"):
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name))
    with pytest.raises(Exception):
        copy.deepcopy(c)


def operands(rows=3, sequences=2):
    c = lm_ops.Kv8(4, 2, 64, device="cpu")
    x = torch.randn(rows, 8, 64)
    return c, x[:, :4], x[:, 4:6], x[:, 6:], ints([[0, 1, -1], [2, 3, -1]])[:sequences], ints([5, 0])[:sequences], ints([0, 1, 3])[:sequences + 1]


def test_rows_that_are_refused():
    c, q, k, v, table, past, first = operands()
    for bad in (k.double(), k.int(), [1.0], None):
        for a in ((bad, v), (k, bad)):
            with pytest.raises(TypeError):
                c.append(*a, table, past, first)
        with pytest.raises(TypeError):
            lm_ops.attention_kv8(bad, c, table, past, first)
    for a in ((k[:, :1], v[:, :1]), (k[..., :63], v[..., :63]), (k[0], v[0]), (k, v[:2]), (k.bfloat16(), v), (k, v[:, :1])):
        with pytest.raises(ValueError, match="of one type"):
            c.append(*a, table, past, first)
    for bad in (q[:, :3], q[..., :63], q[0], q[:, :0]):
        with pytest.raises(ValueError, match="does not go with"):
            lm_ops.attention_kv8(bad, c, table, past, first)
    with pytest.raises(TypeError):
        lm_ops.attention_kv8(q, c.keys, table, past, first)
    for a in ((k.clone().requires_grad_(True), v), (k, v.clone().requires_grad_(True))):
        with pytest.raises(ValueError, match="gradient"):
            c.append(*a, table, past, first)
    with pytest.raises(ValueError, match="gradient"):
        lm_ops.attention_kv8(q.clone().requires_grad_(True), c, table, past, first)
    for scale in (0.0, -1.0, math.inf, math.nan, 2.0 ** 127):
        with pytest.raises(ValueError, match="scale"):
            lm_ops.attention_kv8(q, c, table, past, first, scale=scale)
    for window in (0, -1, 1 << 31):
        with pytest.raises(ValueError, match="window"):
            lm_ops.attention_kv8(q, c, table, past, first, window=window)
    with pytest.raises(TypeError):
        c.read(table, past, first, 3, torch.float64)
    with pytest.raises(ValueError, match="negative"):
        c.read(table, past, first, -1)
    with pytest.raises(TypeError):
        c.read(table, past, first, 3, torch.uint8)


def calls(c, q, k, v):
    return [lambda t, p, f: c.append(k, v, t, p, f), lambda t, p, f: c.read(t, p, f, k.shape[0]), lambda t, p, f: lm_ops.attention_kv8(q, c, t, p, f)]


def test_steps_that_are_refused():
    c, q, k, v, table, past, first = operands()
    for call in calls(c, q, k, v):
        for a in ((table.long(), past, first), (table, past.long(), first), (table, past, first.long()), (table.float(), past, first), (table.tolist(), past, first), (table, [5, 0], first),
                  (table, None, first)):
            with pytest.raises(TypeError):
                call(*a)
        apart, wide = ints([5, 9, 0, 9])[::2], ints([[0, 9, 1, 9], [2, 9, 3, 9]])[:, ::2]
        for a in ((table[0], past, first), (table[None], past, first), (wide, past, first), (table, past[:1], first), (table, past[None], first), (table, apart, first), (table, past, first[:2]),
                  (table, past, ints([0, 9, 1, 9, 3, 9])[::2]), (table, past, past), (table, past, None)):
            with pytest.raises(ValueError):
                call(*a)
        with pytest.raises(ValueError, match="CUDA"):
            call(table, past, first)
    if torch.cuda.is_available():
        there = lm_ops.Kv8(4, 2, 64)
        for call in calls(there, q.cuda(), k.cuda(), v.cuda()):
            for moved in range(3):
                with pytest.raises(ValueError, match="one device"):
                    call(*(x if i == moved else x.cuda() for i, x in enumerate((table, past, first))))
        table, past, first = table.cuda(), past.cuda(), first.cuda()
        for call in calls(there, q, k, v)[::2]:
            with pytest.raises(ValueError, match="one device"):
                call(table, past, first)
        with pytest.raises(ValueError, match="one device"):
            lm_ops.attention_kv8(q.cuda(), there, table, past, first, sinks=torch.zeros(4))


def test_sinks_that_are_refused(monkeypatch):
    c, q, k, v, table, past, first = operands()
    monkeypatch.setattr(lm_ops, "_check_device", lambda *a: None)
    monkeypatch.setattr(lm_ops, "_call", lambda *a: pytest.fail("reached the library"))
    for bad in (torch.zeros(4).double(), torch.zeros(4).bfloat16(), [0.0] * 4):
        with pytest.raises(TypeError):
            lm_ops.attention_kv8(q, c, table, past, first, sinks=bad)
    for bad in (torch.zeros(3), torch.zeros(4, 1), torch.tensor(0.0)):
        with pytest.raises(ValueError, match="sinks"):
            lm_ops.attention_kv8(q, c, table, past, first, sinks=bad)


def test_what_the_library_is_given(monkeypatch):
    """Strides of rows that may be read where they are, a step's description, and no call at all for one without rows."""
    c, q, k, v, table, past, first = operands()
    got = []
    monkeypatch.setattr(lm_ops, "_check_device", lambda *a: None)
    monkeypatch.setattr(lm_ops, "_call", lambda what, device, *a: got.append((what, a)))
    c.append(k, v, table, past, first)
    what, a = got.pop()
    assert what == "kv8_append" and a[0] == C.addressof(c._handle) and a[2:] == (k.data_ptr(), 8 * 64, 64, v.data_ptr(), 8 * 64, 64, _lm_lib.TYPE_FP32)
    assert lm_ops._KV8_STEP.unpack(a[1]) == (table.data_ptr(), 3, past.data_ptr(), first.data_ptr(), 3, 2, 3)
    lm_ops.attention_kv8(q[:2], c, table, past, window=7)
    what, a = got.pop()
    assert what == "kv8_attention" and lm_ops._KV8_STEP.unpack(a[1])[3:] == (0, 3, 2, 2) and a[2:9] == (q.data_ptr(), 8 * 64, 64, 4, _lm_lib.TYPE_FP32, 64 ** -0.5, 7) and a[9] is None
    k, v = c.read(table, past, first, 3, torch.bfloat16)
    assert k.shape == v.shape == (3, 2, 64) and k.dtype == torch.bfloat16 and k.is_contiguous() and got.pop()[0] == "kv8_read"
    none, empty = table[:0], past[:0]
    c.append(k[:0], v[:0], table, past, first)
    assert not c.read(none, empty, first[:1], 5)[0].any() and not c.read(table[:, :0], past, first, 3)[1].any()
    assert lm_ops.attention_kv8(q[:0], c, table, past, first).shape == (0, 4, 64) and not lm_ops.attention_kv8(q, c, none, empty, first[:1]).any()
    assert not got


def test_c_entries_answer_bad_arguments():
    """None of these reaches a device: 0 bytes, or LM_B200_EINVAL."""
    lib = _lm_lib.load()
    at, odd = 1 << 20, (1 << 20) + 8                               # (addresses that are never followed)
    cache = dict(zip([n for n, _ in _lm_lib.Kv8._fields_], (at, at, at, at, 4, 2, 16, 64, _lm_lib.KV8_E4M3)))
    step = (at, 3000, at, at, 3000, 2, 5)
    need = lib.lm_b200_op_kv8_attention_work_bytes(2, 64, 5, 4, _lm_lib.TYPE_BF16, 2, 48000)
    assert need > 0 and lib.lm_b200_op_kv8_attention_work_bytes(2, 64, 5, 4, _lm_lib.TYPE_BF16, 2, 48) == 0 and lib.lm_b200_op_kv8_attention_work_bytes(2, 64, 500, 4, _lm_lib.TYPE_BF16, 2, 48) > need
    for a in ((0, 64, 5, 4, 1, 2), (2, 0, 5, 4, 1, 2), (2, 257, 5, 4, 1, 2), (2, 64, 0, 4, 1, 2), (2, 64, 5, 0, 1, 2), (2, 64, 5, 5, 1, 2), (2, 64, 1 << 30, 4, 1, 2), (1, 64, 5, 4097, 1, 2),
              (2, 64, 5, 4, 7, 2), (2, 64, 5, 4, 1, 0)):
        assert lib.lm_b200_op_kv8_attention_work_bytes(*a, 48000) == 0

    def entries(cache, step, rows=(at, 128, 64), heads=4, kind=1, scale=1.0, window=0, out=at, work=at, bytes=need):
        k = _lm_lib.Kv8(*cache.values()) if cache else None
        where, what = C.addressof(k) if k else None, lm_ops._KV8_STEP.pack(*step) if step else None
        yield "append", lambda: lib.lm_b200_op_kv8_append(where, what, *rows, *rows, kind, None)
        yield "read", lambda: lib.lm_b200_op_kv8_read(where, what, rows[0], out, kind, None)
        yield "attention", lambda: lib.lm_b200_op_kv8_attention(where, what, *rows, heads, kind, scale, window, None, out, work, bytes, None)

    def refused(*names, cache=cache, step=step, **k):
        for name, call in entries(cache, step, **k):
            if name in names:
                assert call() == _lm_lib.E_INVAL, (name, k)

    every = ("append", "read", "attention")
    refused(*every, cache=None)
    refused(*every, step=None)
    for name, bad in (("keys", None), ("keys", odd), ("values", None), ("values", odd), ("key_scales", None), ("value_scales", None), ("pages", 0), ("pages", -1), ("kv_heads", 0),
                      ("kv_heads", 4097), ("page_size", 0), ("page_size", 8), ("page_size", 48), ("page_size", 256), ("dim", 0), ("dim", 257), ("format", 2), ("format", -1)):
        assert name in cache
        refused(*every, cache=cache | {name: bad})
    for i, bad in ((0, 0), (1, -1), (2, 0), (4, 0), (4, -1), (5, 0), (5, -1), (6, 0), (6, -1), (6, 0x7fffffff), (3, 0)):       # (without first: 5 rows of 2 sequences)
        refused(*every, step=step[:i] + (bad,) + step[i + 1:])
    for rows in ((None, 128, 64), (at, -1, 64), (at, 128, -1)):
        refused("append", "attention", rows=rows)
    refused(*every, kind=7)
    refused("read", "attention", out=None)
    refused("read", rows=(None, 0, 0))
    for k in (dict(heads=0), dict(heads=5), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(window=-1), dict(work=None), dict(work=at + 64), dict(bytes=need - 1)):
        refused("attention", **k)


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad
    c, q, k, v, table, past, first = operands()
    with forward_ad.dual_level():
        lift = lambda x: forward_ad.make_dual(x.contiguous(), torch.ones_like(x))              # noqa: E731
        for call in (lambda: c.append(lift(k), v, table, past, first), lambda: c.append(k, lift(v), table, past, first), lambda: lm_ops.attention_kv8(lift(q), c, table, past, first)):
            with pytest.raises((ValueError, NotImplementedError, RuntimeError), match="tangent"):
                call()
