"""What the operators of lm_ops refuse, and how their C entries answer what they do not take: without a GPU."""

import ctypes as C
import math

import pytest
import torch

from dia_tts_prune_b200 import _lm_lib, lm_ops


def test_rows_and_matrices_that_are_refused():
    x = torch.randn(4, 64)
    for bad in (x.double(), x.int(), x.to(torch.complex64)):
        with pytest.raises(TypeError):
            lm_ops.quantize_mxfp4(bad)
    with pytest.raises(TypeError):
        lm_ops.quantize_mxfp4([1.0])
    for bad in (x[0], x[None]):
        with pytest.raises(ValueError, match="two dimensions"):
            lm_ops.quantize_mxfp4(bad)
    with pytest.raises(ValueError, match="gradient"):
        lm_ops.quantize_mxfp4(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="CUDA"):
        lm_ops.quantize_mxfp4(x)


def test_products_that_are_refused():
    w = lm_ops.Mxfp4(8, 64, torch.device("cpu"))
    x = torch.randn(4, 64)
    with pytest.raises(TypeError):
        lm_ops.linear_mxfp4(x, torch.randn(8, 64))
    with pytest.raises(TypeError):
        lm_ops.linear_mxfp4(x.long(), w)
    with pytest.raises(TypeError):
        lm_ops.linear_mxfp4(x, w, out_dtype=torch.float64)
    for bad in (x[:, :63], torch.tensor(1.0)):
        with pytest.raises(ValueError, match="channels"):
            lm_ops.linear_mxfp4(bad, w)
    with pytest.raises(ValueError, match="gradient"):
        lm_ops.linear_mxfp4(x.clone().requires_grad_(True), w)
    with pytest.raises(ValueError, match="CUDA"):
        lm_ops.linear_mxfp4(x, w)
    with pytest.raises(TypeError):
        w.dequantize(torch.float64)
    assert w.shape == (8, 64) and w.device.type == "cpu"
    # 8 rows of 128 channels (64 are there) in half a byte each, one piece of 128 x 4 scales
    assert w.nbytes == 8 * 64 + 512 and w.scales_at == 512


def test_losses_that_are_refused():
    h, w, t = torch.randn(6, 32).bfloat16(), torch.randn(10, 32).bfloat16(), torch.zeros(6, dtype=torch.long)
    f = lm_ops.linear_cross_entropy
    for a in ((h.half(), w, t), (h, w.float(), t), (h, w, t.float()), (h, w, t.bool()), (h, w, [0] * 6)):
        with pytest.raises(TypeError):
            f(*a)
    for a in ((h[:, :31], w, t), (h, w[0], t), (h, w, t[:5]), (h, w, t[:, None]), (h, w[:0], t)):
        with pytest.raises(ValueError):
            f(*a)
    for k in (dict(reduction="max"), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(ignore_index=1 << 63)):
        with pytest.raises(ValueError):
            f(h, w, t, **k)
    for a in ((h.float().requires_grad_(True), w, t), (h.float(), w.clone().requires_grad_(True), t)):
        with pytest.raises(ValueError, match="bfloat16"):
            f(*a)
    with pytest.raises(ValueError, match="CUDA"):
        f(h, w, t)
    if torch.cuda.is_available():
        with pytest.raises(ValueError, match="one device"):
            f(h.cuda(), w, t)


def test_c_entries_answer_bad_arguments():
    """None of these reaches a device: 0 bytes, or LM_B200_EINVAL."""
    lib = _lm_lib.load()
    at, odd = 1 << 20, (1 << 20) + 8                               # (addresses that are never followed)
    q = lib.lm_b200_op_mxfp4_quantize
    for a in ((None, 0, 64, 4, 64, at, at), (at, 3, 64, 4, 64, at, at), (at, 0, 63, 4, 64, at, at), (at, 0, 64, 0, 64, at, at), (at, 0, 64, 4, 0, at, at),
              (at, 0, 64, 4, 64, odd, at), (at, 0, 64, 4, 64, at, None), (at, 0, 1 << 30, 4, 1 << 25, at, at),
              (at, 0, 64, 0x7fffffff, 64, at, at)):
        assert q(*a, None) == _lm_lib.E_INVAL
    for a in ((at, at, 0, 64, at, 0), (at, at, 4, 64, None, 0), (at, at, 4, 64, at, 7), (odd, at, 4, 64, at, 0)):
        assert lib.lm_b200_op_mxfp4_dequantize(*a, None) == _lm_lib.E_INVAL
    assert lib.lm_b200_mxfp4_code_bytes(0, 64) == 0 and lib.lm_b200_mxfp4_code_bytes(3, 65) == 3 * 64 and lib.lm_b200_mxfp4_scale_bytes(129, 129) == 2 * 2 * 512
    need = lib.lm_b200_op_linear_mxfp4_work_bytes(200, 64, 64)
    assert need >= 200 * 64 and lib.lm_b200_op_linear_mxfp4_work_bytes(0, 64, 64) == 0
    f = lib.lm_b200_op_linear_mxfp4
    good = [at, 1, 64, at, at, at, 1, 200, 64, 64, at, need]
    for i, bad in ((0, None), (1, 5), (2, 63), (3, None), (3, odd), (4, None), (5, None), (6, -1), (7, 0), (8, 0), (9, 0), (10, None), (10, at + 64), (11, need - 1)):
        a = list(good)
        a[i] = bad
        assert f(*a, None) == _lm_lib.E_INVAL, i
    need = lib.lm_b200_op_loss_grad_work_bytes(at, 64, at, 64, 100, 300, 64, 1, 1)
    assert need > 0 and lib.lm_b200_op_loss_grad_work_bytes(at, 63, at, 64, 100, 300, 64, 1, 1) == 0
    f = lib.lm_b200_op_loss_grad
    good = [at, 64, at, 64, at, 1, -100, 100, 300, 64, 1.0, at, at, 0, None, at, at, at, need]
    for i, bad in ((0, None), (1, 63), (2, None), (3, 63), (4, None), (7, 0), (8, 0), (9, 0), (10, 0.0), (10, math.nan), (10, math.inf), (11, None), (12, None), (13, -1),
                   (17, None), (17, at + 128), (18, need - 1)):
        a = list(good)
        a[i] = bad
        assert f(*a, None) == _lm_lib.E_INVAL, i
    a = list(good)
    a[15] = a[16] = None
    assert f(*a, None) == _lm_lib.E_INVAL
    f = lib.lm_b200_op_loss
    good = [at, 1, 64, at, 64, at, 1, -100, 100, 300, 64, 1.0, 2, at, at, at, 1 << 30]
    for i, bad in ((0, None), (1, 2), (2, 63), (3, None), (4, 63), (5, None), (8, 0), (9, 0), (10, 0), (11, -1.0), (12, 3), (12, -1), (13, None), (15, None), (15, at + 8), (16, 0)):
        a = list(good)
        a[i] = bad
        assert f(*a, None) == _lm_lib.E_INVAL, i
    assert lib.lm_b200_forward_hidden(None, at, 1, 1, 1, at, None) == _lm_lib.E_INVAL


def test_a_head_is_there_once():
    """engine_create: a head, or codes with their scales"""
    lib, out = _lm_lib.load(), C.c_void_p()
    for codes, scales in ((None, None), (1 << 20, None), (None, 1 << 20), ((1 << 20) + 4, 1 << 20)):
        m = _lm_lib.Model(n_layer=1, width=8, vocab=8, page_size=4, max_pages=1, n_slots=1, max_rows=1, embed=1 << 20, page_table=1 << 20)
        m.final_norm.w = m.final_norm.b = 1 << 20
        m.head_codes, m.head_scales = codes, scales
        m.head = 1 << 20 if scales and not codes else None
        assert lib.lm_b200_engine_create(C.byref(m), (_lm_lib.Layer * 1)(), 0, C.byref(out)) == _lm_lib.E_INVAL


def test_score_command_parses():
    from dia_tts_prune_b200.__main__ import main
    with pytest.raises(SystemExit):
        main(["score", "--model", "x"])
    with pytest.raises(SystemExit):
        main(["generate", "--model", "x", "--prompt", "1", "--head-format", "int4"])


def test_forward_mode_tangents_are_refused():
    """They would be lost: the operators' results are new tensors."""
    from torch.autograd import forward_ad
    x, h, w = torch.randn(4, 64), torch.randn(4, 64).bfloat16(), torch.randn(10, 64).bfloat16()
    q, t = lm_ops.Mxfp4(8, 64, torch.device("cpu")), torch.zeros(4, dtype=torch.long)
    calls = [lambda a: lm_ops.quantize_mxfp4(a(x)), lambda a: lm_ops.linear_mxfp4(a(x), q), lambda a: lm_ops.linear_cross_entropy(a(h), w, t),
             lambda a: lm_ops.linear_cross_entropy(h, a(w), t), lambda a: lm_ops.linear_cross_entropy(a(h[:0]), w, t[:0])]
    with forward_ad.dual_level():
        for call in calls:
            with pytest.raises(ValueError, match="tangent"):
                call(lambda v: forward_ad.make_dual(v, torch.ones_like(v)))
            with pytest.raises(ValueError, match="CUDA"):          # (without one inside a level)
                call(lambda v: v)
    for call, v in zip(calls[:3], (x, x, h)):
        with pytest.raises(ValueError, match="tangent"):
            torch.func.jvp(lambda u: call(lambda _: u), (v,), (torch.ones_like(v),))


def test_score_command_prints_json_whatever_the_scores(monkeypatch, capsys):
    """One object per text: null for what is not a finite number and for a perplexity beyond float64's largest; texts behind it are still there."""
    import json

    from dia_tts_prune_b200 import __main__, registry

    class Model:
        def score(self, texts):
            return [[-1.0, -2.0], [-900.0], [math.nan, -1.0], [-math.inf, -1.0], [], [-math.inf, math.inf], [-0.5]]

    monkeypatch.setattr(registry, "load_model", lambda *a, **k: Model())
    assert __main__.main(["score", "--model", "x"] + ["--tokens", "1 2"] * 7) == 0

    def refuse(name):
        raise AssertionError(f"{name} is not JSON")

    got = [json.loads(line, parse_constant=refuse) for line in capsys.readouterr().out.strip().splitlines()]
    assert [g["tokens"] for g in got] == [2, 1, 2, 2, 0, 2, 1]
    assert [g["logprob"] for g in got] == [-3.0, -900.0, None, None, 0, None, -0.5]
    assert [g["logprobs"] for g in got] == [[-1.0, -2.0], [-900.0], [None, -1.0], [None, -1.0], [], [None, None], [-0.5]]
    assert [g["perplexity"] for g in got] == [math.exp(1.5), None, None, None, None, None, math.exp(0.5)]


def test_scales_that_float32_does_not_hold_are_refused():
    """By the operator and by the C entries: too small, too large, or finite but not so times log2(e)."""
    lib, at = _lm_lib.load(), 1 << 20
    h, w, t = torch.randn(6, 32).bfloat16(), torch.randn(10, 32).bfloat16(), torch.zeros(6, dtype=torch.long)
    loss = [at, 1, 64, at, 64, at, 1, -100, 100, 300, 64, 1.0, 2, at, at, None, 1 << 30]
    grad = [at, 64, at, 64, at, 1, -100, 100, 300, 64, 1.0, at, at, 0, None, at, at, None, 1 << 30]
    for scale in (1e-46, 2.0 ** -127, 2.0 ** 127, 3e38, 1e39, 1e300):
        with pytest.raises(ValueError, match="scale"):
            lm_ops.linear_cross_entropy(h, w, t, scale=scale)
        loss[11] = grad[10] = scale
        assert lib.lm_b200_op_loss(*loss, None) == lib.lm_b200_op_loss_grad(*grad, None) == _lm_lib.E_INVAL
    for scale in (2.0 ** -126, 2.0 ** 126):
        with pytest.raises(ValueError, match="CUDA"):
            lm_ops.linear_cross_entropy(h, w, t, scale=scale)


def test_pairs_of_numbers_that_lie_askew_are_refused():
    """What a loss keeps for its gradient is written and read two numbers at a time."""
    lib, at = _lm_lib.load(), 1 << 20
    loss = [at, 1, 64, at, 64, at, 1, -100, 100, 300, 64, 1.0, 2, at, at + 4, at, 1 << 30]
    grad = [at, 64, at, 64, at, 1, -100, 100, 300, 64, 1.0, at + 4, at, 0, None, at, at, at, 1 << 30]
    assert lib.lm_b200_op_loss(*loss, None) == lib.lm_b200_op_loss_grad(*grad, None) == _lm_lib.E_INVAL


def test_commands_and_loaders_of_an_application(tmp_path, monkeypatch, capsys):
    """A loader registered by an application, without a word of heads: the commands serve its model; a format that it does not know is its to refuse."""
    from dia_tts_prune_b200 import __main__, registry

    class Model:
        def generate(self, prompts, **k):
            return [[1, 2] for _ in prompts]

        def run_step(self):
            pass

        def score(self, texts):
            return [[-1.0] for _ in texts]

    registry.architectures()                                       # (the built-in ones are registered first)
    monkeypatch.setattr(registry, "_LOADERS", dict(registry._LOADERS))
    registry.register("Mine", lambda folder, dtype, device=None, max_tokens=0: Model())
    (tmp_path / "config.json").write_text('{"architecture": "Mine"}')
    assert __main__.main(["generate", "--model", str(tmp_path), "--prompt", "1 2"]) == 0
    assert __main__.main(["score", "--model", str(tmp_path), "--tokens", "1 2"]) == 0
    with pytest.raises(TypeError):
        __main__.main(["score", "--model", str(tmp_path), "--tokens", "1 2", "--head-format", "mxfp4"])
