"""Operators of the language models for callers that hold rows of their own: matrices in 4 bits and their products, and the cross
entropy of rows under a head with its gradient.

They stand beside ``lm_engine.linear``: torch tensors on a CUDA device in, new tensors out, queued on the current stream of the tensors'
device.  Workspaces come from torch's allocator for the length of a call, so calls on several streams and in captured graphs do not share
any.  Arguments are checked on the host (``ValueError``, ``TypeError``); there is no CPU fallback.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lm_lib
from .lm_engine import _stream

_TYPES = {torch.float32: _lm_lib.TYPE_FP32, torch.bfloat16: _lm_lib.TYPE_BF16, torch.float16: _lm_lib.TYPE_FP16}


def _check_rows(x: torch.Tensor, name: str, types=tuple(_TYPES)) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if x.dtype not in types:
        raise TypeError(f"{name} must be one of {', '.join(str(t) for t in types)}, not {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must live on a CUDA device (there is no CPU fallback)")


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """``x [..., K]`` as rows with neighbouring channels (a view where the strides allow one)."""
    x = x.reshape(-1, x.shape[-1])
    # (overlapping or backward rows are copied; a row stride is only read where there are several rows)
    return x if (x.shape[1] == 1 or x.stride(1) == 1) and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _no_grad(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient: detach its inputs or call it under torch.no_grad()")


@dataclass(frozen=True)
class Mxfp4:
    """Rows ``[rows, width]`` in microscaled 4-bit numbers: blocks of 32 channels share a power of two (E8M0), elements are E2M1.
    ``codes`` and ``scales`` are uint8 buffers in the kernels' layout."""
    codes: torch.Tensor
    scales: torch.Tensor
    rows: int
    width: int

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows, self.width))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values ``[rows, width]`` that the 4-bit numbers stand for."""
        if dtype not in _TYPES:
            raise TypeError(f"dtype must be one of {', '.join(str(t) for t in _TYPES)}, not {dtype}")
        out = torch.empty((self.rows, self.width), dtype=dtype, device=self.device)
        if out.numel():
            with torch.cuda.device(self.device):
                _lm_lib.check(_lm_lib.load().lm_b200_op_mxfp4_dequantize(self.codes.data_ptr(), self.scales.data_ptr(), self.rows, self.width,
                                                                         out.data_ptr(), _TYPES[dtype], _stream(self.device)), "mxfp4_dequantize")
        return out


def quantize_mxfp4(x: torch.Tensor) -> Mxfp4:
    """``x [rows, width]`` (float32, bfloat16 or float16; rows of any stride) in MXFP4, rounded as the OCP Microscaling specification
    says: a block's scale is ``2 ** (floor(log2(largest magnitude)) - 2)``, at least ``2 ** -127``; elements go to the nearest of 0, 0.5,
    1, 1.5, 2, 3, 4, 6 times the scale, half way to the even code, what lies beyond 6 to 6.  A block with an infinity or a NaN stands
    for NaNs.  The last block of a row may be short."""
    _check_rows(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must have two dimensions, not {x.dim()}")
    _no_grad("quantize_mxfp4", x)
    rows, width = x.shape
    lib = _lm_lib.load()
    codes = torch.empty(lib.lm_b200_mxfp4_code_bytes(rows, width), dtype=torch.uint8, device=x.device)
    scales = torch.empty(lib.lm_b200_mxfp4_scale_bytes(rows, width), dtype=torch.uint8, device=x.device)
    if x.numel():
        x = _as_rows(x)
        with torch.cuda.device(x.device):
            _lm_lib.check(lib.lm_b200_op_mxfp4_quantize(x.data_ptr(), _TYPES[x.dtype], x.stride(0), rows, width, codes.data_ptr(),
                                                        scales.data_ptr(), _stream(x.device)), "mxfp4_quantize")
    return Mxfp4(codes, scales, rows, width)


def linear_mxfp4(a: torch.Tensor, w: Mxfp4, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``a [..., width] @ w [out, width]^T`` with both sides in MXFP4: the rows of ``a`` are rounded on the way (as
    :func:`quantize_mxfp4` does), products are exact and sums float32, and the result has ``a``'s type unless ``out_dtype`` says another.
    For serving: it has no gradient."""
    _check_rows(a, "a")
    if not isinstance(w, Mxfp4):
        raise TypeError("w must be an Mxfp4 (see quantize_mxfp4)")
    if a.dim() < 1 or a.shape[-1] != w.width:
        raise ValueError(f"a has rows of {a.shape[-1] if a.dim() else 0} channels, w of {w.width}")
    if a.device != w.device:
        raise ValueError(f"a lives on {a.device}, w on {w.device}")
    out_dtype = a.dtype if out_dtype is None else out_dtype
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be one of {', '.join(str(t) for t in _TYPES)}, not {out_dtype}")
    _no_grad("linear_mxfp4", a)
    y = torch.empty((*a.shape[:-1], w.rows), dtype=out_dtype, device=a.device)
    if not y.numel():
        return y
    if not w.width:
        return y.zero_()
    lib, rows = _lm_lib.load(), _as_rows(a)
    M = rows.shape[0]
    need = lib.lm_b200_op_linear_mxfp4_work_bytes(M, w.rows, w.width)
    work = torch.empty(need, dtype=torch.uint8, device=a.device)
    with torch.cuda.device(a.device):
        _lm_lib.check(lib.lm_b200_op_linear_mxfp4(rows.data_ptr(), _TYPES[a.dtype], rows.stride(0), w.codes.data_ptr(), w.scales.data_ptr(),
                                                  y.data_ptr(), _TYPES[out_dtype], M, w.rows, w.width, work.data_ptr() if need else None, need,
                                                  _stream(a.device)), "linear_mxfp4")
    return y


def _loss_operands(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor):
    _check_rows(hidden, "hidden", (torch.float32, torch.bfloat16))
    _check_rows(weight, "weight", (torch.bfloat16,))
    if not isinstance(targets, torch.Tensor):
        raise TypeError("targets must be a tensor")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, not {targets.dtype}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not share a width")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not go with hidden {tuple(hidden.shape)}")
    if weight.device != hidden.device or targets.device != hidden.device:
        raise ValueError("hidden, weight and targets must live on one device")
    if not weight.numel():
        raise ValueError("weight is empty")


class _LinearCrossEntropy(torch.autograd.Function):
    """Losses of rows, or (mean, sum) their total; rows are two-dimensional here."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, scale, ignore_index, reduction):
        lib = _lm_lib.load()
        (M, K), V, device = hidden.shape, weight.shape[0], hidden.device
        loss = torch.empty(M, dtype=torch.float32, device=device) if reduction == "none" else None
        kept, totals = torch.empty(2 * M, dtype=torch.float32, device=device), torch.empty(3, dtype=torch.float32, device=device)
        h, w, t = _as_rows(hidden), _as_rows(weight), targets.contiguous()
        args = h.data_ptr(), _TYPES[h.dtype], h.stride(0), w.data_ptr(), w.stride(0)
        need = lib.lm_b200_op_loss_work_bytes(*args, M, V, K)
        work = torch.empty(need, dtype=torch.uint8, device=device)
        with torch.cuda.device(device):
            _lm_lib.check(lib.lm_b200_op_loss(*args, t.data_ptr(), t.dtype == torch.int64, ignore_index, M, V, K, scale,
                                              None if loss is None else loss.data_ptr(), kept.data_ptr(), totals.data_ptr(), work.data_ptr(), need, _stream(device)), "loss")
        ctx.save_for_backward(hidden, weight, t, kept)
        # (the count stands beside the result, which may be changed in place: not a saved tensor)
        ctx.args = scale, ignore_index, totals[1:2].detach() if reduction == "mean" else None
        return loss if reduction == "none" else totals[2 if reduction == "mean" else 0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, t, kept = ctx.saved_tensors
        scale, ignore_index, count = ctx.args
        need_h, need_w = ctx.needs_input_grad[:2]
        if hidden.dtype != torch.bfloat16:
            raise TypeError("gradients need hidden in bfloat16")
        lib = _lm_lib.load()
        (M, K), V, device = hidden.shape, weight.shape[0], hidden.device
        h, w, grad = _as_rows(hidden), _as_rows(weight), grad.to(torch.float32)
        if grad.dim() and grad.stride(0) < 0:
            grad = grad.contiguous()
        dh = torch.empty((M, K), dtype=hidden.dtype, device=device) if need_h else None
        dw = torch.empty((V, K), dtype=weight.dtype, device=device) if need_w else None
        args = h.data_ptr(), h.stride(0), w.data_ptr(), w.stride(0)
        need = lib.lm_b200_op_loss_grad_work_bytes(*args, M, V, K, need_h, need_w)
        work = torch.empty(need, dtype=torch.uint8, device=device)
        with torch.cuda.device(device):
            _lm_lib.check(lib.lm_b200_op_loss_grad(
                *args, t.data_ptr(), t.dtype == torch.int64, ignore_index, M, V, K, scale, kept.data_ptr(), grad.data_ptr(),
                grad.stride(0) if grad.dim() else 0, count.data_ptr() if count is not None else None,
                dh.data_ptr() if need_h else None, dw.data_ptr() if need_w else None, work.data_ptr(), need, _stream(device)), "loss_grad")
        return dh, dw, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, scale: float = 1.0,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """The cross entropy of ``targets [...]`` under the logits ``scale * hidden [..., width] @ weight [vocab, width]^T``, float32, without
    the logits in memory: ``"none"`` every token's loss, ``"sum"`` or ``"mean"`` over the tokens whose target is not ``ignore_index`` (0
    where there is none).  A token that does not count has loss 0; one whose target is neither ``ignore_index`` nor in ``[0, vocab)`` NaN.

    ``weight`` is bfloat16; ``hidden`` is bfloat16, or float32, which is then multiplied as it is (24 bits) and has no gradient.  The
    gradients by ``hidden`` and ``weight`` take the vocabulary in pieces; rows that do not count have no part in them, whatever they hold.
    """
    _loss_operands(hidden, weight, targets)
    if reduction not in ("none", "sum", "mean"):
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    scale, ignore_index = float(scale), int(ignore_index)
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    if hidden.dtype == torch.float32 and torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        raise ValueError("gradients need hidden in bfloat16")
    if not targets.numel():
        rows = hidden.new_zeros(targets.shape, dtype=torch.float32)
        return rows if reduction == "none" else rows.sum()
    K = hidden.shape[-1]
    loss = _LinearCrossEntropy.apply(hidden.reshape(-1, K), weight, targets.reshape(-1), scale, ignore_index, reduction)
    return loss.view(targets.shape) if reduction == "none" else loss
