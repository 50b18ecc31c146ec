"""Operators of the language models for callers that hold rows of their own: matrices in 4 bits and their products, the cross
entropy of rows under a head with its gradient, and a cache of keys and values in 8 bits with its attention.

They stand beside ``lm_engine.linear``: torch tensors on a CUDA device in, new tensors out, queued on the current stream of the tensors'
device.  Workspaces come from torch's allocator for the length of a call, so calls on several streams and in captured graphs do not share
any.  Arguments are checked on the host (``ValueError``, ``TypeError``); there is no CPU fallback, and forward-mode tangents are refused.
"""

from __future__ import annotations

import ctypes as C
import struct
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _lm_lib

_TYPES = {torch.float32: _lm_lib.TYPE_FP32, torch.bfloat16: _lm_lib.TYPE_BF16, torch.float16: _lm_lib.TYPE_FP16}


def _names(types) -> str:
    return ", ".join(str(t) for t in types)


def _check_rows(x: torch.Tensor, name: str, types=_TYPES) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if x.dtype not in types:
        raise TypeError(f"{name} must be one of {_names(types)}, not {x.dtype}")


def _check_device(device: torch.device, *others: torch.Tensor) -> None:
    for t in others:
        if t.device != device:
            raise ValueError(f"operands live on {device} and {t.device}: they must live on one device")
    if device.type != "cuda":
        raise ValueError(f"operands must live on a CUDA device, not {device} (there is no CPU fallback)")


@lru_cache(maxsize=None)
def _function(what: str):
    return getattr(_lm_lib.load(), "lm_b200_op_" + what)


def _call(what: str, device: torch.device, *args) -> None:
    """The library's function ``lm_b200_op_<what>`` on the device's current stream, as its last argument."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)             # (an integer; a Stream object takes 2 us more)
    if torch._C._cuda_getDevice() == index:
        rc = _function(what)(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = _function(what)(*args, stream)
    if rc:
        _lm_lib.check(rc, what)


# Bytes of a call's workspace go by its sizes and by whether its operands can be read where they are, which the library decides; the answers
# are kept (asking takes the host 1 to 2 us).  Of an address only the alignment counts.
@lru_cache(maxsize=1024)
def _linear_work_bytes(m: int, n: int, k: int) -> int:
    return _lm_lib.load().lm_b200_op_linear_mxfp4_work_bytes(m, n, k)


@lru_cache(maxsize=1024)
def _loss_work_bytes(h_at: int, h_type: int, ldh: int, w_at: int, ldw: int, m: int, v: int, k: int) -> int:
    return _lm_lib.load().lm_b200_op_loss_work_bytes(h_at | 4096, h_type, ldh, w_at | 4096, ldw, m, v, k)


@lru_cache(maxsize=1024)
def _loss_grad_work_bytes(h_at: int, ldh: int, w_at: int, ldw: int, m: int, v: int, k: int, rows: bool, head: bool) -> int:
    return _lm_lib.load().lm_b200_op_loss_grad_work_bytes(h_at | 4096, ldh, w_at | 4096, ldw, m, v, k, rows, head)


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """``x [..., K]`` as rows with neighbouring channels (a view where the strides allow one)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    rows, width = x.shape
    if rows > 0x7fffff00 // 3 or width > 1 << 24:
        raise ValueError(f"{rows} rows of {width} channels are more than an operator takes")
    apart, step = x.stride()
    # (overlapping or backward rows are copied; a row stride is only read where there are several rows)
    return x if (width == 1 or step == 1) and (rows <= 1 or apart >= width) else x.contiguous()


def _no_tangent(what: str, *xs: torch.Tensor) -> None:
    if forward_ad._current_level < 0:                              # (nothing has a tangent outside of a forward-mode level; asking takes 1 us)
        return
    for x in xs:
        if forward_ad.unpack_dual(x).tangent is not None:
            raise ValueError(f"{what} takes no forward-mode tangents")


def _no_grad(what: str, x: torch.Tensor) -> None:
    _no_tangent(what, x)
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} has no gradient: detach its operands or call it under torch.no_grad()")


class Mxfp4:
    """Rows ``[rows, width]`` in microscaled 4-bit numbers: blocks of 32 channels share a power of two (E8M0), elements are E2M1.
    ``data`` holds the codes and, from ``scales_at`` on, the scales, both as the kernels read them (4.25 bits a channel)."""
    __slots__ = ("data", "rows", "width", "scales_at")

    def __init__(self, rows: int, width: int, device: torch.device):
        """Room for so many rows (their numbers are not set; see :func:`quantize_mxfp4`)."""
        stride = (width + 127) // 128 * 128
        self.rows, self.width = rows, width
        self.scales_at = (rows * (stride // 2) + 127) // 128 * 128
        self.data = torch.empty(self.scales_at + (rows + 127) // 128 * (stride // 128) * 512, dtype=torch.uint8, device=device)

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows, self.width))

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values ``[rows, width]`` that the 4-bit numbers stand for."""
        if dtype not in _TYPES:
            raise TypeError(f"dtype must be one of {_names(_TYPES)}, not {dtype}")
        device = self.data.device
        out = torch.empty((self.rows, self.width), dtype=dtype, device=device)
        if self.rows and self.width:
            at = self.data.data_ptr()
            _call("mxfp4_dequantize", device, at, at + self.scales_at, self.rows, self.width, out.data_ptr(), _TYPES[dtype])
        return out


def quantize_mxfp4(x: torch.Tensor) -> Mxfp4:
    """``x [rows, width]`` (float32, bfloat16 or float16; rows of any stride) in MXFP4, rounded as the OCP Microscaling specification
    says: a block's scale is ``2 ** (floor(log2(largest magnitude)) - 2)``, at least ``2 ** -127``; elements go to the nearest of 0, 0.5,
    1, 1.5, 2, 3, 4, 6 times the scale, half way to the even code, what lies beyond 6 to 6.  A block with an infinity or a NaN stands
    for NaNs.  The last block of a row may be short.  It has no gradient."""
    _check_rows(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must have two dimensions, not {x.dim()}")
    _no_grad("quantize_mxfp4", x)
    _check_device(x.device)
    x = _as_rows(x)
    (rows, width), device = x.shape, x.device
    q = Mxfp4(rows, width, device)
    if rows and width:
        at = q.data.data_ptr()
        _call("mxfp4_quantize", device, x.data_ptr(), _TYPES[x.dtype], x.stride(0), rows, width, at, at + q.scales_at)
    return q


def linear_mxfp4(a: torch.Tensor, w: Mxfp4, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``a [..., width] @ w [out, width]^T`` with both sides in MXFP4: the rows of ``a`` are rounded on the way (as
    :func:`quantize_mxfp4` does), products are exact and sums float32 (a tensor core's, which cuts off up to ``2 ** -23`` of a sum at every
    64 channels), and the result has ``a``'s type unless ``out_dtype`` says another.  For serving: it has no gradient."""
    _check_rows(a, "a")
    if not isinstance(w, Mxfp4):
        raise TypeError("w must be an Mxfp4 (see quantize_mxfp4)")
    if not a.dim() or a.shape[-1] != w.width:
        raise ValueError(f"a has rows of {a.shape[-1] if a.dim() else 0} channels, w of {w.width}")
    device = a.device
    if out_dtype is None:
        out_dtype = a.dtype
    elif out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be one of {_names(_TYPES)}, not {out_dtype}")
    _no_grad("linear_mxfp4", a)
    _check_device(device, w.data)
    y = a.new_empty((*a.shape[:-1], w.rows), dtype=out_dtype)
    if not w.width:
        return y.zero_()
    if not y.numel():
        return y
    rows = _as_rows(a)
    M, at = rows.shape[0], w.data.data_ptr()
    need = _linear_work_bytes(M, w.rows, w.width)
    work = a.new_empty(need, dtype=torch.uint8) if need else None
    _call("linear_mxfp4", device, rows.data_ptr(), _TYPES[a.dtype], rows.stride(0), at, at + w.scales_at, y.data_ptr(), _TYPES[out_dtype], M,
          w.rows, w.width, work.data_ptr() if need else None, need)
    return y


def _loss_operands(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor):
    _check_rows(hidden, "hidden", (torch.float32, torch.bfloat16))
    _check_rows(weight, "weight", (torch.bfloat16,))
    if not isinstance(targets, torch.Tensor):
        raise TypeError("targets must be a tensor")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, not {targets.dtype}")
    if not hidden.dim() or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not share a width")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not go with hidden {tuple(hidden.shape)}")
    if not weight.numel():
        raise ValueError("weight is empty")


def _laid_out(x: torch.Tensor) -> torch.Tensor:
    """bfloat16 rows as the loss's kernels read them where they are: themselves, or a copy with rows of whole 16 bytes (zeros behind the
    last channel), for operands that a forward and a backward pass read."""
    (rows, width), device = x.shape, x.device
    if x.dtype != torch.bfloat16 or not (x.data_ptr() & 15 or (x.stride(0) if rows > 1 else width) & 7):
        return x
    out = x.new_empty((rows, (width + 7) // 8 * 8))
    _call("loss_lay_out", device, x.data_ptr(), x.stride(0), rows, width, out.data_ptr())
    return out


_REDUCTIONS = {"none": _lm_lib.LOSS_EACH, "sum": _lm_lib.LOSS_SUM, "mean": _lm_lib.LOSS_MEAN}


def _losses(hidden, weight, targets, scale, ignore_index, reduction, keep):
    """(losses or their sum or mean, what the gradient needs).  The latter, with ``keep``: hidden, weight and targets as they were read, and
    [log-sum, loss] of every row and how many rows count."""
    h, w, t = _as_rows(hidden), _as_rows(weight), targets.contiguous()
    (M, K), V, device = h.shape, w.shape[0], h.device
    if keep:
        h, w = _laid_out(h), _laid_out(w)
    out = h.new_empty(M if reduction == "none" else (), dtype=torch.float32)
    kept = h.new_empty(2 * M + 1, dtype=torch.float32) if keep else None
    h_at, w_at, h_type, ldh, ldw = h.data_ptr(), w.data_ptr(), _TYPES[h.dtype], h.stride(0), w.stride(0)
    need = _loss_work_bytes(h_at & 255, h_type, ldh, w_at & 255, ldw, M, V, K)
    work = h.new_empty(need, dtype=torch.uint8)
    _call("loss", device, h_at, h_type, ldh, w_at, ldw, t.data_ptr(), t.dtype == torch.int64, ignore_index, M, V, K, scale,
          _REDUCTIONS[reduction], out.data_ptr(), kept.data_ptr() if keep else None, work.data_ptr(), need)
    return out, (h, w, t, kept)


class _OnceDifferentiable(torch.autograd.Function):
    """Gradients as they are, of which a further derivative by what they were made of is refused (it would else be taken for zero)."""

    @staticmethod
    def forward(ctx, grad, hidden, weight, *results):
        return tuple(x.view_as(x) for x in results)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("linear_cross_entropy has no second derivative")


class _LinearCrossEntropy(torch.autograd.Function):
    """Losses of rows, or (mean, sum) their total; rows are two-dimensional here."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, scale, ignore_index, reduction):
        out, read = _losses(hidden, weight, targets, scale, ignore_index, reduction, True)
        # (the operands themselves are kept too where they were laid out again: a change of theirs in place shows)
        ctx.save_for_backward(hidden, weight, *read)
        ctx.args = scale, ignore_index, reduction == "mean"
        return out

    @staticmethod
    def backward(ctx, grad):
        hidden, weight, *read = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return *_LinearCrossEntropy.gradients(ctx, grad, hidden, weight, *read), None, None, None, None
        with torch.no_grad():
            got = _LinearCrossEntropy.gradients(ctx, grad, hidden, weight, *read)
        there = iter(_OnceDifferentiable.apply(grad, hidden, weight, *(x for x in got if x is not None)))
        return *(x if x is None else next(there) for x in got), None, None, None, None

    @staticmethod
    def gradients(ctx, grad, hidden, weight, h, w, t, kept):
        scale, ignore_index, mean = ctx.args
        need_h, need_w = ctx.needs_input_grad[:2]
        (M, K), V, device = hidden.shape, weight.shape[0], hidden.device
        if grad.dim() and grad.stride(0) > 0x7fffffff:            # (the library takes strides of 32 bits)
            grad = grad.contiguous()
        dh = hidden.new_empty((M, K)) if need_h else None
        dw = weight.new_empty((V, K)) if need_w else None
        h_at, w_at, ldh, ldw = h.data_ptr(), w.data_ptr(), h.stride(0), w.stride(0)
        need = _loss_grad_work_bytes(h_at & 255, ldh, w_at & 255, ldw, M, V, K, need_h, need_w)
        work = hidden.new_empty(need, dtype=torch.uint8)
        kept_at = kept.data_ptr()
        _call("loss_grad", device, h_at, ldh, w_at, ldw, t.data_ptr(), t.dtype == torch.int64, ignore_index, M, V, K, scale, kept_at,
              grad.data_ptr(), grad.stride(0) if grad.dim() else 0, kept_at + 8 * M if mean else None, dh.data_ptr() if need_h else None,
              dw.data_ptr() if need_w else None, work.data_ptr(), need)
        return dh, dw


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, scale: float = 1.0,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """The cross entropy of ``targets [...]`` under the logits ``scale * hidden [..., width] @ weight [vocab, width]^T``, float32, without
    the logits in memory: ``"none"`` every token's loss, ``"sum"`` or ``"mean"`` over the tokens whose target is not ``ignore_index`` (0
    where there is none).  A token that does not count has loss 0; one whose target is neither ``ignore_index`` nor in ``[0, vocab)`` NaN.

    ``weight`` is bfloat16; ``hidden`` is bfloat16, or float32, which is then multiplied as it is (24 bits) and has no gradient.  The
    gradients by ``hidden`` and ``weight`` take the vocabulary in pieces; rows that do not count have no part in them, whatever they hold.
    There is no second derivative.
    """
    _loss_operands(hidden, weight, targets)
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    scale, ignore_index = float(scale), int(ignore_index)
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:                    # (the kernels hold it, and its product with log2(e), in float32)
        raise ValueError("scale must be positive, from 2 ** -126 to 2 ** 126")
    if not -1 << 63 <= ignore_index < 1 << 63:
        raise ValueError("ignore_index must fit 64 bits")
    with_grad = (hidden.requires_grad or weight.requires_grad) and torch.is_grad_enabled()
    if with_grad and hidden.dtype != torch.bfloat16:
        raise ValueError("gradients need hidden in bfloat16")
    _no_tangent("linear_cross_entropy", hidden, weight)
    _check_device(hidden.device, weight, targets)
    if not targets.numel():                                       # (still a function of both, whose gradients are zeros)
        rows = hidden.float().sum(-1) + weight[:0].float().sum()
        return rows if reduction == "none" else rows.sum()
    rows = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    flat = targets if targets.dim() == 1 else targets.reshape(-1)
    if with_grad:
        loss = _LinearCrossEntropy.apply(rows, weight, flat, scale, ignore_index, reduction)
    else:
        loss = _losses(rows, weight, flat, scale, ignore_index, reduction, False)[0]
    return loss.view(targets.shape) if reduction == "none" and targets.dim() != 1 else loss


_KV8_FORMATS = {"e4m3": _lm_lib.KV8_E4M3, "int8": _lm_lib.KV8_INT8}
_KV8_PAGES = (16, 32, 64, 128)


class Kv8:
    """Keys and values of sequences in pages, 8 bits a number: ``keys`` and ``values`` hold codes ``[pages, kv_heads, page_size, stride]`` (uint8;
    E4M3, or two's complement for ``"int8"``; ``stride`` is ``dim`` padded to 16 with zeros), ``key_scales`` and ``value_scales`` ``[pages, kv_heads]``
    (float32) one power of two for the tokens of a page and head.  A number is its code times that scale.

    Which pages a sequence has is the caller's to keep (``PagedState`` does it for served models): every call takes a ``table [sequences, n]`` of
    page numbers, int32, whose unused places may hold anything.  Together with ``past [sequences]`` and ``first [sequences + 1]`` (int32, on the
    device, so that a captured graph reads them anew) it describes the rows of a step: sequence ``i`` has rows ``first[i]`` to ``first[i + 1]`` of the
    packed ones, at positions ``past[i]`` and on; without ``first``, row ``i`` alone.  ``first`` does not decrease (where it does, calls still end and
    stay within the tensors, but which rows are whose is not said).  A token whose place lies beyond the table, or whose page is not
    in the pool, is not there: it is not written, not seen, and reads as zeros.  A sequence whose ``past`` is negative has no tokens."""
    __slots__ = ("keys", "values", "key_scales", "value_scales", "pages", "kv_heads", "page_size", "dim", "format", "_handle", "_at", "_index")

    def __init__(self, pages: int, kv_heads: int, dim: int, *, page_size: int = 16, format: str = "e4m3", device: torch.device | str = "cuda"):
        """Room for ``pages`` pages (1 <= dim <= 256; page_size 16, 32, 64 or 128), all zeros."""
        if format not in _KV8_FORMATS:
            raise ValueError("format must be 'e4m3' or 'int8'")
        if page_size not in _KV8_PAGES:
            raise ValueError(f"page_size must be one of {', '.join(map(str, _KV8_PAGES))}")
        if not 1 <= dim <= 256:
            raise ValueError("dim must be from 1 to 256")
        if not (1 <= pages < 1 << 31 and 1 <= kv_heads <= 4096):
            raise ValueError("pages and kv_heads must be positive (kv_heads at most 4096)")
        self.pages, self.kv_heads, self.dim, self.page_size, self.format = int(pages), int(kv_heads), int(dim), int(page_size), format
        shape = (self.pages, self.kv_heads, self.page_size, (self.dim + 15) // 16 * 16)
        self.keys, self.values = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
        self.key_scales, self.value_scales = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        self._handle = _lm_lib.Kv8(self.keys.data_ptr(), self.values.data_ptr(), self.key_scales.data_ptr(), self.value_scales.data_ptr(), self.pages,
                                   self.kv_heads, self.page_size, self.dim, _KV8_FORMATS[format])
        self._at, self._index = C.addressof(self._handle), self.keys.get_device()

    def __setattr__(self, name, value):
        if hasattr(self, "_index"):                               # (the handle has their addresses)
            raise AttributeError(f"{name} of a Kv8 stays what it was made with: write into its tensors instead")
        object.__setattr__(self, name, value)

    @property
    def device(self) -> torch.device:
        return self.keys.device

    @property
    def nbytes(self) -> int:
        return 2 * (self.keys.numel() + 4 * self.key_scales.numel())

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, past: torch.Tensor, first: torch.Tensor | None = None) -> None:
        """Writes ``k`` and ``v [rows, kv_heads, dim]`` (float32, bfloat16 or float16; rows and heads of any stride) behind the ``past[i]`` tokens that
        sequence ``i`` holds.  A page's exponent is the smallest, at least -100, for which its largest magnitude so far is at most 448 (``"int8"``: 127)
        times the power; codes go to the nearest, half way to the even one.  Where a page that holds earlier tokens needs a larger exponent, their codes
        are rounded again.  The first token of a page starts it anew, whatever it held.  A number that is not finite makes the page's head stand for NaNs
        until then; finite ones of about 2^128 are read as infinity where that is the nearest number.  No page may be named twice by the places that a call's
        tokens go to."""
        _check_rows(k, "k")
        _check_rows(v, "v")
        shape = k.shape
        if len(shape) != 3 or shape[1] != self.kv_heads or shape[2] != self.dim or v.shape != shape or v.dtype != k.dtype:
            raise ValueError(f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} must be [rows, {self.kv_heads}, {self.dim}] of one type")
        _no_grad("Kv8.append", k)
        _no_grad("Kv8.append", v)
        step = _kv8_step(self, table, past, first, shape[0])
        if not k.get_device() == v.get_device() == self._index >= 0:
            _check_device(self.keys.device, k, v)
        if step is None:
            return
        (k_row, k_head, k_step), (v_row, v_head, v_step) = k.stride(), v.stride()
        if self.dim > 1 and (k_step != 1 or v_step != 1):
            k, v = k.contiguous(), v.contiguous()
            (k_row, k_head, _), (v_row, v_head, _) = k.stride(), v.stride()
        _call("kv8_append", self.keys.device, self._at, step, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head, _TYPES[k.dtype])

    def read(self, table: torch.Tensor, past: torch.Tensor, first: torch.Tensor | None, rows: int, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values ``[rows, kv_heads, dim]`` of the tokens at positions ``past[i]`` and on, as many as ``first`` gives sequence ``i`` rows.  Rows of no
        sequence are zeros."""
        if dtype not in _TYPES:
            raise TypeError(f"dtype must be one of {_names(_TYPES)}, not {dtype}")
        rows = int(rows)
        if rows < 0:
            raise ValueError("rows must not be negative")
        step = _kv8_step(self, table, past, first, rows)
        k = self.key_scales.new_empty((rows, self.kv_heads, self.dim), dtype=dtype)
        v = torch.empty_like(k)
        if step is None:
            return k.zero_(), v.zero_()
        _call("kv8_read", self.keys.device, self._at, step, k.data_ptr(), v.data_ptr(), _TYPES[dtype])
        return k, v


# lm_b200_kv8_step: table, table_ld, past, first, max_pages, n_seq, rows (a ctypes structure takes 1 us more)
_KV8_STEP = struct.Struct("@PqPPiii")


def _check_ints(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, not {t.dtype}")


def _kv8_step(cache: Kv8, table: torch.Tensor, past: torch.Tensor, first: torch.Tensor | None, rows: int) -> bytes | None:
    """The description of a step's rows as the library takes it (None: no row of any sequence)."""
    _check_ints(table, "table")
    _check_ints(past, "past")
    if first is not None:
        _check_ints(first, "first")
    if table.dim() != 2:
        raise ValueError("table must be [sequences, pages of one]")
    (n, width), (apart, step) = table.shape, table.stride()
    if width > 1 and step != 1:
        raise ValueError("table must have a sequence's page numbers beside one another")
    if past.shape != (n,) or not past.is_contiguous():
        raise ValueError(f"past must hold one number for each of {n} sequences")
    index = cache._index
    if first is None:
        if rows != n:
            raise ValueError(f"{rows} rows of {n} sequences need first")
        if not table.get_device() == past.get_device() == index >= 0:
            _check_device(cache.keys.device, table, past)
    else:
        if first.shape != (n + 1,) or not first.is_contiguous():
            raise ValueError(f"first must hold {n + 1} numbers")
        if not table.get_device() == past.get_device() == first.get_device() == index >= 0:
            _check_device(cache.keys.device, table, past, first)
    if rows > 0x7fffff00:
        raise ValueError(f"{rows} rows are more than an operator takes")
    if not (n and rows and width):
        return None
    return _KV8_STEP.pack(table.data_ptr(), apart, past.data_ptr(), 0 if first is None else first.data_ptr(), width, n, rows)


@lru_cache(maxsize=1024)
def _kv8_work_bytes(kv_heads: int, dim: int, rows: int, heads: int, kind: int, n: int, tokens: int) -> int:
    return _lm_lib.load().lm_b200_op_kv8_attention_work_bytes(kv_heads, dim, rows, heads, kind, n, tokens)


def attention_kv8(q: torch.Tensor, cache: Kv8, table: torch.Tensor, past: torch.Tensor, first: torch.Tensor | None = None, *, scale: float | None = None,
                  window: int | None = None, sinks: torch.Tensor | None = None) -> torch.Tensor:
    """Causal grouped-query attention of ``q [rows, heads, dim]`` (float32, bfloat16 or float16; any stride of rows and heads) over the tokens in ``cache``: a row
    sees the tokens at its position and before it, the last ``window`` of them where that is given, so its own have to be there
    (:meth:`Kv8.append` with the same ``table``, ``past`` and ``first``).  Query head ``h`` reads key head ``h // (heads / kv_heads)``; weights are
    ``exp(scale * q . k)``, ``scale`` ``dim ** -0.5`` unless given, and ``sinks [heads]`` (float32) adds ``exp(sinks[h])`` to the denominator.  A row that sees
    nothing, and a row of no sequence, is zeros.

    float32 rows are multiplied with 22 bits, as the language models' attention does; weights are rounded to 22 bits for them, to 11 for the other types (a
    token whose part in a row's result is below 2^-20 of what the largest one's may be, to 2^-31 of that).  Maxima, sums and outputs are float32 until the
    result; of 16-bit prompts the outputs' additions are cut off, not rounded, up to 2^-11 of their sum behind 131072 tokens.  Values in pages whose power is
    2^80 below the largest in a sequence's pages may be taken as zeros.  A row with a number that is not finite is NaN where it sees anything.  Scores are
    float32: a row whose largest number times ``scale``, or that times a page's power, is beyond its range may be NaN.

    It has no gradient: ``q`` or ``sinks`` that want one, or have a tangent, are refused."""
    _check_rows(q, "q")
    if not isinstance(cache, Kv8):
        raise TypeError("cache must be a Kv8")
    shape = q.shape
    if len(shape) != 3 or shape[2] != cache.dim or not shape[1] or shape[1] % cache.kv_heads or shape[1] > 4096:
        raise ValueError(f"q {tuple(shape)} does not go with {cache.kv_heads} key heads of {cache.dim}")
    scale = cache.dim ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:
        raise ValueError("scale must be positive, from 2 ** -126 to 2 ** 126")
    if window is None:
        window = 0
    elif not 1 <= (window := int(window)) < 1 << 31:
        raise ValueError("window must be positive")
    _no_grad("attention_kv8", q)
    rows, heads, _ = shape
    step = _kv8_step(cache, table, past, first, rows)
    if not q.get_device() == cache._index >= 0:
        _check_device(cache.keys.device, q)
    if sinks is not None:
        _check_rows(sinks, "sinks", (torch.float32,))
        if sinks.shape != (heads,):
            raise ValueError(f"sinks must hold one number for each of {heads} heads")
        _no_grad("attention_kv8", sinks)
        _check_device(cache.keys.device, sinks)
        sinks = sinks.contiguous()
    if rows > 0x7fffff00 // heads:
        raise ValueError(f"{rows} rows of {heads} heads are more than an operator takes")
    if step is None:
        return q.new_zeros(shape)
    q_row, q_head, q_step = q.stride()
    if q_step != 1 and cache.dim > 1:
        q = q.contiguous()
        q_row, q_head, _ = q.stride()
    kind = _TYPES[q.dtype]
    n, width = table.shape
    need = _kv8_work_bytes(cache.kv_heads, cache.dim, rows, heads, kind, n, width * cache.page_size)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    work = q.new_empty(need, dtype=torch.uint8) if need else None
    _call("kv8_attention", cache.keys.device, cache._at, step, q.data_ptr(), q_row, q_head, heads, kind, scale, window, None if sinks is None else sinks.data_ptr(),
          out.data_ptr(), work.data_ptr() if need else None, need)
    return out
