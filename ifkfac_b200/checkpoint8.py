"""Activations held in 8 bits, the products that read them, and layer norm.

The rows that a training step keeps for later (a Linear layer's input for its
weight gradient and for the Kronecker factor, a layer norm's input for its
backward pass) can be held as :class:`Q8Rows`: one byte an element and one a
group of 32 columns, in the format of ``include/ifk.h`` (a power-of-two scale a
group and integer codes, so every value is exact in bf16 and fp32).

* :func:`quantize_rows` / :func:`dequantize_rows`: rows to 8 bits and back,
  optionally a gather of rows (the hooks' random row subsample);
* :func:`weight_grad`: dW = delta^T X and db from the 8-bit rows of X;
* :func:`layer_norm_forward` / :func:`layer_norm_backward`: layer norm with its
  weight and bias gradients, from the saved input or its 8-bit rows;
* :class:`Linear8`, :class:`LayerNorm8`: ``nn.Linear`` / ``nn.LayerNorm`` that
  save their input in 8 bits for the backward pass, and :func:`convert`, which
  puts them in the place of a model's own.

``RawActivationHooks(capture_8bit=True)`` (and ``IFKFAC``) keeps its pending rows
this way; next to a :class:`Linear8` it shares that layer's rows.

Everything runs in libifk.so on CUDA tensors (fp32 or bf16); there is no CPU path.
"""
from __future__ import annotations

import weakref
from functools import lru_cache
from typing import Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from ._lib import IFKError

__all__ = ["Q8Rows", "quantize_rows", "dequantize_rows", "weight_grad", "LayerNormSaved", "layer_norm_forward",
           "layer_norm_backward", "Linear8", "LayerNorm8", "convert"]

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_G = _lib.Q8_GROUP


def _code(dtype: torch.dtype) -> int:
    try:
        return _DT[dtype]
    except KeyError:
        raise TypeError(f"ifkfac_b200 supports float32 and bfloat16 tensors, got {dtype}") from None


def _need_cuda(*ts: Optional[torch.Tensor]) -> int:
    """The index of the one CUDA device of the tensors (None entries are skipped)."""
    dev = -2
    for t in ts:
        if t is not None:
            i = t.get_device()
            if i != dev:
                if i < 0:
                    raise ValueError("ifkfac_b200 operates on CUDA tensors only (no CPU path)")
                if dev >= 0:
                    raise ValueError(f"tensors on devices {dev} and {i}: one call works on one device")
                dev = i
    return dev


def _call(name: str, dev: int, *args) -> None:
    """A library call on the current stream of device ``dev``, which is made current for it."""
    fn = getattr(_lib.lib(), name)
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        raise IFKError(rc, name)


@lru_cache(maxsize=1024)
def _workspace(name: str, *sizes: int) -> int:
    """Bytes that the library's ``name`` asks for (they depend on the sizes alone)."""
    return getattr(_lib.lib(), name)(*sizes)


def _rows2d(t: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """(t, rows, columns, leading dimension) of row-major rows with unit column stride; a
    tensor of any other layout is copied.  A single row's stride is not used."""
    if t.dim() != 2:
        raise ValueError(f"{what} must be 2-D rows, got shape {tuple(t.shape)}")
    rows, cols = t.shape
    if cols == 0:
        raise ValueError(f"{what} has no columns")
    ld, unit = t.stride()
    if (unit != 1 and cols > 1) or (ld < cols and rows > 1):
        t, ld = t.contiguous(), cols
    return t, rows, cols, max(ld, cols)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _status(t: Optional[torch.Tensor]):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.numel() != 1:
        raise TypeError(f"status is one int32 on the device, got {t.numel()} of {t.dtype}")
    return t.data_ptr()


class Q8Rows:
    """Rows in 8 bits: ``codes`` (rows x pitch int8, pitch = ``cols`` rounded up to a
    multiple of 32), ``scales`` (rows x pitch / 32 uint8).  Slices along the rows are
    views of the same storage.

    Rows made here keep codes and scales in one uint8 buffer, ``data`` (from byte
    ``start`` on the codes of all rows, then the scales)."""

    __slots__ = ("rows", "cols", "data", "start", "_codes", "_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        cols = int(cols)
        pitch = -(-cols // _G) * _G
        rows = codes.shape[0] if codes.dim() == 2 else -1
        if cols < 1 or codes.shape != (rows, pitch) or scales.shape != (rows, pitch // _G):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not rows of {cols} "
                             f"columns (rows x {pitch} and rows x {pitch // _G})")
        if codes.dtype != torch.int8 or scales.dtype != torch.uint8:
            raise TypeError(f"8-bit rows are int8 codes and uint8 scales, got {codes.dtype} and {scales.dtype}")
        (ldc, uc), (lds, us) = codes.stride(), scales.stride()
        if rows > 1 and (ldc < pitch or lds < pitch // _G) or uc != 1 or (us != 1 and pitch > _G):
            raise ValueError("codes and scales must be row-major")
        self.rows, self.cols, self.data, self.start, self._codes, self._scales = rows, cols, None, 0, codes, scales

    @classmethod
    def empty(cls, rows: int, cols: int, device) -> "Q8Rows":
        return cls.of(torch.empty(cls.size(rows, cols), dtype=torch.uint8, device=device), rows, cols)

    @staticmethod
    def size(rows: int, cols: int) -> int:
        """Bytes of the rows in one buffer."""
        groups = -(-cols // _G)
        return rows * groups * (_G + 1)

    @classmethod
    def of(cls, data: torch.Tensor, rows: int, cols: int, start: int = 0) -> "Q8Rows":
        """The rows in a buffer laid out as ``data`` (``start`` a multiple of 16)."""
        q = cls.__new__(cls)
        q.rows, q.cols, q.data, q.start, q._codes, q._scales = rows, cols, data, start, None, None
        return q

    def _split(self) -> None:
        groups = -(-self.cols // _G)
        mid = self.start + self.rows * groups * _G
        self._codes = self.data[self.start: mid].view(torch.int8).view(self.rows, groups * _G)
        self._scales = self.data[mid: mid + self.rows * groups].view(self.rows, groups)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._split()
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._split()
        return self._scales

    @property
    def device(self) -> torch.device:
        return (self._codes if self.data is None else self.data).device

    @property
    def nbytes(self) -> int:
        return self.size(self.rows, self.cols)

    def tensors(self) -> Tuple[torch.Tensor, ...]:
        """The tensors that hold the rows."""
        return (self._codes, self._scales) if self.data is None else (self.data,)

    def args(self) -> Tuple[int, int, int, int]:
        """(codes, ld, scales, ld) of a library call."""
        groups = -(-self.cols // _G)
        pitch = groups * _G
        if self.data is not None:
            p = self.data.data_ptr() + self.start
            return p, pitch, p + self.rows * pitch, groups
        c, s = self._codes, self._scales
        return c.data_ptr(), max(c.stride(0), pitch), s.data_ptr(), max(s.stride(0), groups)

    def __getitem__(self, rows: slice) -> "Q8Rows":
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("8-bit rows are sliced along the rows, with step 1")
        return Q8Rows(self.codes[rows], self.scales[rows], self.cols)

    def __repr__(self) -> str:
        return f"Q8Rows({self.rows} x {self.cols}, {self.device})"


def _index(index: torch.Tensor, dev: int) -> torch.Tensor:
    if index.dim() != 1 or index.dtype not in (torch.int64, torch.int32):
        raise ValueError("a row index is a 1-D integer tensor")
    return index.to(device=torch.device("cuda", dev), dtype=torch.int64).contiguous()


def quantize_rows(x: torch.Tensor, index: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> Q8Rows:
    """The 8-bit rows of ``x`` (rows x cols, fp32 or bf16), or of its rows ``index``.

    Per group of 32 columns with largest magnitude a, the error is at most a / 64; a
    group that holds a NaN or an infinity reads back as NaN.  An index outside x
    gives a zero row and IFK_ERR_ARG in ``status`` (a device int32, optional)."""
    dev = _need_cuda(x, status)
    x, src, cols, ld = _rows2d(x, "x")
    dt = _code(x.dtype)
    rows = src
    if index is not None:
        index = _index(index, dev)
        rows = index.numel()
    q = Q8Rows.empty(rows, cols, dev)
    _call("ifk_q8_quantize", dev, x.data_ptr(), ld, dt, _ptr(index), src, rows, cols, *q.args(), _status(status))
    return q


def dequantize_rows(q: Q8Rows, dtype: torch.dtype = torch.bfloat16, index: Optional[torch.Tensor] = None,
                    status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of 8-bit rows (or of the rows ``index`` of them), exact in either dtype."""
    dev = _need_cuda(*q.tensors(), status)
    dt = _code(dtype)
    rows = q.rows
    if index is not None:
        index = _index(index, dev)
        rows = index.numel()
    out = torch.empty(rows, q.cols, dtype=dtype, device=dev)
    _call("ifk_q8_dequantize", dev, *q.args(), _ptr(index), q.rows, rows, q.cols, out.data_ptr(), q.cols, dt,
          _status(status))
    return out


def weight_grad(delta: torch.Tensor, q: Q8Rows, bias: bool = False, out: Optional[torch.Tensor] = None,
                out_bias: Optional[torch.Tensor] = None, accumulate: bool = False,
                status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dW, db) of a linear layer y = x W^T + b: dW = delta^T X (n_out x n_in fp32)
    from the 8-bit rows of X, and with ``bias`` (or ``out_bias``) db = the column sums
    of delta, else None.  ``out`` / ``out_bias`` receive them; with ``accumulate`` they
    are added to (gradient accumulation), and both that are wanted must be given.
    If a wait on the device gave up, dW holds NaN, and ``status`` (a device int32,
    optional) IFK_ERR_TIMEOUT."""
    dev = _need_cuda(delta, *q.tensors(), out, out_bias, status)
    delta, rows, n_out, ld = _rows2d(delta, "delta")
    dt = _code(delta.dtype)
    n_in = q.cols
    if rows != q.rows:
        raise ValueError(f"delta has {rows} rows, the layer's input {q.rows}")
    if accumulate and (out is None or (bias and out_bias is None)):
        raise ValueError("accumulate needs the tensors to add to")
    ld_out = n_in
    if out is None:
        out = torch.empty(n_out, n_in, dtype=torch.float32, device=dev)
    else:
        if out.dtype != torch.float32 or out.shape != (n_out, n_in) or (out.stride(1) != 1 and n_in > 1) \
                or (n_out > 1 and out.stride(0) < n_in):
            raise ValueError(f"out must be a row-major {n_out} x {n_in} float32 tensor")
        ld_out = max(out.stride(0), n_in)
    if out_bias is None:
        if bias:
            out_bias = torch.empty(n_out, dtype=torch.float32, device=dev)
    elif out_bias.dtype != torch.float32 or out_bias.shape != (n_out,) or not out_bias.is_contiguous():
        raise ValueError(f"out_bias must be a contiguous float32 tensor of {n_out}")
    p = delta.data_ptr()
    if dt == _lib.BF16 and p % 16 == 0 and ld % 8 == 0:
        dt |= _lib.DELTA_IN_PLACE  # no copy of delta, and no room for one
    nbytes = _workspace("ifk_q8_wgrad_workspace", rows, n_out, n_in, dt)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call("ifk_q8_wgrad", dev, p, ld, dt, *q.args(), rows, n_out, n_in, out.data_ptr(), ld_out,
          _ptr(out_bias), 1 if accumulate else 0, _status(status), ws.data_ptr(), nbytes)
    return out, out_bias


class LayerNormSaved:
    """What layer norm's backward pass needs of its forward pass: the input rows, as they
    were (``x``) or in 8 bits (``q8``), and the statistics: ``data`` begins with the
    rows' means and then their reciprocal deviations (fp32)."""

    __slots__ = ("x", "q8", "data", "x_dtype", "rows", "cols")

    def __init__(self, x: Optional[torch.Tensor], q8: Optional[Q8Rows], data: torch.Tensor, x_dtype: torch.dtype,
                 rows: int, cols: int):
        self.x, self.q8, self.data, self.x_dtype, self.rows, self.cols = x, q8, data, x_dtype, rows, cols

    @classmethod
    def empty(cls, rows: int, cols: int, x_dtype: torch.dtype, device, x: Optional[torch.Tensor]) -> "LayerNormSaved":
        """Room for the statistics of ``x`` and, where the rows themselves are not kept
        (``x`` None), for them in 8 bits."""
        start = -(-8 * rows // 16) * 16
        nbytes = start if x is not None else start + Q8Rows.size(rows, cols)
        return cls.of(torch.empty(nbytes, dtype=torch.uint8, device=device), rows, cols, x_dtype, x)

    @classmethod
    def of(cls, data: torch.Tensor, rows: int, cols: int, x_dtype: torch.dtype,
           x: Optional[torch.Tensor] = None) -> "LayerNormSaved":
        start = -(-8 * rows // 16) * 16
        return cls(x, None if x is not None else Q8Rows.of(data, rows, cols, start), data, x_dtype, rows, cols)

    @property
    def mean(self) -> torch.Tensor:
        return self.data[: 4 * self.rows].view(torch.float32)

    @property
    def rstd(self) -> torch.Tensor:
        return self.data[4 * self.rows: 8 * self.rows].view(torch.float32)


def _affine(n: int, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]) -> int:
    t = weight if weight is not None else bias
    if t is None:
        return _lib.F32
    for p in (weight, bias):
        if p is not None and (p.dim() != 1 or p.numel() != n or not p.is_contiguous()):
            raise ValueError(f"weight and bias must hold {n} contiguous values, got shape {tuple(p.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias share a dtype, got {weight.dtype} and {bias.dtype}")
    return _code(t.dtype)


_NO_ROWS = (None, 0, None, 0)


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None, save: bool = False,
                       checkpoint: bool = False) -> Tuple[torch.Tensor, Optional[LayerNormSaved]]:
    """y = (x - mean) * rstd * weight + bias over the columns of ``x`` (rows x cols),
    in ``out_dtype`` (x's by default).  With ``save`` the second value holds what
    :func:`layer_norm_backward` needs; with ``checkpoint`` the input is held there
    in 8 bits, written in the same pass, instead of as itself."""
    dev = _need_cuda(x, weight, bias)
    x, rows, n, ld = _rows2d(x, "x")
    dt = _code(x.dtype)
    if out_dtype is None:
        out_dtype = x.dtype
    ydt = _code(out_dtype)
    wdt = _affine(n, weight, bias)
    y = torch.empty(rows, n, dtype=out_dtype, device=dev)
    saved = mean = rstd = None
    q = _NO_ROWS
    if save:
        saved = LayerNormSaved.empty(rows, n, x.dtype, dev, None if checkpoint else x)
        mean = saved.data.data_ptr()
        rstd = mean + 4 * rows
        if checkpoint:
            q = saved.q8.args()
    _call("ifk_layernorm", dev, x.data_ptr(), ld, dt, _ptr(weight), _ptr(bias), wdt, rows, n, float(eps),
          y.data_ptr(), n, ydt, mean, rstd, *q)
    return y, saved


def layer_norm_backward(dy: torch.Tensor, saved: LayerNormSaved, weight: Optional[torch.Tensor] = None,
                        weight_grads: bool = True, status: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dw, db) of :func:`layer_norm_forward`: dx in the input's dtype, dw and db
    fp32 (None without ``weight_grads``).  ``status`` (a device int32, optional)
    receives IFK_ERR_TIMEOUT if a wait on the device gave up; dw, db and the rows of dx
    that were left are then NaN."""
    dev = _need_cuda(dy, saved.data, weight, status)
    dy, rows, n, ld = _rows2d(dy, "dy")
    dt, xdt = _code(dy.dtype), _code(saved.x_dtype)
    if rows != saved.rows or n != saved.cols:
        raise ValueError(f"dy is {rows} x {n}, the input was {saved.rows} x {saved.cols}")
    wdt = _affine(n, weight, None)
    if saved.x is None:
        x, ldx, q = None, 0, saved.q8.args()
    else:
        x, ldx, q = saved.x.data_ptr(), max(saved.x.stride(0), n), _NO_ROWS
    dx = torch.empty(rows, n, dtype=saved.x_dtype, device=dev)
    dw = db = ws = None
    nbytes = 0
    if weight_grads:
        dw = torch.empty(n, dtype=torch.float32, device=dev)
        db = torch.empty(n, dtype=torch.float32, device=dev)
        nbytes = _workspace("ifk_layernorm_backward_workspace", rows, n)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    mean = saved.data.data_ptr()
    _call("ifk_layernorm_backward", dev, dy.data_ptr(), ld, dt, x, ldx, xdt, *q, mean, mean + 4 * rows, _ptr(weight),
          wdt, rows, n, dx.data_ptr(), n, _ptr(dw), _ptr(db), _status(status), _ptr(ws), nbytes)
    return dx, dw, db


# ---- autograd and modules ----

def _autocast_dtype() -> Optional[torch.dtype]:
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None


class _LinearQ8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, dtype, q):
        with torch.autocast("cuda", enabled=False):
            w = weight.to(dtype)
            y = F.linear(x.to(dtype), w, None if bias is None else bias.to(dtype))
        ctx.save_for_backward(w, *(() if q is None else (q.data,)))
        ctx.x_shape, ctx.x_dtype = x.shape, x.dtype
        ctx.w_dtype, ctx.b_dtype = weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        w, *saved = ctx.saved_tensors
        dx = dw = db = None
        with torch.autocast("cuda", enabled=False):
            d2 = dy.reshape(-1, dy.shape[-1])
            if ctx.needs_input_grad[0]:
                dx = (d2 @ w).reshape(ctx.x_shape).to(ctx.x_dtype)
            if ctx.needs_input_grad[1]:
                q = Q8Rows.of(saved[0], d2.shape[0], ctx.x_shape[-1])
                dw, db = weight_grad(d2, q, bias=ctx.needs_input_grad[2])
                dw = dw.to(ctx.w_dtype)
                db = None if db is None else db.to(ctx.b_dtype)
            elif ctx.needs_input_grad[2]:
                db = d2.sum(0, dtype=torch.float32).to(ctx.b_dtype)
        return dx, dw, db, None, None


_HOOKS = tuple(k for k, v in nn.Module().__dict__.items() if "_hook" in k and isinstance(v, dict))


def _take_over(new: nn.Module, m: nn.Module) -> nn.Module:
    """``new`` with the parameters, buffers, submodules and attributes of ``m`` (not its hooks)."""
    for k, v in m.__dict__.items():
        if k in ("_parameters", "_buffers", "_modules", "_non_persistent_buffers_set"):
            new.__dict__[k] = v.copy()
        elif k not in _HOOKS and k not in ("_is_full_backward_hook", "forward"):
            new.__dict__[k] = v
    return new


class _PassRows:
    """The rows of one forward pass on their way to the hooks: ``left`` sets of hooks have yet to
    take them, at the call whose output is ``out``.  A copy or a pickle of the layer has none."""

    __slots__ = ("rows", "out", "left")

    def __init__(self, rows: Optional[Q8Rows] = None, out: Optional[torch.Tensor] = None, left: int = 0):
        self.rows, self.out, self.left = rows, None if out is None else weakref.ref(out), left

    def __reduce__(self):
        return _PassRows, ()


class Linear8(nn.Linear):
    """``nn.Linear`` that keeps its input in 8 bits for the weight gradient.

    Forward and input gradient are ``nn.Linear``'s (in the autocast dtype under
    autocast); the weight and bias gradients come from :func:`weight_grad`, summed in
    fp32.  While hooks that capture in 8 bits are attached (``share_rows``), ``take_rows``
    hands each set of them the rows of the forward pass, so they are quantised once.
    Layers that read the same tensor each keep 8-bit rows of their own."""

    _share_rows = 0                       # sets of hooks that want the rows
    _pass: Optional[_PassRows] = None

    @classmethod
    def from_linear(cls, m: nn.Linear) -> "Linear8":
        """A Linear8 on the parameters of ``m``, with its attributes."""
        return _take_over(cls(m.in_features, m.out_features, bias=m.bias is not None, device="meta"), m)

    @property
    def _last_rows(self) -> Optional[Q8Rows]:
        """The rows that not every set of hooks has taken yet."""
        p = self._pass
        return None if p is None else p.rows

    def share_rows(self) -> None:
        """One more set of hooks takes the rows of each forward pass ..."""
        self._share_rows += 1

    def unshare_rows(self) -> None:
        """... and one no longer does."""
        self._share_rows = max(self._share_rows - 1, 0)
        self._pass = None

    def take_rows(self, out: Optional[torch.Tensor] = None) -> Optional[Q8Rows]:
        """The rows of the forward pass whose output is ``out`` (None: of the last one), for one
        set of hooks; None when that pass had none, or another one (a thread's) has come since."""
        p = self._pass
        if p is None or p.rows is None or (out is not None and p.out() is not out):
            return None
        p.left -= 1
        if p.left <= 0 and self._pass is p:
            self._pass = None
        return p.rows

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        x = input
        _need_cuda(x, self.weight, self.bias)
        dtype = _autocast_dtype() or self.weight.dtype
        _code(dtype)
        if dtype != x.dtype and not torch.is_autocast_enabled("cuda"):
            raise TypeError(f"input {x.dtype} and weight {self.weight.dtype} differ")
        q = None
        if torch.is_grad_enabled() and self.weight.requires_grad:
            q = quantize_rows(x.detach().reshape(-1, x.shape[-1]))
        y = _LinearQ8.apply(x, self.weight, self.bias, dtype, q)
        if self._share_rows:
            # none as well: rows that no hook has taken are not this pass's
            self._pass = None if q is None else _PassRows(q, y, self._share_rows)
        return y


class _LayerNormQ8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, dtype, save):
        y, s = layer_norm_forward(x.reshape(-1, x.shape[-1]), weight, bias, eps, dtype, save=save, checkpoint=True)
        if s is not None:
            ctx.save_for_backward(s.data, *(() if weight is None else (weight,)))
        ctx.x_dtype, ctx.x_shape = x.dtype, x.shape
        ctx.b_dtype = None if bias is None else bias.dtype
        return y.reshape(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        data, *w = ctx.saved_tensors
        n = ctx.x_shape[-1]
        saved = LayerNormSaved.of(data, ctx.x_shape.numel() // n, n, ctx.x_dtype)
        weight = w[0] if w else None
        dx, dw, db = layer_norm_backward(dy.reshape(-1, n), saved, weight,
                                         weight_grads=ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return (dx.reshape(ctx.x_shape) if ctx.needs_input_grad[0] else None,
                dw.to(weight.dtype) if ctx.needs_input_grad[1] else None,
                db.to(ctx.b_dtype) if ctx.needs_input_grad[2] else None, None, None, None)


class LayerNorm8(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension that keeps its input in 8 bits for the
    backward pass.  The output has the input's dtype.  Under autocast it has the autocast
    dtype, which costs nothing where only Linear layers read it (they would cast it), but is
    a rounding where it is a residual stream itself; with ``autocast_output=False`` it is
    fp32 there, as nn.LayerNorm's."""

    autocast_output = True

    def __init__(self, normalized_shape, *args, autocast_output: bool = True, **kwargs):
        super().__init__(normalized_shape, *args, **kwargs)
        self.autocast_output = autocast_output
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm8 normalises the last dimension, got {tuple(self.normalized_shape)}")

    @classmethod
    def from_layer_norm(cls, m: nn.LayerNorm, autocast_output: bool = True) -> "LayerNorm8":
        """A LayerNorm8 on the parameters of ``m``, with its attributes."""
        return _take_over(cls(m.normalized_shape, eps=m.eps, elementwise_affine=m.elementwise_affine,
                              bias=m.bias is not None, device="meta", autocast_output=autocast_output), m)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        x = input
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"input of width {x.shape[-1]} for a layer norm of {self.normalized_shape[0]}")
        dtype = _autocast_dtype()
        if dtype is None:
            dtype = x.dtype
        elif not self.autocast_output:
            dtype = torch.float32
        params = [p for p in (x, self.weight, self.bias) if p is not None]
        save = torch.is_grad_enabled() and any(p.requires_grad for p in params)
        return _LayerNormQ8.apply(x, self.weight, self.bias, self.eps, dtype, save)


def convert(model: nn.Module, linear: bool = True, layer_norm: bool = True, autocast_norms: bool = False) -> nn.Module:
    """``model`` with each nn.Linear (``linear``) and each nn.LayerNorm over one dimension
    (``layer_norm``) replaced, in place, by :class:`Linear8` / :class:`LayerNorm8` on
    the same parameters, with the layer's attributes.  Subclasses, layers that already
    carry hooks of any kind (a call's, a backward pass's, a state dict's) and layers with a
    ``forward`` of their own are left as they are: convert before an optimizer attaches
    its hooks.  A model that is itself such a layer is returned replaced.

    Under autocast the layer norms' outputs stay fp32, as nn.LayerNorm's are; with
    ``autocast_norms`` they have the autocast dtype, for models whose norms only Linear
    layers read (see :class:`LayerNorm8`)."""

    def swap(m: nn.Module) -> nn.Module:
        if any(m.__dict__.get(k) for k in _HOOKS) or "forward" in m.__dict__:
            return m
        if linear and type(m) is nn.Linear:
            return Linear8.from_linear(m)
        if layer_norm and type(m) is nn.LayerNorm and len(m.normalized_shape) == 1:
            return LayerNorm8.from_layer_norm(m, autocast_norms)
        return m

    done = {}
    for parent in list(model.modules()):
        for name, child in list(parent._modules.items()):
            if child is None:
                continue
            if child not in done:  # a layer used in two places stays one layer
                done[child] = swap(child)
            if done[child] is not child:
                parent._modules[name] = done[child]
    return swap(model)
