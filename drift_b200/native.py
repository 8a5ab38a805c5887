"""The links of a training step in the hardware's own arithmetic.

Next to the emulated step (Quant.quantize, gemm_dev, mlp.softmax_xent,
drift_adam_dev) these run the same links as the tensor cores and a usual
mixed-precision trainer run them, on torch CUDA tensors:

* `mx4_quantize_dev`, `mx4_dequantize_dev`, `mx4_gemm_dev`: the "mxfp4" cast
  packed as the hardware holds it, and the product of packed matrices;
* `linear_xent_dev`, `linear_xent_grad_dev`, `linear_xent_mean_dev`: a linear
  layer's softmax cross entropy over a vocabulary, in pieces of it, with its
  gradients;
* `AdamW`: one update over many tensors, moments in 32 or in 8 bits.

Every call runs on torch's current stream of the tensors' device unless
`stream` is given, and on the calling thread's context (`Context.current()`)
unless `ctx` is; the tensors must live on the context's device. Outputs and
scratch come from torch's allocator under that stream, so calls may be
captured into CUDA graphs, after a first call on the thread (which opens its
context). Errors that only the device sees (a NaN cast to e2m1, a target outside
the vocabulary) are raised by `check_dev`; a graph reports its own to the context
it was captured with, which has to stay open as long as it is replayed: a thread's
own context closes with the thread.
"""
from __future__ import annotations

import array
import ctypes
import functools
import operator
from typing import List, Optional, Sequence

import numpy as np

from . import _lib
from .fmt import Formats, Rounding
from .kernel import NumericPolicy, Scaling

_F64, _F32, _BF16, _FP16 = range(4)

torch = None    # imported by the first call: the package itself does not need it
_LIB = None
_TYPES = {}
_DTYPE_OF = operator.attrgetter("dtype")


def _start():
    global torch, _LIB
    import torch as _torch

    _LIB = _lib.load()
    _TYPES.update({_torch.float64: _F64, _torch.float32: _F32, _torch.bfloat16: _BF16,
                   _torch.float16: _FP16})
    torch = _torch  # last: whoever finds it set, on any thread, finds the rest


def _types():
    if torch is None:
        _start()
    return _TYPES


def _type_of(dtype, what: str, allowed=(_F64, _F32, _BF16, _FP16)) -> int:
    t = _TYPES.get(dtype)
    if t not in allowed:
        raise TypeError(f"{what}: unsupported dtype {dtype}")
    return t


class _Call:
    """The device, context and stream of one call: torch's current stream of the
    device that `first` lives on."""

    __slots__ = ("dev", "device", "handle", "stream")

    def __init__(self, first, ctx):
        dev = first.get_device()
        if dev < 0:
            raise TypeError("expected a CUDA tensor")
        if ctx is None:
            ctx = _lib.Context.current()
        if ctx.device != dev:
            raise ValueError(f"tensor on device {dev}, context on device {ctx.device}")
        self.dev, self.device, self.handle = dev, first.device, ctx.handle
        self.stream = torch._C._cuda_getCurrentRawStream(dev)

    def ptr(self, t, what: str, dtype=None, numel: Optional[int] = None, contiguous=True):
        if t is None:
            return None
        if t.get_device() != self.dev:
            raise ValueError(f"{what}: on {t.device}, expected {self.device}")
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")
        if numel is not None and t.numel() != numel:
            raise ValueError(f"{what}: expected {numel} elements, got {t.numel()}")
        if contiguous and not t.is_contiguous():
            raise ValueError(f"{what}: must be contiguous")
        return t.data_ptr()


def _streamed(fn):
    """Gives fn's callers a `stream` argument: the call then runs, and its outputs
    and scratch are allocated, with that stream current."""

    @functools.wraps(fn)
    def call(*args, stream=None, **kw):
        if torch is None:
            _start()
        if stream is None:
            return fn(*args, **kw)
        ctx = kw.get("ctx") or getattr(args[0] if args else None, "ctx", None) or _lib.Context.current()
        if stream.device.index != ctx.device:
            raise ValueError(f"stream on {stream.device}, context on device {ctx.device}")
        with torch.cuda.stream(stream):
            return fn(*args, **kw)

    return call


# ------------------------------------------------------------------ microscaled 4-bit

class Mx4:
    """A matrix in microscaled 4-bit floating point: e2m1 codes, two a byte, and
    one power-of-two scale byte per 32 elements of a row, in the layouts that
    struct drift_mx4 describes. `codes` and `scales` are uint8 tensors."""

    __slots__ = ("_codes", "_scales", "_one", "rows", "cols", "c")

    def __init__(self, codes, scales, rows: int, cols: int):
        blocks = (cols + 31) // 32
        if codes.numel() != rows * blocks * 16:
            raise ValueError("codes: wrong size")
        if scales.numel() != (rows + 127) // 128 * ((cols + 255) // 256) * 1024:
            raise ValueError("scales: wrong size")
        if not (codes.is_contiguous() and scales.is_contiguous()
                and codes.element_size() == 1 and scales.element_size() == 1):
            raise ValueError("codes and scales must be contiguous bytes")
        if codes.device != scales.device:
            raise ValueError("codes and scales on different devices")
        self._codes, self._scales, self._one, self.rows, self.cols = codes, scales, None, rows, cols
        self.c = _lib.DriftMx4(rows, cols, codes.data_ptr(), scales.data_ptr())

    @classmethod
    def _empty(cls, device, rows: int, cols: int) -> "Mx4":
        """Both arrays in one allocation, the scales behind the codes."""
        q = cls.__new__(cls)
        n = rows * ((cols + 31) // 32) * 16
        q._one = torch.empty(n + (rows + 127) // 128 * ((cols + 255) // 256) * 1024,
                             dtype=torch.uint8, device=device)
        q._codes = q._scales = None
        q.rows, q.cols = rows, cols
        at = q._one.data_ptr()
        q.c = _lib.DriftMx4(rows, cols, at, at + n)
        return q

    @property
    def codes(self):
        if self._codes is None:
            row = (self.cols + 31) // 32 * 16
            self._codes = self._one[:self.rows * row].view(self.rows, row)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            self._scales = self._one[self.rows * ((self.cols + 31) // 32) * 16:]
        return self._scales

    @property
    def _any(self):
        return self._codes if self._one is None else self._one

    @property
    def shape(self):
        return self.rows, self.cols

    @property
    def device(self):
        return self._any.device

    @staticmethod
    def from_parts(codes, scales, cols: Optional[int] = None) -> "Mx4":
        """From plain arrays, as a file holds them: `codes` uint8 (rows, ceil(cols/32)*16),
        the even element in the low nibble, and `scales`
        uint8 (rows, ceil(cols/32)), exponent + 127; 255 makes its block NaN. Both
        are copied; codes past `cols` are read as 0."""
        if torch is None:
            _start()
        rows, blocks = scales.shape
        cols = blocks * 32 if cols is None else cols
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales: expected uint8")
        if blocks != (cols + 31) // 32 or tuple(codes.shape) != (rows, blocks * 16):
            raise ValueError("codes and scales do not match the shape")
        tiles_r, tiles_k = (rows + 127) // 128, (cols + 255) // 256 * 2
        full = torch.full((tiles_r * 128, tiles_k * 4), 127, dtype=torch.uint8,
                          device=scales.device)
        full[:rows, :blocks] = scales
        # Row r, block b of a 128 x 4 tile is byte (r % 32) * 16 + (r / 32) * 4 + b.
        tiled = full.view(tiles_r, 4, 32, tiles_k, 4).permute(0, 3, 2, 1, 4).contiguous()
        # Copies of its own, so that both arrays are aligned and the padding is zero.
        own = codes.clone(memory_format=torch.contiguous_format)
        own[:, (cols + 1) // 2:] = 0
        if cols % 2:
            own[:, cols // 2] &= 15
        return Mx4(own, tiled.view(-1), rows, cols)

    def to_parts(self):
        """The plain arrays that from_parts takes."""
        tiles_r, tiles_k = (self.rows + 127) // 128, (self.cols + 255) // 256 * 2
        blocks = (self.cols + 31) // 32
        full = self.scales.view(tiles_r, tiles_k, 32, 4, 4).permute(0, 3, 2, 1, 4)
        full = full.reshape(tiles_r * 128, tiles_k * 4)
        return self.codes.view(self.rows, blocks * 16), full[:self.rows, :blocks].contiguous()


def _mx4_policy(p: NumericPolicy):
    """The policy as it crosses the ABI and its input rounding, checked once and
    kept with the (frozen) policy."""
    c = p.__dict__.get("_mx4")
    if c is None:
        if p.scaling != Scaling.MX_BLOCK or p.scale_block != 32 or \
                Formats.E2M1.id not in (f.id for f in (p.input_format, p.grad_format) if f):
            raise ValueError("the packed cast needs a policy with e2m1 elements and MX blocks of "
                             "32")
        c = p.__dict__["_mx4"] = (p.to_c(), int(p.input_rounding))
    return c


@_streamed
def mx4_quantize_dev(p: NumericPolicy, src, rm: Optional[Rounding] = None, *,
                     axis: Optional[int] = 1, d_rng_state=None, d_clamped=None,
                     d_clamped_t=None, ctx=None):
    """The policy's MX cast of the matrix `src` (float64, float32, bfloat16 or
    float16; any strides), packed. axis 1: blocks along rows, the matrix
    itself. axis 0: blocks down columns, as the transpose (cols x rows). None:
    both, as a pair, from one read of src. The values are Quant.quantize's
    under the policy for each row (column) alone. `rm` defaults to the policy's
    input rounding; stochastic rounding needs d_rng_state (int64, one element),
    which is advanced by src.numel() draws a direction. Clamp counts are
    added to d_clamped (blocks along rows) and d_clamped_t (down columns)."""
    pc, rounding = _mx4_policy(p)
    if axis != 1 and axis is not None and axis != 0:
        raise ValueError("axis must be 0, 1 or None")
    if src.dim() != 2:
        raise ValueError("src: expected a matrix")
    call = _Call(src, ctx)
    t = _type_of(src.dtype, "src")
    if src.is_neg():
        src = src.resolve_neg()
    rng = cl = cl_t = None
    if d_rng_state is not None:
        rng = call.ptr(d_rng_state, "d_rng_state", torch.int64, 1)
    if d_clamped is not None:
        cl = call.ptr(d_clamped, "d_clamped", torch.int64, 1)
    if d_clamped_t is not None:
        cl_t = call.ptr(d_clamped_t, "d_clamped_t", torch.int64, 1)
    rows, cols = src.shape
    stride, step = src.stride()
    if (cols > 1 and step != 1) or (rows > 1 and stride < cols):
        src = src.detach().contiguous()
        stride = cols
    row = Mx4._empty(call.device, rows, cols) if axis != 0 else None
    col = Mx4._empty(call.device, cols, rows) if axis != 1 else None
    a, b = (row.c.codes, row.c.scales) if row is not None else (None, None)
    c, d = (col.c.codes, col.c.scales) if col is not None else (None, None)
    _lib.check(_LIB.drift_mx4_quantize_dev(
        call.handle, pc, rounding if rm is None else int(Rounding(rm)), t, src.data_ptr(), rows,
        cols, stride if rows > 1 else cols, a, b, c, d, rng, cl, cl_t, call.stream))
    return (row, col) if axis is None else row if axis == 1 else col


@_streamed
def mx4_dequantize_dev(q: Mx4, *, dtype=None, out=None, ctx=None):
    """The values of a packed matrix, float64 unless `dtype` or `out` says
    otherwise. Rows of `out` may be apart; its columns may not."""
    call = _Call(q._any, ctx)
    if out is None:
        out = torch.empty(q.shape, dtype=dtype or torch.float64, device=call.device)
    else:
        _matrix_out(call, out, q.shape, "out")
    _lib.check(_LIB.drift_mx4_dequantize_dev(call.handle, q.c, _type_of(out.dtype, "out"),
                                             out.data_ptr(), _row_stride(out), call.stream))
    return out


def _row_stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _matrix_out(call: _Call, t, shape, what: str) -> None:
    call.ptr(t, what, contiguous=False)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{what}: columns must be contiguous and rows must not overlap")


@_streamed
def mx4_gemm_dev(a: Mx4, b: Mx4, *, bias=None, dtype=None, out=None, ctx=None):
    """The product a b^T (+ bias) of packed matrices that share their contracted
    length: a.rows x b.rows, sums in fp32, rounded once to `dtype` (float32
    unless given; float64 holds the fp32 result). bias: float32, b.rows."""
    if a.cols != b.cols:
        raise ValueError(f"contracted lengths differ: {a.cols} and {b.cols}")
    m, n = a.rows, b.rows
    call = _Call(a._any, ctx)
    if b._any.get_device() != call.dev:
        raise ValueError(f"b: on {b.device}, expected {call.device}")
    bp = call.ptr(bias, "bias", torch.float32, n)
    if out is None:
        out = torch.empty((m, n), dtype=dtype or torch.float32, device=call.device)
        stride = n
    else:
        _matrix_out(call, out, (m, n), "out")
        stride = _row_stride(out)
    _lib.check(_LIB.drift_mx4_gemm_dev(call.handle, a.c, b.c, bp, _type_of(out.dtype, "out"),
                                       out.data_ptr(), stride, call.stream))
    return out


# ------------------------------------------------------------------ linear cross entropy

def _xent_rows(call: _Call, t, what: str):
    """`t` with 16-byte aligned rows: itself, or a copy padded to whole groups
    of eight columns."""
    if t.dim() != 2:
        raise ValueError(f"{what}: expected a matrix")
    call.ptr(t, what, contiguous=False)
    if t.is_neg():
        t = t.resolve_neg()
    rows, d = t.shape
    s0, s1 = t.stride()
    if rows <= 1:
        s0 = d
    if (d == 1 or s1 == 1) and t.data_ptr() % 16 == 0 and s0 % 8 == 0 and s0 >= d:
        return t, s0
    pad = torch.empty((rows, (d + 7) // 8 * 8), dtype=t.dtype, device=t.device)
    pad[:, :d] = t.detach()
    return pad, pad.shape[1]


def _xent_op(call: _Call, x, w, targets, bias, ignore_index):
    t = _type_of(x.dtype, "x", (_BF16, _FP16))
    if w.dtype != x.dtype:
        raise TypeError(f"w: expected {x.dtype}, got {w.dtype}")
    xa, xs = _xent_rows(call, x, "x")
    wa, ws = _xent_rows(call, w, "w")
    n, d = x.shape
    v = w.shape[0]
    if w.shape[1] != d or v < 1 or d < 1:
        raise ValueError(f"w: expected (vocab, {d}), got {tuple(w.shape)}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError("targets: expected int32 or int64")
    tp = call.ptr(targets, "targets", numel=n)
    bp = call.ptr(bias, "bias", torch.float32, v)
    op = _lib.DriftXent(n, d, v, xs, ws, xa.data_ptr(), wa.data_ptr(), bp, tp, int(ignore_index),
                        64 if targets.dtype == torch.int64 else 32, t)
    return op, (xa, wa)


def _xent_ws(call: _Call, op, grad: int):
    need = ctypes.c_int64()
    _lib.check(_LIB.drift_linear_xent_workspace(op, grad, need))
    return torch.empty(need.value, dtype=torch.uint8, device=call.device)


def _xent_outputs(call, op, x, need_dx, need_dw, with_bias):
    dev = call.device
    dx = torch.empty((op.tokens, op.depth), dtype=x.dtype, device=dev) if need_dx else None
    dw = torch.empty((op.vocab, op.depth), dtype=x.dtype, device=dev) if need_dw else None
    db = torch.empty(op.vocab, dtype=torch.float32, device=dev) if with_bias else None
    return dx, dw, db, [None if t is None else t.data_ptr() for t in (dx, dw, db)]


@_streamed
def linear_xent_dev(x, w, targets, *, bias=None, ignore_index: int = -100, ctx=None):
    """Softmax cross entropy of the logits x w^T (+ bias) against `targets`, row
    by row, without keeping the logits: (loss, lse), both float32. x (tokens,
    depth) and w (vocab, depth) are bfloat16 or float16, bias float32, targets
    int32 or int64. Rows whose target is ignore_index have loss 0. `lse` is
    what linear_xent_grad_dev needs."""
    call = _Call(x, ctx)
    op, keep = _xent_op(call, x, w, targets, bias, ignore_index)
    loss = torch.empty(op.tokens, dtype=torch.float32, device=call.device)
    lse = torch.empty(op.tokens, dtype=torch.float32, device=call.device)
    ws = _xent_ws(call, op, 0)
    _lib.check(_LIB.drift_linear_xent_dev(call.handle, op, loss.data_ptr(), lse.data_ptr(), None,
                                          ws.data_ptr(), ws.numel(), call.stream))
    return loss, lse


@_streamed
def linear_xent_grad_dev(x, w, targets, lse, d_loss, *, bias=None, ignore_index: int = -100,
                         need_dx: bool = True, need_dw: bool = True, ctx=None):
    """Gradients of linear_xent_dev's losses weighted by `d_loss` (float32, one
    per row, or one element for all rows): (dx, dw, db), in x's type, w's type
    and float32; db is None without a bias, dx and dw where not needed."""
    call = _Call(x, ctx)
    op, keep = _xent_op(call, x, w, targets, bias, ignore_index)
    call.ptr(lse, "lse", torch.float32, op.tokens)
    one = d_loss.numel() == 1
    g = call.ptr(d_loss, "d_loss", torch.float32, None if one else op.tokens)
    ws = _xent_ws(call, op, 1)
    dx, dw, db, (px, pw, pb) = _xent_outputs(call, op, x, need_dx, need_dw, bias is not None)
    _lib.check(_LIB.drift_linear_xent_grad_dev(
        call.handle, op, lse.data_ptr(), g, 0 if one else 1, px, op.depth, pw, op.depth, pb,
        ws.data_ptr(), ws.numel(), call.stream))
    return dx, dw, db


@_streamed
def linear_xent_mean_dev(x, w, targets, *, bias=None, ignore_index: int = -100, ctx=None):
    """mlp.softmax_xent's counterpart for a whole output layer: the mean loss of
    the rows that are not ignored (a float32 scalar tensor; 0 when all are) and its
    gradients: (loss, dx, dw, db). Up to 2^24 logits in rows of up to 2^15 are kept
    from the loss to its gradients; beyond, they are computed again, a piece of the
    vocabulary at a time."""
    call = _Call(x, ctx)
    op, keep = _xent_op(call, x, w, targets, bias, ignore_index)
    mean = torch.empty((), dtype=torch.float32, device=call.device)
    ws = _xent_ws(call, op, 2)
    dx, dw, db, (px, pw, pb) = _xent_outputs(call, op, x, True, True, bias is not None)
    _lib.check(_LIB.drift_linear_xent_mean_dev(
        call.handle, op, mean.data_ptr(), px, op.depth, pw, op.depth, pb, ws.data_ptr(),
        ws.numel(), call.stream))
    return mean, dx, dw, db


# ------------------------------------------------------------------ AdamW

class AdamW:
    """AdamW over a fixed list of parameters, one launch a step for up to 256 of
    them (drift_adamw_dev). Parameters and gradients are float32, bfloat16 or
    float16, contiguous, and may differ in type; arithmetic is float32.

    state_bits 32 keeps both moments in float32. state_bits 8 keeps them as
    float8_e4m3fn codes with one float32 scale per 256 elements: the first
    moment itself and the root of the second. `rounding` then may be
    Rounding.STOCHASTIC, with d_rng_state (int64, one element).

    A gradient that is Inf or NaN leaves its moments so: in 8 bits its whole block of
    256 reads as NaN from then on.

    The moments start at zero (on the stream current at construction), or are `state`:
    [m, v] or [m, m_scale, r, r_scale], each a list like `params`. The step count lives on the device
    (d_step, int64), so a captured step replays as the next one. `copies`
    (a list with None where there is none) receive the new parameters in their
    own type, for low-precision copies of float32 masters. All of them keep the
    memory they have here: new values are copied into it."""

    def __init__(self, params: Sequence, *, lr: float = 1e-3, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, state_bits: int = 32,
                 rounding: Rounding = Rounding.NEAREST_EVEN, state: Optional[List] = None,
                 copies: Optional[Sequence] = None, d_step=None, d_rng_state=None, ctx=None):
        if torch is None:
            _start()
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        self.state_bits = state_bits
        self.rounding = Rounding(rounding)
        if self.rounding != Rounding.NEAREST_EVEN and \
                (state_bits != 8 or self.rounding != Rounding.STOCHASTIC):
            raise ValueError("rounding: nearest even, or stochastic with 8-bit moments")
        if self.rounding == Rounding.STOCHASTIC and d_rng_state is None:
            raise ValueError("stochastic rounding needs d_rng_state")
        self.hyper = _lib.DriftAdamW(float(lr), float(betas[0]), float(betas[1]), float(eps),
                                     float(weight_decay), state_bits, int(self.rounding))
        self.ctx = ctx
        call = _Call(self.params[0], ctx)
        dev = call.device
        n = self._sizes = self._run = [p.numel() for p in self.params]
        self._dtypes = None
        if state is None:
            def zeros(dtype, sizes):
                return [torch.zeros(k, dtype=dtype, device=dev) for k in sizes]
            if state_bits == 32:
                state = [zeros(torch.float32, n), zeros(torch.float32, n)]
            else:
                nb = [(k + 255) // 256 for k in n]
                f8 = torch.float8_e4m3fn
                state = [zeros(f8, n), zeros(torch.float32, nb), zeros(f8, n),
                         zeros(torch.float32, nb)]
        if len(state) != (2 if state_bits == 32 else 4) or \
                any(len(x) != len(n) for x in state):
            raise ValueError("state does not match the parameters")
        self.state = [list(x) for x in state]
        self.copies = list(copies) if copies is not None else [None] * len(n)
        if len(self.copies) != len(n):
            raise ValueError("copies do not match the parameters")
        self.d_step = d_step if d_step is not None else torch.zeros(1, dtype=torch.int64,
                                                                    device=dev)
        self.d_rng_state = d_rng_state
        self._step = call.ptr(self.d_step, "d_step", torch.int64, 1)
        self._rng = call.ptr(d_rng_state, "d_rng_state", torch.int64, 1)
        self._scalars = torch.zeros(8, dtype=torch.float32, device=dev)
        low = (_F32, _BF16, _FP16)
        self._table = (_lib.DriftAdamWTensor * len(n))()
        self._columns = np.frombuffer(self._table, dtype=np.dtype(
            [(k, np.uint64 if c is ctypes.c_void_p else c) for k, c in
             _lib.DriftAdamWTensor._fields_]))
        code = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        for i, p in enumerate(self.params):
            t = self._table[i]
            t.param = call.ptr(p, f"params[{i}]")
            t.param_type = _type_of(p.dtype, f"params[{i}]", low)
            t.n = n[i]
            if state_bits == 32:
                m, v, ms, vs = self.state[0][i], self.state[1][i], None, None
            else:
                m, ms, v, vs = (x[i] for x in self.state)
                nb = (n[i] + 255) // 256
                t.m_scale = call.ptr(ms, f"m_scale[{i}]", torch.float32, nb)
                t.v_scale = call.ptr(vs, f"v_scale[{i}]", torch.float32, nb)
            t.m = call.ptr(m, f"m[{i}]", code, n[i])
            t.v = call.ptr(v, f"v[{i}]", code, n[i])
            c = self.copies[i]
            if c is not None:
                t.copy = call.ptr(c, f"copies[{i}]", numel=n[i])
                t.copy_type = _type_of(c.dtype, f"copies[{i}]", low)
        # Everything a step writes, in order of address: no two may share memory. It is held
        # here too, so that the table's addresses stay good whatever becomes of the lists.
        self._held = [x.detach() for part in (self.params, *self.state, self.copies,
                                              [self.d_step, d_rng_state])
                      for x in part if x is not None]
        self._at = [p.data_ptr() for p in self.params]
        written = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size())
                         for x in self._held if x.numel())
        if any(a[1] > b[0] for a, b in zip(written, written[1:])):
            raise ValueError("parameters, moments and copies must not share memory")

    @_streamed
    def step(self, grads: Sequence, *, lr: Optional[float] = None, d_lr=None,
             d_grad_scale=None) -> None:
        """One update with `grads` (a list like the parameters; None skips one).
        `lr` sets the rate from this step on; d_lr (float32, one element)
        replaces it for this step from the device; d_grad_scale (float32, one
        element) multiplies the gradients."""
        if len(grads) != len(self.params):
            raise ValueError("grads do not match the parameters")
        if lr is not None:
            self.hyper.lr = float(lr)
        call = _Call(self.params[0], self.ctx)
        if list(map(torch.Tensor.data_ptr, self.params)) != self._at:
            raise ValueError("a parameter's memory was replaced: it belongs to the optimizer")
        sizes = self._sizes
        want = run = sizes
        try:
            dtypes = list(map(_DTYPE_OF, grads))
        except AttributeError:  # some are None
            first = self.params[0]
            want = [first.numel() if g is None else k for k, g in zip(sizes, grads)]
            run = [0 if g is None else k for k, g in zip(sizes, grads)]
            grads = [first if g is None else g for g in grads]  # skipped: never read
            dtypes = list(map(_DTYPE_OF, grads))
        tensor = torch.Tensor
        if dtypes != self._dtypes:  # as a rule the same as the step before
            types = [_TYPES.get(t, 0) for t in dtypes]
            if not all(types):
                raise ValueError("grads: expected float32, bfloat16 or float16 tensors")
            self._columns["grad_type"] = types
            self._dtypes = dtypes
        if list(map(tensor.numel, grads)) != want or \
                set(map(tensor.get_device, grads)) != {call.dev} or \
                not all(map(tensor.is_contiguous, grads)):
            raise ValueError("grads: expected contiguous tensors of the parameters' sizes on "
                             f"{call.device}")
        # In whole columns: attribute by attribute the table would cost a microsecond a tensor.
        self._columns["grad"] = array.array("Q", map(tensor.data_ptr, grads))
        if run is not self._run:
            self._columns["n"] = run
            self._run = run
        _lib.check(_LIB.drift_adamw_dev(
            call.handle, self.hyper, self._table, len(sizes), self._step, self._scalars.data_ptr(),
            call.ptr(d_lr, "d_lr", torch.float32, 1),
            call.ptr(d_grad_scale, "d_grad_scale", torch.float32, 1), self._rng, call.stream))
