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
captured into CUDA graphs. Errors that only the device sees (a NaN cast to
e2m1, a target outside the vocabulary) are raised by `check_dev`.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence

from . import _lib
from .fmt import Formats, Rounding
from .kernel import NumericPolicy, Scaling

_F64, _F32, _BF16, _FP16 = range(4)
_TYPES = None


def _types():
    global _TYPES
    if _TYPES is None:
        import torch

        _TYPES = {torch.float64: _F64, torch.float32: _F32, torch.bfloat16: _BF16,
                  torch.float16: _FP16}
    return _TYPES


def _type_of(dtype, what: str, allowed=(_F64, _F32, _BF16, _FP16)) -> int:
    t = _types().get(dtype)
    if t not in allowed:
        raise TypeError(f"{what}: unsupported dtype {dtype}")
    return t


class _Call:
    """The context, stream and device of one call, with torch's current stream
    set to it, so that what the call allocates belongs to that stream."""

    def __init__(self, first, stream, ctx):
        import torch

        if not first.is_cuda:
            raise TypeError("expected a CUDA tensor")
        self.torch = torch
        self.device = first.device
        self.ctx = ctx or _lib.Context.current()
        if self.ctx.device != self.device.index:
            raise ValueError(f"tensor on {self.device}, context on device {self.ctx.device}")
        self.given = stream
        s = stream if stream is not None else torch.cuda.current_stream(self.device)
        if s.device != self.device:
            raise ValueError(f"stream on {s.device}, tensor on {self.device}")
        self.stream = s.cuda_stream

    def __enter__(self):
        self.scope = None
        if self.given is not None:
            self.scope = self.torch.cuda.stream(self.given)
            self.scope.__enter__()
        return self

    def __exit__(self, *exc):
        if self.scope is not None:
            self.scope.__exit__(*exc)
        return False

    def empty(self, shape, dtype):
        return self.torch.empty(shape, dtype=dtype, device=self.device)

    def scratch(self, n: int):
        return self.torch.empty(n, dtype=self.torch.uint8, device=self.device) if n else None

    def ptr(self, t, what: str, dtype=None, numel: Optional[int] = None, contiguous=True):
        if t is None:
            return None
        if t.device != self.device:
            raise ValueError(f"{what}: on {t.device}, expected {self.device}")
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{what}: expected {dtype}, got {t.dtype}")
        if numel is not None and t.numel() != numel:
            raise ValueError(f"{what}: expected {numel} elements, got {t.numel()}")
        if contiguous and not t.is_contiguous():
            raise ValueError(f"{what}: must be contiguous")
        return t.data_ptr()


# ------------------------------------------------------------------ microscaled 4-bit

class Mx4:
    """A matrix in microscaled 4-bit floating point: e2m1 codes, two a byte, and
    one power-of-two scale byte per 32 elements of a row, in the layouts that
    struct drift_mx4 describes. `codes` and `scales` are uint8 tensors."""

    __slots__ = ("codes", "scales", "rows", "cols", "c")

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
        self.codes, self.scales, self.rows, self.cols = codes, scales, rows, cols
        self.c = _lib.DriftMx4(rows, cols, codes.data_ptr(), scales.data_ptr())

    @property
    def shape(self):
        return self.rows, self.cols

    @property
    def device(self):
        return self.codes.device

    @staticmethod
    def from_parts(codes, scales, cols: Optional[int] = None) -> "Mx4":
        """From plain arrays, as a file holds them: `codes` uint8 (rows, ceil(cols/32)*16),
        the even element in the low nibble and padding codes 0, and `scales`
        uint8 (rows, ceil(cols/32)), exponent + 127, none of them 255."""
        import torch

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
        return Mx4(codes.contiguous(), tiled.view(-1), rows, cols)

    def to_parts(self):
        """The plain arrays that from_parts takes."""
        tiles_r, tiles_k = (self.rows + 127) // 128, (self.cols + 255) // 256 * 2
        blocks = (self.cols + 31) // 32
        full = self.scales.view(tiles_r, tiles_k, 32, 4, 4).permute(0, 3, 2, 1, 4)
        full = full.reshape(tiles_r * 128, tiles_k * 4)
        return self.codes.view(self.rows, blocks * 16), full[:self.rows, :blocks].contiguous()


def _mx4_empty(call: _Call, rows: int, cols: int) -> Mx4:
    u8 = call.torch.uint8
    blocks = (cols + 31) // 32
    return Mx4(call.empty((rows, blocks * 16), u8),
               call.empty((rows + 127) // 128 * ((cols + 255) // 256) * 1024, u8), rows, cols)


def mx4_quantize_dev(p: NumericPolicy, src, rm: Optional[Rounding] = None, *,
                     axis: Optional[int] = 1, d_rng_state=None, d_clamped=None,
                     d_clamped_t=None, stream=None, ctx=None):
    """The policy's MX cast of the matrix `src` (float64, float32, bfloat16 or
    float16; any strides), packed. axis 1: blocks along rows, the matrix
    itself. axis 0: blocks down columns, as the transpose (cols x rows). None:
    both, as a pair, from one read of src. The values are Quant.quantize's
    under the policy for each row (column) alone. `rm` defaults to the policy's
    input rounding; stochastic rounding needs d_rng_state (int64, one element),
    which is advanced by src.numel() draws a direction. Clamp counts are
    added to d_clamped (blocks along rows) and d_clamped_t (down columns)."""
    rm = p.input_rounding if rm is None else Rounding(rm)
    if axis not in (0, 1, None):
        raise ValueError("axis must be 0, 1 or None")
    if p.scaling != Scaling.MX_BLOCK or p.scale_block != 32 or \
            Formats.E2M1 not in (p.input_format, p.grad_format):
        raise ValueError("the packed cast needs a policy with e2m1 elements and MX blocks of 32")
    if src.dim() != 2:
        raise ValueError("src: expected a matrix")
    with _Call(src, stream, ctx) as call:
        t = _type_of(src.dtype, "src")
        i64 = call.torch.int64
        rng = call.ptr(d_rng_state, "d_rng_state", i64, 1)
        cl, cl_t = call.ptr(d_clamped, "d_clamped", i64, 1), call.ptr(d_clamped_t, "d_clamped_t",
                                                                     i64, 1)
        rows, cols = src.shape
        if (cols > 1 and src.stride(1) != 1) or (rows > 1 and src.stride(0) < cols):
            src = src.contiguous()
        row = _mx4_empty(call, rows, cols) if axis != 0 else None
        col = _mx4_empty(call, cols, rows) if axis != 1 else None
        a, b = (row.c.codes, row.c.scales) if row else (None, None)
        c, d = (col.c.codes, col.c.scales) if col else (None, None)
        pc = p.to_c()
        _lib.check(_lib.load().drift_mx4_quantize_dev(
            call.ctx.handle, ctypes.byref(pc), int(rm), t, src.data_ptr(), rows, cols,
            src.stride(0) if rows > 1 else cols, a, b, c, d, rng, cl, cl_t, call.stream))
    return (row, col) if axis is None else row if axis == 1 else col


def mx4_dequantize_dev(q: Mx4, *, dtype=None, out=None, stream=None, ctx=None):
    """The values of a packed matrix, float64 unless `dtype` or `out` says
    otherwise. Rows of `out` may be apart; its columns may not."""
    with _Call(q.codes, stream, ctx) as call:
        if out is None:
            out = call.empty(q.shape, dtype or call.torch.float64)
        _matrix_out(call, out, q.shape, "out")
        _lib.check(_lib.load().drift_mx4_dequantize_dev(
            call.ctx.handle, ctypes.byref(q.c), _type_of(out.dtype, "out"), out.data_ptr(),
            _row_stride(out), call.stream))
    return out


def _row_stride(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _matrix_out(call: _Call, t, shape, what: str) -> None:
    call.ptr(t, what, contiguous=False)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{what}: columns must be contiguous and rows must not overlap")


def mx4_gemm_dev(a: Mx4, b: Mx4, *, bias=None, dtype=None, out=None, stream=None, ctx=None):
    """The product a b^T (+ bias) of packed matrices that share their contracted
    length: a.rows x b.rows, sums in fp32, rounded once to `dtype` (float32
    unless given; float64 holds the fp32 result). bias: float32, b.rows."""
    if a.cols != b.cols:
        raise ValueError(f"contracted lengths differ: {a.cols} and {b.cols}")
    with _Call(a.codes, stream, ctx) as call:
        call.ptr(b.codes, "b")
        bp = call.ptr(bias, "bias", call.torch.float32, b.rows)
        if out is None:
            out = call.empty((a.rows, b.rows), dtype or call.torch.float32)
        _matrix_out(call, out, (a.rows, b.rows), "out")
        lib = _lib.load()
        need = ctypes.c_int64()
        _lib.check(lib.drift_mx4_gemm_workspace(a.rows, b.rows, a.cols, ctypes.byref(need)))
        ws = call.scratch(need.value)
        _lib.check(lib.drift_mx4_gemm_dev(
            call.ctx.handle, ctypes.byref(a.c), ctypes.byref(b.c), bp,
            _type_of(out.dtype, "out"), out.data_ptr(), _row_stride(out),
            None if ws is None else ws.data_ptr(), need.value, call.stream))
    return out


# ------------------------------------------------------------------ linear cross entropy

def _xent_rows(call: _Call, t, what: str):
    """`t` with 16-byte aligned rows: itself, or a copy padded to whole groups
    of eight columns."""
    if t.dim() != 2:
        raise ValueError(f"{what}: expected a matrix")
    call.ptr(t, what, contiguous=False)
    rows, d = t.shape
    ok = (d == 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0 and \
        (rows <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= d)) and (rows > 1 or d % 8 == 0)
    if ok:
        return t, t.stride(0) if rows > 1 else d
    pad = call.empty((rows, (d + 7) // 8 * 8), t.dtype)
    pad[:, :d] = t
    return pad, pad.shape[1]


def _xent_op(call: _Call, x, w, targets, bias, ignore_index):
    torch = call.torch
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


def _xent_ws(call: _Call, op, grad: bool):
    need = ctypes.c_int64()
    _lib.check(_lib.load().drift_linear_xent_workspace(ctypes.byref(op), int(grad),
                                                       ctypes.byref(need)))
    return call.scratch(need.value)


def _xent_forward(call, op, loss, lse, mean, ws):
    _lib.check(_lib.load().drift_linear_xent_dev(
        call.ctx.handle, ctypes.byref(op), None if loss is None else loss.data_ptr(),
        lse.data_ptr(), None if mean is None else mean.data_ptr(), ws.data_ptr(), ws.numel(),
        call.stream))


def _xent_backward(call, op, x, lse, g, g_stride, with_bias, ws, need):
    torch = call.torch
    dx = call.empty((op.tokens, op.depth), x.dtype) if need[0] else None
    dw = call.empty((op.vocab, op.depth), x.dtype) if need[1] else None
    db = call.empty((op.vocab,), torch.float32) if with_bias else None
    _lib.check(_lib.load().drift_linear_xent_grad_dev(
        call.ctx.handle, ctypes.byref(op), lse.data_ptr(), g, g_stride,
        None if dx is None else dx.data_ptr(), op.depth,
        None if dw is None else dw.data_ptr(), op.depth,
        None if db is None else db.data_ptr(), ws.data_ptr(), ws.numel(), call.stream))
    return dx, dw, db


def linear_xent_dev(x, w, targets, *, bias=None, ignore_index: int = -100, stream=None, ctx=None):
    """Softmax cross entropy of the logits x w^T (+ bias) against `targets`, row
    by row, without keeping the logits: (loss, lse), both float32. x (tokens,
    depth) and w (vocab, depth) are bfloat16 or float16, bias float32, targets
    int32 or int64. Rows whose target is ignore_index have loss 0. `lse` is
    what linear_xent_grad_dev needs."""
    with _Call(x, stream, ctx) as call:
        op, keep = _xent_op(call, x, w, targets, bias, ignore_index)
        f32 = call.torch.float32
        loss, lse = call.empty((op.tokens,), f32), call.empty((op.tokens,), f32)
        _xent_forward(call, op, loss, lse, None, _xent_ws(call, op, False))
    return loss, lse


def linear_xent_grad_dev(x, w, targets, lse, d_loss, *, bias=None, ignore_index: int = -100,
                         need_dx: bool = True, need_dw: bool = True, stream=None, ctx=None):
    """Gradients of linear_xent_dev's losses weighted by `d_loss` (float32, one
    per row, or one element for all rows): (dx, dw, db), in x's type, w's type
    and float32; db is None without a bias, dx and dw where not needed."""
    with _Call(x, stream, ctx) as call:
        op, keep = _xent_op(call, x, w, targets, bias, ignore_index)
        f32 = call.torch.float32
        call.ptr(lse, "lse", f32, op.tokens)
        one = d_loss.numel() == 1
        g = call.ptr(d_loss, "d_loss", f32, None if one else op.tokens)
        return _xent_backward(call, op, x, lse, g, 0 if one else 1, bias is not None,
                              _xent_ws(call, op, True), (need_dx, need_dw))


def linear_xent_mean_dev(x, w, targets, *, bias=None, ignore_index: int = -100, stream=None,
                         ctx=None):
    """mlp.softmax_xent's counterpart for a whole output layer: the mean loss of
    the rows that are not ignored (a float32 scalar tensor; 0 when all are) and its
    gradients: (loss, dx, dw, db)."""
    with _Call(x, stream, ctx) as call:
        op, keep = _xent_op(call, x, w, targets, bias, ignore_index)
        f32 = call.torch.float32
        lse, mean = call.empty((op.tokens,), f32), call.empty((2,), f32)
        ws = _xent_ws(call, op, True)
        _xent_forward(call, op, None, lse, mean, ws)
        grads = _xent_backward(call, op, x, lse, mean.data_ptr() + 4, 0, bias is not None, ws,
                               (True, True))
    return (mean[0], *grads)


# ------------------------------------------------------------------ AdamW

class AdamW:
    """AdamW over a fixed list of parameters, one launch a step for up to 128 of
    them (drift_adamw_dev). Parameters and gradients are float32, bfloat16 or
    float16, contiguous, and may differ in type; arithmetic is float32.

    state_bits 32 keeps both moments in float32. state_bits 8 keeps them as
    float8_e4m3fn codes with one float32 scale per 256 elements: the first
    moment itself and the root of the second. `rounding` then may be
    Rounding.STOCHASTIC, with d_rng_state (int64, one element).

    The moments start at zero, or are `state`: [m, v] or [m, m_scale, r,
    r_scale], each a list like `params`. The step count lives on the device
    (d_step, int64), so a captured step replays as the next one. `copies`
    (a list with None where there is none) receive the new parameters in their
    own type, for low-precision copies of float32 masters."""

    def __init__(self, params: Sequence, *, lr: float = 1e-3, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, state_bits: int = 32,
                 rounding: Rounding = Rounding.NEAREST_EVEN, state: Optional[List] = None,
                 copies: Optional[Sequence] = None, d_step=None, d_rng_state=None, ctx=None):
        import torch

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
        dev = self.params[0].device
        with _Call(self.params[0], None, ctx) as call:
            n = [p.numel() for p in self.params]
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

    def step(self, grads: Sequence, *, lr: Optional[float] = None, d_lr=None, d_grad_scale=None,
             stream=None) -> None:
        """One update with `grads` (a list like the parameters; None skips one).
        `lr` sets the rate from this step on; d_lr (float32, one element)
        replaces it for this step from the device; d_grad_scale (float32, one
        element) multiplies the gradients."""
        if len(grads) != len(self.params):
            raise ValueError("grads do not match the parameters")
        if lr is not None:
            self.hyper.lr = float(lr)
        with _Call(self.params[0], stream, self.ctx) as call:
            f32 = call.torch.float32
            table = self._table
            types = _types()
            dev = call.device
            for i, g in enumerate(grads):
                t = table[i]
                if g is None:
                    t.n = 0
                    continue
                n = self.params[i].numel()
                ty = types.get(g.dtype)
                if g.device != dev or not ty or g.numel() != n or not g.is_contiguous():
                    raise ValueError(f"grads[{i}]: expected {n} contiguous float32, bfloat16 or "
                                     f"float16 elements on {dev}")
                t.grad, t.grad_type, t.n = g.data_ptr(), ty, n
            _lib.check(_lib.load().drift_adamw_dev(
                call.ctx.handle, ctypes.byref(self.hyper), table, len(table), self._step,
                self._scalars.data_ptr(), call.ptr(d_lr, "d_lr", f32, 1),
                call.ptr(d_grad_scale, "d_grad_scale", f32, 1), self._rng, call.stream))
