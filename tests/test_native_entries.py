"""The native operators' C entries, called as a C program calls them: parts that the
Python layer ties together on their own, strides, buffers of the caller's that hold
anything, and vocabularies of several pieces."""
import ctypes
import pickle

import pytest

import drift_b200 as d
from drift_b200 import _lib, native
from tests.test_native_xent import DT, IG, check_grads, check_losses, exact, inputs, logit_error

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

LIB = _lib.load()
GUARD = 64 << 20  # bytes behind a workspace


def xent_op(x, w, tg, b=None, ignore=IG):
    return _lib.DriftXent(x.shape[0], x.shape[1], w.shape[0], x.stride(0), w.stride(0),
                          x.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(),
                          tg.data_ptr(), ignore, 64 if tg.dtype == torch.int64 else 32,
                          native._BF16 if x.dtype == torch.bfloat16 else native._FP16)


def workspace_bytes(op, mode):
    n = ctypes.c_int64()
    _lib.check(LIB.drift_linear_xent_workspace(op, mode, n))
    return n.value


def ptr(t):
    return None if t is None else t.data_ptr()


class Entry:
    """Outputs, and a workspace of exactly the bytes asked for with a guard behind it."""

    def __init__(self, x, w, tg, b=None):
        self.op = xent_op(x, w, tg, b)
        self.keep = (x, w, tg, b)
        self.dx, self.dw = torch.empty(x.shape, dtype=x.dtype, device="cuda"), torch.empty(
            w.shape, dtype=w.dtype, device="cuda")
        self.db = torch.empty(w.shape[0], device="cuda")

    def workspace(self, mode, fill=0xA5):
        n = workspace_bytes(self.op, mode)
        self.buf = torch.full((n + GUARD,), fill, dtype=torch.uint8, device="cuda")
        return self.buf.data_ptr(), n

    def check_guard(self):
        d.check_dev()
        n = self.buf.numel() - GUARD
        assert (self.buf[n:] == 0xA5).all()

    def gradients(self, lse, g, stride, need_db=True):
        at, n = self.workspace(1)
        dep = self.op.depth
        _lib.check(LIB.drift_linear_xent_grad_dev(
            d.Context.current().handle, self.op, lse.data_ptr(), g.data_ptr(), stride, ptr(self.dx),
            dep, ptr(self.dw), dep, ptr(self.db) if need_db else None, at, n,
            torch.cuda.current_stream().cuda_stream))
        self.check_guard()
        return self.dx, self.dw, self.db

    def mean(self):
        at, n = self.workspace(2)
        dep, loss = self.op.depth, torch.empty((), device="cuda")
        _lib.check(LIB.drift_linear_xent_mean_dev(
            d.Context.current().handle, self.op, loss.data_ptr(), ptr(self.dx), dep, ptr(self.dw),
            dep, ptr(self.db), at, n, torch.cuda.current_stream().cuda_stream))
        self.check_guard()
        return loss, self.dx, self.dw, self.db


# ------------------------------------------------------------------ db without a bias

@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("tokens,depth,vocab", [(1, 8, 1), (600, 72, 33000), (4096, 64, 32769),
                                                (1 << 20, 24, 2600)])
def test_the_workspace_holds_column_sums_without_a_bias(tokens, depth, vocab, mode):
    """db may be wanted without one: a float for 32 tokens and a column of a piece."""
    op = _lib.DriftXent(tokens=tokens, depth=depth, vocab=vocab)
    without = workspace_bytes(op, mode)
    op.bias = 256
    assert workspace_bytes(op, mode) == without
    if mode == 1:
        piece = min(-(-vocab // 8) * 8, max(256, (128 << 20) // tokens // 256 * 256))
        assert without >= 2 * tokens * piece + -(-tokens // 32) * 4 * min(piece, vocab)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("t,dep,v", [(33, 40, 257), (600, 72, 33000)])
def test_bias_gradients_without_a_bias(t, dep, v, dt):
    """Bit for bit those of a bias of zeros, and nothing behind the workspace is written."""
    x, w, tg, _ = inputs(t, dep, v, dt, bias=False)
    zero = torch.zeros(v, device="cuda")
    _, lse = d.linear_xent_dev(x, w, tg)
    g = torch.randn(t, device="cuda")
    want = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=zero)
    for a, c in zip(Entry(x, w, tg).gradients(lse, g, 1), want):
        assert torch.equal(a, c)
    want = d.linear_xent_mean_dev(x, w, tg, bias=zero)
    for a, c in zip(Entry(x, w, tg).mean(), want):
        assert torch.equal(a, c)


# ------------------------------------------------------------------ weights by row

@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("stride", [1, 2, 7])
@pytest.mark.parametrize("t,dep,v", [(1, 64, 96), (65, 40, 257), (300, 72, 1000)])
def test_strided_weights(t, dep, v, dt, stride):
    """Row i's weight is d_dloss[i * dloss_stride]; what lies between is not read."""
    x, w, tg, b = inputs(t, dep, v, dt, seed=1)
    _, lse = d.linear_xent_dev(x, w, tg, bias=b)
    g = torch.randn(t, device="cuda")
    apart = torch.full((t * stride,), float("nan"), device="cuda")
    apart[::stride] = g
    # One row's weight by the C entry is a weight by row, through Python one for all rows.
    if t == 1:
        return check_grads(x, w, tg, b, g, Entry(x, w, tg, b).gradients(lse, apart, stride))
    want = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=b)
    check_grads(x, w, tg, b, g, want)
    for a, c in zip(Entry(x, w, tg, b).gradients(lse, apart, stride), want):
        assert torch.equal(a, c)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("weight", [1e30, 3e38, float("inf"), float("nan")])
@pytest.mark.parametrize("t,dep,v", [(65, 40, 257), (300, 72, 1000)])
def test_weights_of_ignored_rows_change_nothing(t, dep, v, dt, weight):
    """Nor those of rows whose target is outside the vocabulary. (float16 holds the
    logits' gradient times a power of two that the weights choose.)"""
    x, w, tg, b = inputs(t, dep, v, dt, ignored=0.3, seed=2)
    tg[5] = v + 3
    off = (tg == IG) | (tg >= v)
    _, lse = d.linear_xent_dev(x, w, tg, bias=b)
    with pytest.raises(d.DriftError):
        d.check_dev()
    g = torch.randn(t, device="cuda")
    clean, dirty = g.masked_fill(off, 0.0), g.masked_fill(off, weight)
    want = d.linear_xent_grad_dev(x, w, tg, lse, clean, bias=b)
    valid = torch.where(off, IG, tg)
    check_grads(x, w, valid, b, clean, want)
    for a, c in zip(d.linear_xent_grad_dev(x, w, tg, lse, dirty, bias=b), want):
        assert torch.equal(a, c)


@gpu
@pytest.mark.parametrize("dt", list(DT))
def test_weights_of_rows_that_are_all_ignored(dt):
    x, w, _, b = inputs(40, 64, 300, dt)
    tg = torch.full((40,), IG, device="cuda")
    _, lse = d.linear_xent_dev(x, w, tg, bias=b)
    for weight in (1.0, 1e30, float("inf"), float("nan")):
        for a in d.linear_xent_grad_dev(x, w, tg, lse, torch.full((40,), weight, device="cuda"),
                                        bias=b):
            assert not a.any()


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("weight", [float("inf"), float("nan")])
def test_a_weight_that_is_not_finite_spoils_its_own_row_of_dx(dt, weight):
    """The others are as with 0 there, small weights as a mean's among them."""
    x, w, tg, b = inputs(65, 40, 257, dt, ignored=0.0, seed=3)
    _, lse = d.linear_xent_dev(x, w, tg, bias=b)
    g = torch.rand(65, device="cuda") * 1e-6
    g[7] = 0.0
    want = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=b)
    check_grads(x, w, tg, b, g, want)
    g[7] = weight
    dx = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=b)[0]
    assert not torch.isfinite(dx[7]).any()
    dx[7] = want[0][7]
    assert torch.equal(dx, want[0])


# ------------------------------------------------------------------ addresses

@gpu
def test_misaligned_addresses_are_refused():
    """Before any launch: every output, counter and scalar at its type's alignment."""
    ctx, st = d.Context.current().handle, torch.cuda.current_stream().cuda_stream
    x, w, tg, b = inputs(5, 64, 96, ignored=0.0)
    op, buf = xent_op(x, w, tg, b), torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    n = [workspace_bytes(op, m) for m in range(3)]
    ws = torch.empty(max(n), dtype=torch.uint8, device="cuda").data_ptr()
    at = lambda k: buf.data_ptr() + 4096 * k  # noqa: E731
    p = d.policies.by_name("mxfp4").to_c()
    h = _lib.DriftAdamW(1e-3, 0.9, 0.999, 1e-8, 0.01, 8, int(d.Rounding.STOCHASTIC))
    table = (_lib.DriftAdamWTensor * 1)(_lib.DriftAdamWTensor(
        at(8), at(9), at(10), at(11), at(12), at(13), None, 64, native._F32, native._F32))
    entries = [
        # entry, arguments, and the bytes by which each pointer among them may not be off
        (LIB.drift_mx4_quantize_dev,
         [ctx, p, 2, native._BF16, x.data_ptr(), 5, 64, 64, at(0), at(1), at(2), at(3), at(4), at(5),
          at(6), st], {4: 1, 8: 8, 9: 8, 10: 8, 11: 8, 12: 4, 13: 4, 14: 4}),
        (LIB.drift_linear_xent_dev, [ctx, op, at(0), at(1), at(2), ws, n[0], st],
         {2: 2, 3: 2, 4: 2, 5: 128}),
        (LIB.drift_linear_xent_grad_dev,
         [ctx, op, at(0), at(1), 1, at(2), 64, at(4), 64, at(8), ws, n[1], st],
         {2: 2, 3: 2, 5: 1, 7: 1, 9: 2, 10: 128}),
        (LIB.drift_linear_xent_mean_dev, [ctx, op, at(0), at(1), 64, at(4), 64, at(8), ws, n[2], st],
         {2: 2, 3: 1, 5: 1, 7: 2, 8: 128}),
        (LIB.drift_adamw_dev, [ctx, h, table, 1, at(0), at(1), at(2), at(3), at(4), st],
         {4: 4, 5: 4, 6: 2, 7: 2, 8: 4})]
    for entry, args, off in entries:
        for k, by in off.items():
            bad = list(args)
            bad[k] += by
            assert entry(*bad) == _lib.EINVAL, (entry.__name__, k)
        _lib.check(entry(*args))
    d.check_dev()


# ------------------------------------------------------------------ first use


def test_the_first_use_is_published_last(monkeypatch):
    """Another thread takes a `torch` that is set for all of it being set."""
    seen = []

    class Table(dict):
        def update(self, *a):
            seen.append(native.torch)
            super().update(*a)

    monkeypatch.setattr(native, "torch", None)
    monkeypatch.setattr(native, "_LIB", None)
    monkeypatch.setattr(native, "_TYPES", Table())
    native._start()
    assert seen == [None] and native.torch is torch and native._LIB is not None
    assert native._TYPES[torch.float16] == native._FP16


# ------------------------------------------------------------------ the scale byte 255

@gpu
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
def test_the_scale_byte_255_reads_as_nan(dtype):
    """E8M0's NaN: its block's values are NaN in every type, and no other block's."""
    gen = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 256, (5, 3 * 16), dtype=torch.uint8, generator=gen).cuda()
    scales = torch.full((5, 3), 127, dtype=torch.uint8, device="cuda")
    plain = d.mx4_dequantize_dev(d.Mx4.from_parts(codes, scales, 90), dtype=dtype)
    scales[2, 1] = 255
    got = d.mx4_dequantize_dev(d.Mx4.from_parts(codes, scales, 90), dtype=dtype)
    assert torch.isnan(got[2, 32:64]).all()
    got[2, 32:64] = plain[2, 32:64]
    assert torch.equal(got, plain)


@gpu
@pytest.mark.parametrize("m", [5, 40, 200, 5000])
def test_products_of_the_scale_byte_255_are_nan(m):
    """Whichever side holds it; its row (column) alone."""
    gen = torch.Generator().manual_seed(4)
    n, k = 600, 300
    codes = [torch.randint(0, 256, (r, 160), dtype=torch.uint8, generator=gen).cuda() for r in (m, n)]
    scales = [torch.full((r, 10), 127, dtype=torch.uint8, device="cuda") for r in (m, n)]
    a, b = (d.Mx4.from_parts(c, s, k) for c, s in zip(codes, scales))
    plain = d.mx4_gemm_dev(a, b)
    assert torch.isfinite(plain).all()
    scales[0][3, 2] = scales[1][577, 9] = 255
    bad = [d.Mx4.from_parts(c, s, k) for c, s in zip(codes, scales)]
    got = d.mx4_gemm_dev(bad[0], b)
    assert torch.isnan(got[3]).all()
    got[3] = plain[3]
    assert torch.equal(got, plain)
    got = d.mx4_gemm_dev(a, bad[1])
    assert torch.isnan(got[:, 577]).all()
    got[:, 577] = plain[:, 577]
    assert torch.equal(got, plain)


# ------------------------------------------------------------------ strided views of x

@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("t,v", [(65, 257), (70, 33000)])
@pytest.mark.parametrize("dep", [1, 37, 44])
def test_columns_past_the_depth_are_not_read(t, v, dep, dt):
    """A row ends at its depth, the last one perhaps the buffer with it: what follows
    shows up nowhere, nor in the copy of x that the gradients make."""
    x, w, tg, b = inputs(t, dep, v, dt)
    wide = torch.full((t, 48), 0x7b7b, dtype=torch.int16, device="cuda").view(DT[dt])
    wide[:, :dep] = x
    wp = torch.zeros(v, 48, dtype=DT[dt], device="cuda")
    wp[:, :dep] = w
    _, lse = d.linear_xent_dev(x, w, tg, bias=b)
    g = torch.randn(t, device="cuda")
    want = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=b)
    mean = d.linear_xent_mean_dev(x, w, tg, bias=b)
    e = Entry(wide[:, :dep], wp[:, :dep], tg, b)
    e.dx, e.dw = torch.empty_like(x), torch.empty_like(w)
    for call, ref, mode in ((lambda: e.gradients(lse, g, 1), want, 1), (e.mean, mean, 2)):
        assert all(torch.equal(a, c) for a, c in zip(call(), ref))
        words = e.buf[:workspace_bytes(e.op, mode) // 2 * 2].view(torch.int16) == 0x7b7b
        assert not (words[:-2] & words[1:-1] & words[2:]).any()


# ------------------------------------------------------------------ padding

@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (129, 257), (300, 1000), (257, 40), (1500, 1025)])
@pytest.mark.parametrize("axis", [0, 1, None])
@pytest.mark.parametrize("dt", [torch.float64, torch.float32, torch.bfloat16])
def test_every_padding_byte_is_written(rows, cols, axis, dt):
    """Into buffers of the caller's that hold 0xFF throughout: padding codes become 0
    and padding scale bytes 127, and the bytes behind either array stay."""
    gen = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=gen, dtype=torch.float64).to(dt).cuda()
    kinds = {torch.float64: native._F64, torch.float32: native._F32, torch.bfloat16: native._BF16}
    held, call = [], []
    for r, c, on in ((rows, cols, axis != 0), (cols, rows, axis != 1)):
        sizes = (ctypes.c_int64(), ctypes.c_int64())
        _lib.check(LIB.drift_mx4_sizes(r, c, *sizes))
        bufs = [torch.full((s.value + 4096,), 255, dtype=torch.uint8, device="cuda") for s in sizes]
        call += [b.data_ptr() if on else None for b in bufs]
        if on:
            held.append((r, c, *((b, s.value) for b, s in zip(bufs, sizes))))
    _lib.check(LIB.drift_mx4_quantize_dev(
        d.Context.current().handle, d.policies.by_name("mxfp4").to_c(), 0, kinds[dt], x.data_ptr(),
        rows, cols, cols, *call, None, None, None, torch.cuda.current_stream().cuda_stream))
    d.check_dev()
    for r, c, (codes, nc), (scales, ns) in held:
        assert (codes[nc:] == 255).all() and (scales[ns:] == 255).all()
        nib = torch.stack((codes[:nc] & 15, codes[:nc] >> 4), -1).view(r, -1)
        assert not nib[:, c:].any()
        # Every byte, padding included, as from_parts lays the plain scales out.
        q = d.Mx4(codes[:nc], scales[:ns].clone(), r, c)
        again = d.Mx4.from_parts(*q.to_parts(), cols=c)
        assert torch.equal(again.scales, scales[:ns])


# ------------------------------------------------------------------ vocabularies of several pieces

def check_pieces(x, w, tg, b, g, loss, lse, grads, rows=1 << 16):
    """check_losses and check_grads, rows at a time: dw's and db's sums and bounds add up."""
    half, tiny = torch.finfo(x.dtype).eps / 2, 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    W = w.double().abs()
    t, dep = x.shape
    ww, lw = torch.zeros_like(W), torch.zeros_like(W)
    wb, lb = (torch.zeros(len(w), dtype=torch.float64, device="cuda") for _ in range(2))
    floor = 2.0 ** -38 * float(g.abs().max()) if x.dtype == torch.float16 else 0.0
    dx, dw, db = grads
    for a in range(0, t, rows):
        c = slice(a, a + rows)
        X, T, G = x[c], tg[c], g[c]
        check_losses(X, w, T, b, loss[c], lse[c])
        _, z, p, dl, wx, dw1, db1 = exact(X, w, T, b, G)
        e = logit_error(X, w, b)
        e = e + e.amax(1, keepdim=True) + 2.0 ** -17 + 2.0 ** -22 * z.abs()[:, None]
        on = (G.double().abs() * (T != IG))[:, None]
        soft = p * torch.expm1(e.clamp(max=10.0)) * on + 2.0 ** -22 * dl.abs()
        el = soft + half * (dl.abs() + soft) + floor * (on > 0)
        lim = (el + (len(w) + 2) * 2.0 ** -23 * dl.abs()) @ W
        assert ((dx[c].double() - wx).abs() <= lim + half * (wx.abs() + lim) + tiny).all()
        assert not dx[c][T == IG].any()
        ww += dw1
        lw += (el + (t + 2) * 2.0 ** -23 * dl.abs()).T @ X.double().abs()
        wb += db1
        lb += (soft + (t + 2) * 2.0 ** -23 * dl.abs()).sum(0)
    assert ((dw.double() - ww).abs() <= lw + half * (ww.abs() + lw) + tiny).all()
    assert ((db.double() - wb).abs() <= lb).all()


@gpu
@pytest.mark.parametrize("t,dep,v,dt", [
    (600, 72, 250_001, "bf16"), (600, 72, 250_001, "f16"),  # gradients: two pieces, dx in parts
    ((1 << 20) + 3, 24, 2600, "bf16")])  # the loss: three pieces; gradients: eleven
def test_vocabularies_of_several_pieces(t, dep, v, dt):
    """Row statistics run on from piece to piece, the target lies in any of them, dx adds
    up over them, and the last one is short."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB free")
    x, w, tg, b = inputs(t, dep, v, dt, seed=12)
    g = torch.randn(t, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    loss, lse = d.linear_xent_dev(x, w, tg, bias=b)
    got = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=b)
    check_pieces(x, w, tg, b, g, loss, lse, got)
    again = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=b)
    assert all(torch.equal(a, c) for a, c in zip(got, again))
    mean, *got = d.linear_xent_mean_dev(x, w, tg, bias=b)
    n = int((tg != IG).sum())
    # Positive losses, t / 1024 additions a thread, then 5 in a warp and 32 over them.
    want = float(loss.double().sum()) / n
    assert abs(float(mean) - want) <= (t / 1024 + 40) * 2.0 ** -24 * want
    inv = torch.tensor([1.0 / n], device="cuda")
    for a, c in zip(got, d.linear_xent_grad_dev(x, w, tg, lse, inv, bias=b)):
        assert torch.equal(a, c)
    d.check_dev()


# ------------------------------------------------------------------ the longest sides

@pytest.mark.parametrize("rows,cols,fits", [
    ((1 << 31) - (1 << 17), 257, True), ((1 << 31) - 128, 257, False),
    (((1 << 32) - (1 << 17)) // 4, 1024, True), ((1 << 30) - 128, 1024, False)])
def test_packed_sizes_leave_a_stride_below_32_bits(rows, cols, fits):
    """The cast counts chunks of 256 elements in 32 bits, a grid's stride at a time."""
    assert LIB.drift_mx4_sizes(rows, cols, None, None) == (0 if fits else _lib.EINVAL)


# ------------------------------------------------------------------ several chunks a warp

@gpu
@pytest.mark.parametrize("kind", ["nearest", "truncate", "stochastic"])
@pytest.mark.parametrize("dt", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
def test_long_casts_equal_their_rows(dt, kind):
    """A matrix whose warps take several chunks of a row, with Inf, zeros and signed
    zeros in it, against its rows cast one by one: codes, scales and clamps. Element (i, j)
    uses draw i * cols + j."""
    rows, cols, seed, golden = 900, 2090, 0x0123456789ABCDEF, 0x9E3779B97F4A7C15
    gen = torch.Generator(device="cuda").manual_seed(17)
    x = torch.randn(rows, cols, device="cuda", generator=gen, dtype=torch.float64)
    x *= torch.randn(rows, cols, device="cuda", generator=gen, dtype=torch.float64).exp()
    x = x.to(dt)
    x[::37, ::101] = float("inf")
    x[5::41, 3::97] = float("-inf")
    x[11] = 0.0
    x[12, 64:128] = -0.0
    p = d.policies.by_name("mxfp4")
    rm = {"nearest": d.Rounding.NEAREST_EVEN, "truncate": d.Rounding.TRUNCATE,
          "stochastic": d.Rounding.STOCHASTIC}[kind]

    def signed(k):
        k &= 2 ** 64 - 1
        return k - (k >> 63 << 64)

    st = torch.tensor([seed], dtype=torch.int64, device="cuda")
    clamps, each = (torch.zeros(1, dtype=torch.int64, device="cuda") for _ in range(2))
    q = d.mx4_quantize_dev(p, x, rm, d_rng_state=st, d_clamped=clamps)
    assert int(st) == (signed(seed + rows * cols * golden) if kind == "stochastic" else seed)
    starts = torch.tensor([signed(seed + i * cols * golden) for i in range(rows)], device="cuda")
    got, scale = q.to_parts()
    for i in range(rows):
        one = d.mx4_quantize_dev(p, x[i:i + 1], rm, d_rng_state=starts[i:i + 1], d_clamped=each)
        c, s = one.to_parts()
        assert torch.equal(got[i], c[0]) and torch.equal(scale[i], s[0])
    assert torch.equal(clamps, each)
    d.check_dev()


# ------------------------------------------------------------------ policies and views

def test_a_policy_from_another_process_is_the_same_policy():
    """Its formats are copies; what they are counts, not which."""
    p = pickle.loads(pickle.dumps(d.policies.by_name("mxfp4-headroom").to_builder("p").build()))
    c, rounding = native._mx4_policy(p)
    assert c.mx_headroom == p.mx_headroom and rounding == int(p.input_rounding)
    with pytest.raises(ValueError):
        native._mx4_policy(pickle.loads(pickle.dumps(d.policies.by_name("fp8-mx"))))


@gpu
@pytest.mark.parametrize("cols", [1, 40])
def test_negated_views_are_cast_by_their_values(cols):
    """The imaginary part of a conjugate is a view whose memory holds the opposite sign."""
    z = torch.randn(50, cols, dtype=torch.complex64, device="cuda")
    p = d.policies.by_name("mxfp4")
    for x in (z.conj().imag, torch._neg_view(z.real.contiguous())):
        for got, want in zip(d.mx4_quantize_dev(p, x, axis=None),
                             d.mx4_quantize_dev(p, x.resolve_neg(), axis=None)):
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    x, w, tg, b = inputs(50, cols, 96)
    want = d.linear_xent_mean_dev(x, w, tg, bias=b)
    got = d.linear_xent_mean_dev(torch._neg_view(-x), torch._neg_view(-w), tg, bias=b)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
