"""The packed 4-bit cast and the product of packed matrices, on the GPU, against
the oracle's MX cast (row by row) and the product in 64 bits."""
import numpy as np
import pytest

import drift_b200 as d
from drift_b200.native import _types
from tests.helpers import heavy_tailed

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

P = {"nearest": d.policies.by_name("mxfp4"), "headroom": d.policies.by_name("mxfp4-headroom"),
     "truncate": d.policies.by_name("mxfp4").to_builder("t")
     .input_rounding(d.Rounding.TRUNCATE).build(),
     "sr": d.policies.by_name("mxfp4-sr")}
DT = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def oracle_rows(x, p):
    """The oracle's cast of each row on its own: values and clamps."""
    from oracle import oracle as O

    op = O.policy(input_format=2, scaling=2, mx_headroom=p.mx_headroom,
                  input_rounding=int(p.input_rounding))
    out, clamps = np.empty_like(x), 0
    for i in range(x.shape[0]):
        row = np.ascontiguousarray(x[i])
        out[i], c, _ = O.quantize(op, 2, int(p.input_rounding), row, 1.0)
        clamps += c
    return out, clamps


@pytest.mark.parametrize("headroom", [-4, 2, 5])
@pytest.mark.parametrize("dt", list(DT))
def test_cast_with_other_headrooms(headroom, dt):
    p = P["nearest"].to_builder("h").mx_headroom(headroom).build()
    x = source(70, 200, dt, 21)
    x[0, :32] = torch.tensor([2.0 ** -130, 2.0 ** -132] + [0.0] * 30).to(DT[dt])
    x[1, :32] = 3e38 if dt != "f16" else 6e4
    host = x.double().cpu().numpy()
    for axis, h in ((1, host), (0, np.ascontiguousarray(host.T))):
        want, clamps = oracle_rows(h, p)
        c = torch.zeros(1, dtype=torch.int64, device="cuda")
        q = d.mx4_quantize_dev(p, x, axis=axis, **{"d_clamped" if axis else "d_clamped_t": c})
        v = d.mx4_dequantize_dev(q).cpu().numpy()
        assert (v.view(np.int64) == want.view(np.int64)).all() and int(c) == clamps


def source(rows, cols, dt, seed, edges=True):
    rs = np.random.default_rng(seed)
    x = heavy_tailed(rs, rows * cols, 2.0).reshape(rows, cols)
    if edges and rows * cols >= 16:
        flat = x.reshape(-1)
        for k, v in enumerate([0.0, -0.0, np.inf, -np.inf, 1e-30, -1e-40, 65000.0, 7.0, 6.0, 5.0,
                               0.25, -0.75, 2.5]):
            flat[rs.integers(flat.size)] = v
        x[rs.integers(rows)] = 0.0
    return torch.from_numpy(x).to(DT[dt]).cuda()


SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (5, 255), (127, 64), (129, 257), (64, 2048),
          (300, 1000), (1000, 40)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("kind", ["nearest", "headroom", "truncate"])
def test_cast_equals_the_oracle_along_both_axes(rows, cols, dt, kind):
    p = P[kind]
    x = source(rows, cols, dt, rows * 7919 + cols)
    host = x.double().cpu().numpy()
    want, clamps = oracle_rows(host, p)
    want_t, clamps_t = oracle_rows(np.ascontiguousarray(host.T), p)
    for axis in (1, 0, None):
        c = torch.zeros(2, dtype=torch.int64, device="cuda")
        got = d.mx4_quantize_dev(p, x, axis=axis, d_clamped=c[:1], d_clamped_t=c[1:])
        row, col = got if axis is None else (got, None) if axis == 1 else (None, got)
        if row is not None:
            assert row.shape == (rows, cols)
            v = d.mx4_dequantize_dev(row).cpu().numpy()
            assert (v.view(np.int64) == want.view(np.int64)).all()
            assert int(c[0]) == clamps
        if col is not None:
            assert col.shape == (cols, rows)
            v = d.mx4_dequantize_dev(col).cpu().numpy()
            assert (v.view(np.int64) == want_t.view(np.int64)).all()
            assert int(c[1]) == clamps_t
    d.check_dev()


@pytest.mark.parametrize("rows,cols", [(1, 1), (129, 257), (300, 1000), (257, 40)])
@pytest.mark.parametrize("axis", [0, 1, None])
def test_padding_is_written(rows, cols, axis):
    """Padding codes are 0 and padding scale bytes 127, whatever the memory held."""
    torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")  # returned to the allocator dirty
    got = d.mx4_quantize_dev(P["nearest"], source(rows, cols, "bf16", 5), axis=axis)
    for q in got if axis is None else (got,):
        again = d.Mx4.from_parts(*q.to_parts(), cols=q.cols)
        assert torch.equal(again.scales, q.scales.view(-1))
        pad = q.to_parts()[0].cpu().numpy()
        nib = np.stack((pad & 15, pad >> 4), -1).reshape(q.rows, -1)
        assert (nib[:, q.cols:] == 0).all()


def test_exponents_clamp_and_subnormals_cast():
    p = P["nearest"]
    x = torch.tensor([[2.0 ** -140, 2.0 ** -149, 0, -2.0 ** -133] + [0.0] * 28,
                      [3.0e38, -1e38, 1.0, 2e37] + [0.0] * 28], device="cuda")
    want, _ = oracle_rows(x.double().cpu().numpy(), p)
    assert (d.mx4_dequantize_dev(d.mx4_quantize_dev(p, x)).cpu().numpy() == want).all()
    x = x.bfloat16()
    want, _ = oracle_rows(x.double().cpu().numpy(), p)
    assert (d.mx4_dequantize_dev(d.mx4_quantize_dev(p, x)).cpu().numpy() == want).all()
    x = x.T.contiguous()  # the same rows as columns
    got = d.mx4_dequantize_dev(d.mx4_quantize_dev(p, x, axis=0)).cpu().numpy()
    assert (got.view(np.int64) == want.view(np.int64)).all()
    y = torch.tensor([[1e300, -1e290, 5e-324, 1.0] + [0.0] * 28, [1e-300] * 32], device="cuda",
                     dtype=torch.float64)
    want, _ = oracle_rows(y.cpu().numpy(), p)
    assert (d.mx4_dequantize_dev(d.mx4_quantize_dev(p, y)).cpu().numpy() == want).all()


def test_doubles_next_to_a_midpoint_are_not_rounded_twice():
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    v = np.concatenate([mids, np.nextafter(mids, 0), np.nextafter(mids, 9), [4.0], -mids,
                        [0.0] * 3])[:32]
    x = torch.from_numpy(v.reshape(1, 32)).cuda()
    want, _ = oracle_rows(x.cpu().numpy(), P["nearest"])
    got = d.mx4_dequantize_dev(d.mx4_quantize_dev(P["nearest"], x)).cpu().numpy()
    assert (got.view(np.int64) == want.view(np.int64)).all()


@pytest.mark.parametrize("axis", [0, 1])
def test_nan_is_reported_and_held_as_zero(axis):
    x = torch.ones(40, 40, device="cuda")
    x[3, 5] = float("nan")
    q = d.mx4_quantize_dev(P["nearest"], x, axis=axis)
    with pytest.raises(d.DriftError) as e:
        d.check_dev()
    assert e.value.status == d._lib.ENAN_FINITE
    v = d.mx4_dequantize_dev(q).cpu()
    v = v if axis == 1 else v.T
    want = torch.ones(40, 40, dtype=torch.float64)
    want[3, 5] = 0
    assert torch.equal(v, want)


def splitmix(state, k):
    with np.errstate(over="ignore"):
        z = np.uint64(state) + (k.astype(np.uint64) + np.uint64(1)) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return (z ^ (z >> np.uint64(31))) >> np.uint64(11)


def stochastic_rows(x, state, draws):
    """The definition in doubles: element rounded up where its draw is below the
    fraction of the step that truncation drops."""
    rows, cols = x.shape
    out = np.zeros_like(x)
    for b in range(0, cols, 32):
        blk = x[:, b:b + 32]
        amax = np.abs(blk).max(1, keepdims=True)
        e = np.where(amax > 0, np.floor(np.log2(np.where(amax > 0, amax, 1))) - 2, 0)
        a = np.minimum(np.abs(blk) / 2.0 ** e, 6.0)
        step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
        lo = np.floor(a / step) * step
        up = splitmix(state, draws[:, b:b + 32]) * 2.0 ** -53 < (a - lo) / step
        out[:, b:b + 32] = np.copysign((lo + up * step) * 2.0 ** e, blk)
    return out


@pytest.mark.parametrize("dt", ["f64", "f32", "bf16"])
@pytest.mark.parametrize("axis", [0, 1, None])
def test_stochastic_cast_follows_its_stream(dt, axis):
    rows, cols, seed = 70, 90, 0x1234567890ABCDEF
    x = source(rows, cols, dt, 11, edges=False)
    st = torch.tensor([seed], dtype=torch.int64, device="cuda")
    got = d.mx4_quantize_dev(P["sr"], x, axis=axis, d_rng_state=st)
    host, n = x.double().cpu().numpy(), rows * cols
    index = np.arange(n).reshape(rows, cols)
    row, col = got if axis is None else (got, None) if axis == 1 else (None, got)
    if row is not None:
        assert (d.mx4_dequantize_dev(row).cpu().numpy() == stochastic_rows(host, seed, index)).all()
    if col is not None:
        first = n if axis is None else 0
        want = stochastic_rows(np.ascontiguousarray(host.T), seed,
                               np.ascontiguousarray(index.T) + first)
        assert (d.mx4_dequantize_dev(col).cpu().numpy() == want).all()
    drawn = n * (2 if axis is None else 1)
    assert int(st) & (2 ** 64 - 1) == (seed + drawn * 0x9E3779B97F4A7C15) & (2 ** 64 - 1)


@pytest.mark.parametrize("dt", ["bf16", "f32", "f64"])
def test_strided_sources(dt):
    big = source(150, 300, dt, 3, edges=False)
    for x in (big[:, 1:290], big[3:140:2, 7:], big.T, big[:, ::3], big[5:6, 3:9], big[:0], big[:, :0]):
        got = d.mx4_quantize_dev(P["nearest"], x, axis=None)
        want = d.mx4_quantize_dev(P["nearest"], x.clone(memory_format=torch.contiguous_format),
                                  axis=None)
        for a, b in zip(got, want):
            assert a.shape == b.shape and torch.equal(a.codes, b.codes)
            assert torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("dt", list(DT))
def test_values_in_every_type(dt):
    q = d.mx4_quantize_dev(P["nearest"], source(37, 133, "f32", 9, edges=False))
    full = d.mx4_dequantize_dev(q)
    assert torch.equal(d.mx4_dequantize_dev(q, dtype=DT[dt]), full.to(DT[dt]))
    out = torch.zeros(37, 200, dtype=DT[dt], device="cuda")
    d.mx4_dequantize_dev(q, out=out[:, 3:136])
    assert torch.equal(out[:, 3:136], full.to(DT[dt])) and not out[:, 136:].any()


# ------------------------------------------------------------------ the product

GEMMS = [(1, 1, 1), (1, 64, 32), (1, 8192, 256), (2, 100, 4096), (5, 96, 2048), (16, 130, 100),
         (17, 1000, 257), (64, 2048, 2048), (65, 127, 512), (128, 128, 128), (129, 257, 1023),
         (200, 40, 5000), (256, 256, 256), (300, 520, 96), (1001, 333, 777), (2000, 96, 64),
         (33, 4100, 33), (513, 1025, 2049)]


def packed(rows, cols, seed, spread=1.0):
    rs = np.random.default_rng(seed)
    x = heavy_tailed(rs, rows * cols, spread).reshape(rows, cols).astype(np.float32)
    return d.mx4_quantize_dev(P["nearest"], torch.from_numpy(x).cuda())


def bound(a, b, want, dtype):
    """Sums: up to K additions, each off by at most one unit of fp32 in the last
    place of a partial sum, none above sum |a b|; then the rounding to dtype."""
    k = a.shape[1]
    sums = (k + 2) * 2.0 ** -23 * (a.abs() @ b.abs().T)
    if dtype == torch.float64:
        return sums
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half if dtype == torch.float16 else 0.0
    return sums + half * (want.abs() + sums) + tiny


@pytest.mark.parametrize("m,n,k", GEMMS)
@pytest.mark.parametrize("bias", [False, True])
def test_product_against_64_bits(m, n, k, bias):
    A, B = packed(m, k, m + 1), packed(n, k, n + 2)
    a, b = d.mx4_dequantize_dev(A), d.mx4_dequantize_dev(B)
    bv = torch.randn(n, device="cuda") if bias else None
    want = a @ b.T + (bv.double() if bias else 0)
    for dtype in (torch.float32, torch.bfloat16, torch.float16, torch.float64):
        got = d.mx4_gemm_dev(A, B, bias=bv, dtype=dtype)
        assert got.shape == (m, n) and got.dtype == dtype
        lim = bound(a, b, want, dtype)
        if bias:
            lim = lim + 2.0 ** -23 * (want.abs() + bv.double().abs())
        big = want.abs() > 60000 if dtype == torch.float16 else torch.zeros_like(want).bool()
        assert ((got.double() - want).abs() <= lim)[~big].all()
    d.check_dev()


@pytest.mark.parametrize("m,n,k", [(1, 300, 500), (40, 300, 500), (300, 300, 500)])
def test_product_into_a_strided_output_leaves_the_rest(m, n, k):
    A, B = packed(m, k, 1), packed(n, k, 2)
    want = d.mx4_gemm_dev(A, B)
    for lead in (0, 1, 3):
        buf = torch.full((m + 2, n + 7), 5.0, device="cuda")
        d.mx4_gemm_dev(A, B, out=buf[1:m + 1, lead:lead + n])
        assert torch.equal(buf[1:m + 1, lead:lead + n], want)
        buf[1:m + 1, lead:lead + n] = 5.0
        assert (buf == 5.0).all()


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (48, 512, 4096), (600, 512, 4096)])
def test_product_is_the_same_every_time(m, n, k):
    A, B = packed(m, k, 1, 2.0), packed(n, k, 2, 2.0)
    first = d.mx4_gemm_dev(A, B)
    for _ in range(3):
        assert torch.equal(d.mx4_gemm_dev(A, B), first)


def test_products_of_nothing():
    A, B = packed(4, 64, 1), packed(6, 64, 2)
    none = d.mx4_quantize_dev(P["nearest"], torch.zeros(0, 64, device="cuda"))
    assert d.mx4_gemm_dev(none, B).shape == (0, 6) and d.mx4_gemm_dev(A, none).shape == (4, 0)
    thin = [d.mx4_quantize_dev(P["nearest"], torch.zeros(r, 0, device="cuda")) for r in (4, 6)]
    bias = torch.arange(6.0, device="cuda")
    assert torch.equal(d.mx4_gemm_dev(*thin, bias=bias), bias.expand(4, 6))
    assert not d.mx4_gemm_dev(*thin).any()


def test_product_overflows_to_infinity_and_keeps_exact_zeros():
    x = torch.full((130, 64), 3.0e38, device="cuda")
    q = d.mx4_quantize_dev(P["nearest"], x)
    assert torch.isinf(d.mx4_gemm_dev(q, q)).all()
    z = d.mx4_quantize_dev(P["nearest"], torch.zeros(40, 64, device="cuda"))
    assert not d.mx4_gemm_dev(q, z).any()


@pytest.mark.parametrize("m,n,k", [(3, 200, 300), (400, 300, 300)])
@pytest.mark.parametrize("ea,eb", [(-100, 90), (-125, 120), (-128, 120), (-133, 120), (120, -126)])
def test_scales_at_both_ends_of_their_range(m, n, k, ea, eb):
    """Small values times large ones, down to the scale byte 0 (2^-127) and up to
    those near 254: products in fp32's normal range keep their bits. (At 2^-133 the
    exponent is clamped at -127 and every element rounds to zero.)"""
    rs = np.random.default_rng(1)
    A, B = (d.mx4_quantize_dev(P["nearest"], torch.from_numpy(rs.standard_normal((r, k))
                                                              * 2.0 ** e).cuda())
            for r, e in ((m, ea), (n, eb)))
    a, b = d.mx4_dequantize_dev(A), d.mx4_dequantize_dev(B)
    want = a @ b.T
    got = d.mx4_gemm_dev(A, B).double()
    assert ((got - want).abs() <= bound(a, b, want, torch.float32)).all()
    assert want.any() == (ea > -133)


def test_refusals():
    A, B = packed(4, 64, 1), packed(6, 96, 2)
    with pytest.raises(ValueError):
        d.mx4_gemm_dev(A, B)
    with pytest.raises(ValueError):
        d.mx4_gemm_dev(A, A, bias=torch.zeros(5, device="cuda"))
    with pytest.raises(TypeError):
        d.mx4_gemm_dev(A, A, bias=torch.zeros(4, device="cuda", dtype=torch.float64))
    with pytest.raises(TypeError):
        d.mx4_gemm_dev(A, A, dtype=torch.int32)
    with pytest.raises(ValueError):
        d.mx4_gemm_dev(A, A, out=torch.zeros(4, 5, device="cuda"))
    with pytest.raises(ValueError):
        d.mx4_gemm_dev(A, A, out=torch.zeros(8, 4, device="cuda").T[:4].T[:4].T)
    with pytest.raises(TypeError):
        d.mx4_quantize_dev(P["nearest"], torch.zeros(4, 4, dtype=torch.int32, device="cuda"))
    with pytest.raises(d.DriftError):
        d.mx4_quantize_dev(P["sr"], torch.zeros(4, 4, device="cuda"))
    with pytest.raises(ValueError):
        d.mx4_dequantize_dev(A, out=torch.zeros(4, 63, device="cuda"))


@pytest.mark.parametrize("m", [1, 64, 400])
def test_linear_layer_captured_and_replayed(m):
    """Cast and product in a graph, replayed on new inputs; two graphs in flight on
    two streams do not share scratch."""
    n, k = 300, 1000
    W = packed(n, k, 7)
    p = P["nearest"]
    graphs = []
    for g in range(2):
        x = torch.randn(m, k, device="cuda")
        d.mx4_gemm_dev(d.mx4_quantize_dev(p, x), W)  # first use outside the capture
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = d.mx4_gemm_dev(d.mx4_quantize_dev(p, x), W)
        graphs.append((gr, x, y, torch.cuda.Stream()))
    for seed in range(3):
        fresh = [torch.randn(m, k, device="cuda") for _ in graphs]
        want = [d.mx4_gemm_dev(d.mx4_quantize_dev(p, f), W) for f in fresh]
        torch.cuda.synchronize()
        for (gr, x, y, s), f in zip(graphs, fresh):
            with torch.cuda.stream(s):
                x.copy_(f)
                gr.replay()
        torch.cuda.synchronize()
        for (gr, x, y, s), w in zip(graphs, want):
            assert torch.equal(y, w)


def test_a_stream_of_its_own():
    s = torch.cuda.Stream()
    x = torch.randn(200, 640, device="cuda")
    W = packed(300, 640, 7)
    want = d.mx4_gemm_dev(d.mx4_quantize_dev(P["nearest"], x), W)
    torch.cuda.synchronize()
    q = d.mx4_quantize_dev(P["nearest"], x, stream=s)
    got = d.mx4_gemm_dev(q, W, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    got = d.mx4_gemm_dev(a=q, b=W, stream=s)
    s.synchronize()
    assert torch.equal(got, want)


def test_types_are_the_header_s():
    assert _types()[torch.float64] == 0 and _types()[torch.float16] == 3
