"""AdamW over many tensors, on the GPU, against the same operations in numpy's
fp32 (the moments and codes bit for bit) and the formula in 64 bits."""
import numpy as np
import pytest

import drift_b200 as d

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F = np.float32
HYP = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.1)
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = [1, 7, 8, 255, 256, 257, 4095, 4096, 4097, 10001]


def to8(x):
    """Codes (as their values) and scales of a float32 vector, block by block."""
    n = x.size
    b = np.zeros((-(-n // 256), 256), dtype=F)
    b.reshape(-1)[:n] = x
    amax = np.abs(b).max(1, keepdims=True)
    tiny = amax < F(2.0 ** -100)
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.where(tiny, F(0), (F(1) / amax) * F(448))
    y = np.clip(b * inv, F(-448), F(448))
    code = torch.from_numpy(y.reshape(-1)[:n].copy()).to(torch.float8_e4m3fn)
    return code, np.where(tiny, F(1), amax * (F(1) / F(448)))[:, 0].astype(F)


def from8(code, scale):
    n = code.numel()
    return (code.float().numpy() * np.repeat(scale, 256)[:n]).astype(F)


def fma(a, b, c):
    """Rounded once: the product of two floats is exact in the wider type, and the
    sum's 64 bits leave fp32's rounding where it was but for a tie's neighbourhood."""
    wide = np.longdouble
    return (wide(a) * np.asarray(b, dtype=wide) + np.asarray(c, dtype=wide)).astype(F)


def update(p, g, m, v, step):
    """One step of one tensor: each operation rounded to fp32."""
    b1, b2 = HYP["betas"]
    a1, rc2 = F(HYP["lr"] / (1 - b1 ** step)), F(1 / np.sqrt(1 - b2 ** step))
    m = F(b1) * m + F(1 - b1) * g
    v = F(b2) * v + (F(1 - b2) * g) * g
    r = np.sqrt(v)
    u = (a1 * m) / fma(rc2, r, F(HYP["eps"]))
    return fma(F(1 - HYP["lr"] * HYP["weight_decay"]), p, -u), m, v, r, u


def tensors(sizes, pt, gt, seed, offset=0):
    g = torch.Generator().manual_seed(seed)

    def make(n, scale, dt):
        return (torch.randn(n + offset, generator=g) * scale).to(DT[dt]).cuda()[offset:]

    return [make(n, 0.05, pt) for n in sizes], [[make(n, 1e-2, gt) for n in sizes]
                                                for _ in range(3)]


def near(got, want, u, dtype):
    """The two scalars of a step come from the device's pow, each within a unit of
    fp32 of numpy's; the quotient is a product with a reciprocal, within two, of a
    root within one; the plain quotient and root have their own halves: the update is
    within six units. Then one
    rounding to the type (and its subnormals), where the plain value's own rounding
    may fall on the other side."""
    err = np.abs(got.double().cpu().numpy() - want.astype(np.float64))
    eps = torch.finfo(dtype).eps
    assert (err <= 6 * 2.0 ** -23 * np.abs(u) + eps * np.abs(want) + 2.0 ** -24).all()


@pytest.mark.parametrize("pt,gt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"),
                                   ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("offset", [0, 1])
def test_moments_in_32_bits(pt, gt, offset):
    params, steps = tensors(SIZES, pt, gt, 5, offset)
    opt = d.AdamW(params, **HYP)
    m = [np.zeros(n, F) for n in SIZES]
    v = [np.zeros(n, F) for n in SIZES]
    for t, grads in enumerate(steps, 1):
        before = [p.float().cpu().numpy() for p in params]
        opt.step(grads)
        for i in range(len(SIZES)):
            want, m[i], v[i], _, u = update(before[i], grads[i].float().cpu().numpy(), m[i], v[i], t)
            assert (opt.state[0][i].cpu().numpy() == m[i]).all()
            assert (opt.state[1][i].cpu().numpy() == v[i]).all()
            near(params[i], want, u, DT[pt])
    assert int(opt.d_step) == 3


@pytest.mark.parametrize("pt,gt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("offset", [0, 1])
def test_moments_in_8_bits(pt, gt, offset):
    params, steps = tensors(SIZES, pt, gt, 6, offset)
    opt = d.AdamW(params, state_bits=8, **HYP)
    held = [[to8(np.zeros(n, F)) for n in SIZES] for _ in range(2)]
    held = [[(c, np.zeros_like(s)) for c, s in x] for x in held]  # a fresh state's scales are 0
    for t, grads in enumerate(steps, 1):
        before = [p.float().cpu().numpy() for p in params]
        opt.step(grads)
        for i in range(len(SIZES)):
            m, r = from8(*held[0][i]), from8(*held[1][i])
            want, m, _, r, u = update(before[i], grads[i].float().cpu().numpy(), m, r * r, t)
            held[0][i], held[1][i] = to8(m), to8(r)
            near(params[i], want, u, DT[pt])
            code, scale = (opt.state[k][i].cpu() for k in (0, 1))
            assert (code.view(torch.uint8) == held[0][i][0].view(torch.uint8)).all()
            assert (scale.numpy() == held[0][i][1]).all()
            # The root is within a unit of the nearest float, and so is a block's
            # largest, its scale with it: x / scale is within 3 units of the plain one,
            # and the code within that of a nearest one. The device's state goes on.
            code, scale = opt.state[2][i].cpu(), opt.state[3][i].cpu().numpy()
            assert (np.abs(scale - held[1][i][1]) <= 2 * 2.0 ** -23 * scale).all()
            y = r / np.repeat(held[1][i][1], 256)[:r.size].astype(np.float64)
            got = code.double().numpy()
            step = 2.0 ** np.maximum(np.floor(np.log2(np.maximum(got, 2.0 ** -9))) - 3, -9)
            assert (np.abs(got - y) <= step / 2 + 4 * 2.0 ** -23 * y).all()
            held[1][i] = (code, scale)


def test_against_the_formula_in_64_bits():
    """Ten steps in double: every fp32 operation of a step is off by half a unit,
    and ten steps of fewer than sixteen operations by less than 160 halves."""
    params, _ = tensors([5000], "f32", "f32", 7)
    p = params[0].double().cpu().numpy()
    opt = d.AdamW(params, **HYP)
    (b1, b2), m, v = HYP["betas"], 0.0, 0.0
    path = np.abs(p)
    for t in range(1, 11):
        g = torch.randn(5000, device="cuda") * 1e-2
        opt.step([g])
        gd = g.double().cpu().numpy()
        m, v = b1 * m + (1 - b1) * gd, b2 * v + (1 - b2) * gd * gd
        u = HYP["lr"] * (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + HYP["eps"])
        p = p * (1 - HYP["lr"] * HYP["weight_decay"]) - u
        # the first moment's own rounding, relative to its terms, not to their sum
        path = path + np.abs(p) + HYP["lr"] * 10
    assert (np.abs(params[0].double().cpu().numpy() - p) <= 160 * 2.0 ** -24 * path).all()


def test_without_decay_it_is_the_trainer_s_adam():
    """drift_adam_dev in double, at betas 0.9 and 0.999 and eps 1e-8, one step:
    fp32 operations against double, fewer than sixteen."""
    n = 3000
    p = torch.randn(n, device="cuda")
    g = torch.randn(n, device="cuda") * 1e-3
    p64, m64, v64 = p.double(), torch.zeros(n, device="cuda").double(), torch.zeros(n, device="cuda").double()
    before = p.clone()
    d.AdamW([p], lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0).step([g])
    ctx = d.Context.current()
    g64 = g.double()
    d._lib.check(d._lib.load().drift_adam_dev(ctx.handle, p64.data_ptr(), g64.data_ptr(),
                                              m64.data_ptr(), v64.data_ptr(), n, 1, 1e-3, 0,
                                              torch.cuda.current_stream().cuda_stream))
    # u = lr g / (|g| + eps) here: 16 halves of 1e-3, and the last rounding of p
    lim = 16 * 2.0 ** -24 * 1e-3 + 2.0 ** -24 * before.double().abs() + 2.0 ** -24 * 1e-3
    assert ((p.double() - p64).abs() <= lim).all()


def test_many_tensors_copies_skips_and_scaled_gradients():
    """More tensors than one launch takes, empty ones, gradients that are None,
    low-precision copies and a gradient scale; equal to the tensors one by one."""
    sizes = [(37 * i) % 900 for i in range(300)]
    params, _ = tensors(sizes, "f32", "bf16", 8)
    twin = [p.clone() for p in params]
    copies = [torch.empty(n, dtype=torch.bfloat16, device="cuda") if i % 3 else None
              for i, n in enumerate(sizes)]
    scale = torch.tensor([0.125], device="cuda")
    opt = d.AdamW(params, copies=copies, **HYP)
    solo = [d.AdamW([t], **HYP) for t in twin]
    for step in range(2):
        grads = [torch.randn(n, device="cuda").bfloat16() if (i + step) % 5 else None
                 for i, n in enumerate(sizes)]
        opt.step(grads, d_grad_scale=scale)
        for s, g in zip(solo, grads):
            s.step([None if g is None else g.float() * 0.125])
    for i, (a, b) in enumerate(zip(params, twin)):
        assert torch.equal(a, b)
        if copies[i] is not None and sizes[i]:
            assert torch.equal(copies[i], a.bfloat16()) or grads[i] is None


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_as_the_next(bits):
    params, steps = tensors([1000, 5000], "f32", "f32", 9)
    twin = [p.clone() for p in params]
    a, b = (d.AdamW(x, state_bits=bits, **HYP) for x in (params, twin))
    held = [torch.zeros_like(g) for g in steps[0]]
    lr = torch.tensor([1e-3], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(held, d_lr=lr)
    for k, grads in enumerate(steps):
        lr.fill_(1e-3 * (k + 1))
        for h, g in zip(held, grads):
            h.copy_(g)
        graph.replay()
        b.step(grads, d_lr=lr)
        for x, y in zip(params, twin):
            assert torch.equal(x, y)
        for x, y in zip(a.state, b.state):
            assert all(torch.equal(s.view(torch.uint8) if bits == 8 and s.dtype != torch.float32
                                   else s, t.view(torch.uint8)
                                   if bits == 8 and t.dtype != torch.float32 else t)
                       for s, t in zip(x, y))
    assert int(a.d_step) == len(steps)


def test_stochastic_codes_are_neighbours_and_unbiased():
    n = 256 * 64
    g = torch.randn(n, device="cuda") * 1e-2
    st = torch.tensor([99], dtype=torch.int64, device="cuda")
    total = np.zeros(n)
    runs = 200
    for k in range(runs):
        p = torch.zeros(n, device="cuda")
        opt = d.AdamW([p], state_bits=8, rounding=d.Rounding.STOCHASTIC, d_rng_state=st, **HYP)
        opt.step([g])
        total += from8(opt.state[0][0].cpu(), opt.state[1][0].cpu().numpy())
    assert int(st) & (2 ** 64 - 1) == (99 + runs * n * 0x9E3779B97F4A7C15) & (2 ** 64 - 1)
    m = (F(1 - 0.9) * g.cpu().numpy()).astype(F)
    s = opt.state[1][0].cpu().numpy().repeat(256)
    y = np.abs(m) / s
    quantum = np.where(y < 2.0 ** -6, 2.0 ** -9, 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)) * s
    last = from8(opt.state[0][0].cpu(), opt.state[1][0].cpu().numpy())
    assert (np.abs(last - m) <= quantum * 1.0001).all()
    # One draw's spread is at most half a quantum, so the mean of 200 over all n
    # elements, in quanta, is within 6 / (2 sqrt(200 n)) of 0.
    bias = ((total / runs - m) / quantum).mean()
    assert abs(bias) <= 6 / (2 * np.sqrt(runs * n))


def test_zero_and_non_finite_blocks():
    p = torch.ones(768, device="cuda")
    g = torch.zeros(768, device="cuda")
    g[300] = float("inf")
    g[600] = 1e-20
    opt = d.AdamW([p], state_bits=8, lr=1e-3, weight_decay=0.0)
    opt.step([g])
    m, ms, r, rs = (x[0].cpu() for x in opt.state)
    assert not m[:256].float().any() and ms[0] == 1 and rs[0] == 1
    assert torch.isnan(ms[1]) and torch.isnan(m[256:512].float()).all()
    assert m[600].float() == 448 and m[512:600].float().abs().max() == 0
    assert (p[:256] == 1).all() and torch.isfinite(p[512:]).all()


def test_memory_taken_at_construction_is_kept_and_replacing_it_is_refused():
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt, ref = d.AdamW([p.clone()]), d.AdamW([p])
    opt.state[0][0] = torch.zeros(300, device="cuda")  # the list's, not the optimizer's
    junk = [torch.full((300,), float("nan"), device="cuda") for _ in range(8)]
    for _ in range(2):
        opt.step([g])
        ref.step([g])
    assert torch.equal(opt.params[0], ref.params[0])
    assert all(torch.isnan(j).all() for j in junk)
    opt.params[0].data = torch.ones(300, device="cuda")
    with pytest.raises(ValueError):
        opt.step([g])


def test_refusals():
    p = torch.zeros(8, device="cuda")
    opt = d.AdamW([p])
    with pytest.raises(ValueError):
        opt.step([])
    with pytest.raises(ValueError):
        opt.step([torch.zeros(9, device="cuda")])
    with pytest.raises(ValueError):
        opt.step([torch.zeros(8)])
    with pytest.raises(ValueError):
        opt.step([torch.zeros(8, dtype=torch.float64, device="cuda")])
    with pytest.raises(ValueError):
        opt.step([torch.zeros(16, device="cuda")[::2]])
    with pytest.raises(TypeError):
        d.AdamW([torch.zeros(8, dtype=torch.float64, device="cuda")])
    with pytest.raises(ValueError):
        d.AdamW([torch.zeros(4, 4, device="cuda").T[:2].T])
    with pytest.raises(ValueError):
        d.AdamW([p, p])
    with pytest.raises(ValueError):
        d.AdamW([p, p[4:]])
    m = torch.zeros(8, device="cuda")
    with pytest.raises(ValueError):
        d.AdamW([p], state=[[m], [m]])
    with pytest.raises(ValueError):
        d.AdamW([p], copies=[p])
    with pytest.raises(d.DriftError):
        d.AdamW([p], eps=1e-35).step([torch.zeros(8, device="cuda")])
    with pytest.raises(d.DriftError):
        d.AdamW([p], betas=(1.0, 0.9)).step([torch.zeros(8, device="cuda")])
