"""Linear softmax cross entropy without kept logits, on the GPU, against the
formulas in 64 bits and against differences."""
import pytest

import drift_b200 as d

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

IG = -100
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def inputs(t, dep, v, dt="bf16", bias=True, ignored=0.2, seed=0, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * t + v)
    x = torch.randn(t, dep, device="cuda", generator=g).to(DT[dt])
    w = (torch.randn(v, dep, device="cuda", generator=g) * scale * dep ** -0.5).to(DT[dt])
    b = torch.randn(v, device="cuda", generator=g) * 0.3 if bias else None
    tg = torch.randint(0, v, (t,), device="cuda", generator=g)
    drop = torch.rand(t, device="cuda", generator=g) < ignored
    return x, w, torch.where(drop, IG, tg), b


def exact(x, w, tg, b, g=None):
    """Losses, log sums, d and the gradients in double."""
    x, w = x.double(), w.double()
    logits = x @ w.T + (0 if b is None else b.double())
    lse = torch.logsumexp(logits, 1)
    on = tg != IG
    at = torch.where(on, tg, 0).long()[:, None]
    loss = torch.where(on, lse - logits.gather(1, at)[:, 0], 0.0)
    if g is None:
        return loss, lse
    p = torch.softmax(logits, 1)
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    dl = (p - one) * (g.double() * on)[:, None]
    return loss, lse, p, dl, dl @ w, dl.T @ x, dl.sum(0)


def logit_error(x, w, b):
    """How far a logit may be off: depth additions, each within one unit of fp32
    of the largest partial sum, and the bias added."""
    mag = x.double().abs() @ w.double().abs().T + (0 if b is None else b.double().abs())
    return (x.shape[1] + 2) * 2.0 ** -23 * mag


def check_losses(x, w, tg, b, loss, lse):
    want, z = exact(x, w, tg, b)
    # A log sum moves by at most the largest logit error, and by the sum's own
    # roundings: fewer than 2^6 units of fp32 from the exponentials (2 each), the
    # pairwise joins (each rescales by one more exponential) and the logarithm.
    e = logit_error(x, w, b).amax(1) + 2.0 ** -17 + 2.0 ** -22 * z.abs()
    assert ((lse.double() - z).abs() <= e).all()
    assert ((loss.double() - want).abs() <= 2 * e + 2.0 ** -22 * want.abs()).all()
    assert (loss[tg == IG] == 0).all()


SHAPES = [(1, 8, 1), (1, 64, 96), (1, 2048, 5000), (3, 16, 7), (64, 2048, 96), (65, 40, 257),
          (127, 128, 129), (128, 256, 256), (300, 72, 1000), (257, 520, 3001), (2, 1024, 20011),
          (1000, 64, 33)]


@pytest.mark.parametrize("t,dep,v", SHAPES)
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("bias", [False, True])
def test_losses(t, dep, v, dt, bias):
    x, w, tg, b = inputs(t, dep, v, dt, bias)
    loss, lse = d.linear_xent_dev(x, w, tg, bias=b)
    check_losses(x, w, tg, b, loss, lse)
    again = d.linear_xent_dev(x, w, tg.int(), bias=b)
    assert torch.equal(again[0], loss) and torch.equal(again[1], lse)
    d.check_dev()


def check_grads(x, w, tg, b, g, got):
    """d is off by its exponential's argument (two logit errors) and its 16-bit
    rounding; the products' sums by one unit of fp32 an addition; results by
    their rounding. Everything relative to sums of magnitudes."""
    dx, dw, db = got
    _, z, p, dl, wx, ww, wb = exact(x, w, tg, b, g)
    half = torch.finfo(x.dtype).eps / 2
    e = logit_error(x, w, b)
    e = e + e.amax(1, keepdim=True) + 2.0 ** -17 + 2.0 ** -22 * z.abs()[:, None]
    on = (g.double().abs() * (tg != IG))[:, None]
    soft = p * torch.expm1(e.clamp(max=10.0)) * on + 2.0 ** -22 * dl.abs()
    # f16 holds d scaled by a power of two near 2^15 / max |g|, so that its
    # smallest step, 2^-24, stands for 2^-38 of the largest gradient.
    floor = 2.0 ** -38 * float(g.abs().max()) * (on > 0) if x.dtype == torch.float16 else 0.0
    el = soft + half * (dl.abs() + soft) + floor
    X, W = x.double().abs(), w.double().abs()
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0  # half a step of f16's subnormals
    if dx is not None:
        lim = (el + (w.shape[0] + 2) * 2.0 ** -23 * dl.abs()) @ W
        assert ((dx.double() - wx).abs() <= lim + half * (wx.abs() + lim) + tiny).all()
        assert (dx[tg == IG] == 0).all()
    if dw is not None:
        lim = (el + (x.shape[0] + 2) * 2.0 ** -23 * dl.abs()).T @ X
        assert ((dw.double() - ww).abs() <= lim + half * (ww.abs() + lim) + tiny).all()
    if db is not None:
        lim = (soft + (x.shape[0] + 2) * 2.0 ** -23 * dl.abs()).sum(0)
        assert ((db.double() - wb).abs() <= lim).all()


@pytest.mark.parametrize("t,dep,v", SHAPES)
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("bias", [False, True])
def test_gradients(t, dep, v, dt, bias):
    x, w, tg, b = inputs(t, dep, v, dt, bias, seed=1)
    g = torch.randn(t, device="cuda")
    _, lse = d.linear_xent_dev(x, w, tg, bias=b)
    got = d.linear_xent_grad_dev(x, w, tg, lse, g, bias=b)
    check_grads(x, w, tg, b, g, got)
    assert (got[2] is not None) == bias
    # one weight for all rows, and the parts on their own
    one = torch.tensor([0.25], device="cuda")
    both = d.linear_xent_grad_dev(x, w, tg, lse, one, bias=b)
    check_grads(x, w, tg, b, one.expand(t), both)
    left = d.linear_xent_grad_dev(x, w, tg, lse, one, bias=b, need_dw=False)
    right = d.linear_xent_grad_dev(x, w, tg, lse, one, bias=b, need_dx=False)
    assert left[1] is None and right[0] is None
    assert torch.equal(left[0], both[0]) and torch.equal(right[1], both[1])


@pytest.mark.parametrize("t,dep,v", [(64, 2048, 96), (200, 136, 2500)])
@pytest.mark.parametrize("ignored", [0.0, 0.3, 1.0])
def test_mean_loss_and_its_gradients(t, dep, v, ignored):
    x, w, tg, b = inputs(t, dep, v, ignored=ignored, seed=2)
    loss, dx, dw, db = d.linear_xent_mean_dev(x, w, tg, bias=b)
    n = max(1, int((tg != IG).sum()))
    rows, _ = d.linear_xent_dev(x, w, tg, bias=b)
    want = rows.double().sum() / n
    assert abs(float(loss) - float(want)) <= 2.0 ** -22 * abs(float(want)) * 12
    check_grads(x, w, tg, b, torch.full((t,), 1.0 / n, device="cuda"), (dx, dw, db))
    if ignored == 1.0:
        assert float(loss) == 0 and not dx.any() and not dw.any() and not db.any()


def test_the_gradient_against_differences():
    """The mean loss, in double, along a random direction of x, w and bias."""
    x, w, tg, b = inputs(40, 64, 300, seed=3)
    _, dx, dw, db = d.linear_xent_mean_dev(x, w, tg, bias=b)
    n = int((tg != IG).sum())
    gen = torch.Generator(device="cuda").manual_seed(4)
    ux, uw, ub = (torch.randn(a.shape, device="cuda", generator=gen, dtype=torch.float64)
                  for a in (x, w, b))

    def mean(h):
        return float(exact(x.double() + h * ux, w.double() + h * uw, tg, b.double() + h * ub)[0].sum() / n)

    h = 1e-4
    slope = (mean(h) - mean(-h)) / (2 * h)
    got = float((dx.double() * ux).sum() + (dw.double() * uw).sum() + (db.double() * ub).sum())
    # d's and the results' roundings, 2^-8 each at most and independent: far below
    # their sum of magnitudes; differences in double leave h^2.
    mags = float((dx.double() * ux).abs().sum() + (dw.double() * uw).abs().sum())
    assert abs(got - slope) <= 2 * 2.0 ** -8 * mags / 10 + 1e-5


@pytest.mark.parametrize("bias", [False, True])
def test_strides_and_odd_depths(bias):
    """Rows apart, depths that are not whole groups of eight, and views: equal to
    the contiguous call's, or to one padded with zero columns."""
    t, v = 70, 300
    for dep, lead in ((40, 8), (37, 0), (1, 0), (33, 3)):
        big_x = torch.randn(t, dep + 24, device="cuda").bfloat16()
        big_w = torch.randn(v, dep + 24, device="cuda").bfloat16()
        x, w = big_x[:, lead:lead + dep], big_w[:, lead:lead + dep]
        tg = torch.randint(0, v, (t,), device="cuda")
        b = torch.randn(v, device="cuda") if bias else None
        pad = (-dep) % 8
        zx, zw = (torch.nn.functional.pad(a, (0, pad)).contiguous() for a in (x, w))
        got = d.linear_xent_mean_dev(x, w, tg, bias=b)
        want = d.linear_xent_mean_dev(zx, zw, tg, bias=b)
        assert torch.equal(got[0], want[0])
        assert got[1].shape == (t, dep) and torch.equal(got[1], want[1][:, :dep])
        assert got[2].shape == (v, dep) and torch.equal(got[2], want[2][:, :dep])
        xt = x.T.contiguous().T
        assert torch.equal(d.linear_xent_mean_dev(xt, w, tg, bias=b)[1], got[1])


def test_masked_vocabulary_entries_and_far_logits():
    """A bias of -inf takes an entry out; the type's lowest value does too; logits
    of hundreds neither overflow nor lose the loss."""
    x, w, tg, b = inputs(130, 64, 700, ignored=0.0, seed=5, scale=60.0)
    for low in (float("-inf"), torch.finfo(torch.float32).min):
        tg = tg % 300
        masked = b.clone()
        masked[300:] = low
        loss, lse = d.linear_xent_dev(x, w, tg, bias=masked)
        check_losses(x, w[:300], tg, b[:300], loss, lse)
        _, dx, dw, db = d.linear_xent_mean_dev(x, w, tg, bias=masked)
        assert not dw[300:].any() and not db[300:].any()
        assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


def test_a_row_without_any_entry_and_nan_inputs():
    x, w, tg, b = inputs(66, 64, 500, ignored=0.0, seed=6)
    x = x.clone()
    x[7] = float("nan")
    loss, lse = d.linear_xent_dev(x, w, tg, bias=b)
    bad = torch.isnan(loss)
    assert bad[7] and int(bad.sum()) == 1 and torch.isnan(lse[7])
    off = torch.full_like(b, float("-inf"))
    loss, lse = d.linear_xent_dev(x, w, tg, bias=off)
    assert not torch.isfinite(lse).any() and not torch.isfinite(loss).any()


@pytest.mark.parametrize("t,v", [(70, 300), (70, 40000)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_ignored_rows_may_hold_anything(t, v, bad):
    """Padded positions full of NaN or Inf: losses and gradients as with zeros there."""
    x, w, tg, b = inputs(t, 72, v, ignored=0.3, seed=9)
    clean, dirty = x.clone(), x.clone()
    clean[tg == IG] = 0
    dirty[tg == IG] = bad
    for bias in (None, b):
        want = d.linear_xent_mean_dev(clean, w, tg, bias=bias)
        got = d.linear_xent_mean_dev(dirty, w, tg, bias=bias)
        for a, c in zip(got, want):
            assert (a is None and c is None) or torch.equal(a, c)
        loss, lse = d.linear_xent_dev(dirty, w, tg, bias=bias)
        assert torch.equal(loss, d.linear_xent_dev(clean, w, tg, bias=bias)[0])
        g = torch.randn(t, device="cuda")
        for a, c in zip(d.linear_xent_grad_dev(dirty, w, tg, lse, g, bias=bias),
                        d.linear_xent_grad_dev(clean, w, tg, lse, g, bias=bias)):
            assert (a is None and c is None) or torch.equal(a, c)


def test_targets_outside_the_vocabulary():
    x, w, tg, b = inputs(20, 32, 50, ignored=0.0, seed=7)
    for wrong in (50, -1, 2 ** 40, -2 ** 40):
        bad = tg.clone()
        bad[3] = wrong
        loss, lse = d.linear_xent_dev(x, w, bad, bias=b)
        with pytest.raises(d.DriftError) as e:
            d.check_dev()
        assert e.value.status == d._lib.EINVAL
        assert loss[3] == 0
        _, dx, _, _ = d.linear_xent_mean_dev(x, w, bad, bias=b)
        assert not dx[3].any()
        with pytest.raises(d.DriftError):
            d.check_dev()
    # ignore_index may be a vocabulary entry
    loss, _ = d.linear_xent_dev(x, w, tg, bias=b, ignore_index=int(tg[0]))
    assert (loss[tg == tg[0]] == 0).all()
    d.check_dev()


def test_no_rows():
    x, w = torch.zeros(0, 32, device="cuda").bfloat16(), torch.ones(9, 32, device="cuda").bfloat16()
    tg = torch.zeros(0, dtype=torch.int64, device="cuda")
    loss, lse = d.linear_xent_dev(x, w, tg)
    assert loss.shape == lse.shape == (0,)
    loss, dx, dw, db = d.linear_xent_mean_dev(x, w, tg, bias=torch.zeros(9, device="cuda"))
    assert float(loss) == 0 and dx.shape == (0, 32) and not dw.any() and not db.any()


@pytest.mark.parametrize("t,dep,v", [(1, 64, 5000), (64, 256, 96), (500, 256, 4000)])
def test_captured_replayed_and_repeated(t, dep, v):
    x, w, tg, b = inputs(t, dep, v, ignored=0.0, seed=8)
    first = d.linear_xent_mean_dev(x, w, tg, bias=b)
    held = (torch.zeros_like(x), w, torch.zeros_like(tg), b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = d.linear_xent_mean_dev(held[0], held[1], held[2], bias=held[3])
    held[0].copy_(x)
    held[2].copy_(tg)
    graph.replay()
    for a, c in zip(out, first):
        assert torch.equal(a, c)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for a, c in zip(d.linear_xent_mean_dev(x, w, tg, bias=b, stream=s), first):
        s.synchronize()
        assert torch.equal(a, c)


def test_refusals():
    x, w, tg, b = inputs(4, 32, 9)
    with pytest.raises(TypeError):
        d.linear_xent_dev(x.float(), w.float(), tg)
    with pytest.raises(TypeError):
        d.linear_xent_dev(x, w.half(), tg)
    with pytest.raises(ValueError):
        d.linear_xent_dev(x, w[:, :24], tg)
    with pytest.raises(ValueError):
        d.linear_xent_dev(x, w, tg[:3])
    with pytest.raises(TypeError):
        d.linear_xent_dev(x, w, tg.float())
    with pytest.raises(ValueError):
        d.linear_xent_dev(x, w, tg, bias=b[:8])
    with pytest.raises(ValueError):
        d.linear_xent_dev(x, w[:0], tg)
    with pytest.raises(ValueError):
        d.linear_xent_grad_dev(x, w, tg, torch.zeros(3, device="cuda"), torch.ones(1, device="cuda"))
    with pytest.raises(ValueError):
        d.linear_xent_grad_dev(x, w, tg, torch.zeros(4, device="cuda"), torch.ones(3, device="cuda"))
