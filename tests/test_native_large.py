"""The native operators where offsets pass 32 bits, against themselves on the rows
that lie there alone (whose values the other tests compare with the formulas), and
calls of two threads at once."""
import threading

import pytest

import drift_b200 as d
from tests.test_native_mx4 import bound
from tests.test_native_xent import IG, check_grads, check_losses

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

P = d.policies.by_name("mxfp4")


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB free")
    yield
    torch.cuda.empty_cache()


def rand(*shape, dt=torch.bfloat16, seed=1, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=dt).mul_(scale)


def test_a_cast_of_more_than_2_31_elements():
    rows, cols = 70_001, 40_008
    x = rand(rows, cols)
    q, qt = d.mx4_quantize_dev(P, x, axis=None)
    back = d.mx4_dequantize_dev(q, dtype=torch.bfloat16)
    for r in (0, 53_700, rows - 1):  # 53 700 x 40 008 is just past 2^31
        one = d.mx4_quantize_dev(P, x[r:r + 1])
        assert torch.equal(q.codes.view(rows, -1)[r], one.codes.view(-1))
        assert torch.equal(back[r:r + 1], d.mx4_dequantize_dev(one, dtype=torch.bfloat16))
    back = d.mx4_dequantize_dev(qt, dtype=torch.bfloat16)
    for c in (0, 30_700, cols - 1):
        one = d.mx4_quantize_dev(P, x[:, c:c + 1].t().contiguous())
        assert torch.equal(back[c:c + 1], d.mx4_dequantize_dev(one, dtype=torch.bfloat16))
    y = d.mx4_gemm_dev(q, d.mx4_quantize_dev(P, x[:200]))
    top = d.mx4_dequantize_dev(q, dtype=torch.float32)[-200:].double()
    low = d.mx4_dequantize_dev(d.mx4_quantize_dev(P, x[:200]))
    want = top @ low.T
    assert ((y[-200:].double() - want).abs() <= bound(top, low, want, torch.float32)).all()


def test_a_product_of_more_than_2_31_elements():
    m, n, k = 66_003, 40_005, 64
    a, b = rand(m, k), rand(n, k, seed=2)
    y = d.mx4_gemm_dev(d.mx4_quantize_dev(P, a), d.mx4_quantize_dev(P, b), dtype=torch.bfloat16)
    for lo, hi in ((0, 300), (53_600, 53_900), (m - 300, m)):
        va, vb = (d.mx4_dequantize_dev(d.mx4_quantize_dev(P, t)) for t in (a[lo:hi], b))
        want = va @ vb.T
        assert ((y[lo:hi].double() - want).abs() <= bound(va, vb, want, torch.bfloat16)).all()


def test_tokens_times_depth_past_2_31():
    """All rows but the first and the last 300 are ignored, so that the gradients are
    those 600 rows' alone."""
    t, dep, v = 1_050_003, 2056, 40
    x, w = rand(t, dep, scale=0.5), rand(v, dep, seed=2, scale=0.05)
    tg = torch.full((t,), IG, device="cuda")
    on = torch.cat((torch.arange(300), torch.arange(t - 300, t))).cuda()
    tg[on] = torch.arange(600, device="cuda") % v
    loss, lse = d.linear_xent_dev(x, w, tg)
    xs, ts = x[on], tg[on]
    check_losses(xs, w, ts, None, loss[on], lse[on])
    assert int((loss != 0).sum()) == 600
    mean, dx, dw, _ = d.linear_xent_mean_dev(x, w, tg)
    # The rows' losses are positive and at most 600 additions move their sum.
    assert abs(float(mean) - float(loss.double().sum()) / 600) <= 602 * 2.0 ** -24 * float(mean)
    g = torch.full((600,), 1 / 600, device="cuda")
    check_grads(xs, w, ts, None, g, (dx[on], dw, None))
    assert not dx[300:t - 300].any()


def test_vocabulary_times_depth_past_2_31():
    t, dep, v = 3, 2000, 1_100_001
    x, w = rand(t, dep, scale=0.5), rand(v, dep, seed=2, scale=0.05)
    tg = torch.tensor([v - 1, 5, 1_073_800], device="cuda")
    loss, lse = d.linear_xent_dev(x, w, tg)
    X = x.double()
    parts = [p.double() for p in w.split(100_000)]
    logits = torch.cat([X @ p.T for p in parts], 1)
    e = (dep + 2) * 2.0 ** -23 * torch.cat([X.abs() @ p.abs().T for p in parts], 1)
    z = logits.logsumexp(1)
    want = z - logits[range(t), tg]
    # As for the smaller shapes: the largest logit error, and the sum's roundings.
    most = e.amax(1) + 2.0 ** -17 + 2.0 ** -22 * z.abs()
    assert ((lse.double() - z).abs() <= most).all()
    assert ((loss.double() - want).abs() <= 2 * most + 2.0 ** -22 * want.abs()).all()
    mean, dx, dw, _ = d.linear_xent_mean_dev(x, w, tg)
    p = torch.softmax(logits, 1) / t
    dl = p.clone()
    dl[range(t), tg] -= 1 / t
    e = e + e.amax(1, keepdim=True) + 2.0 ** -17 + 2.0 ** -22 * z.abs()[:, None]
    soft = p * torch.expm1(e) + 2.0 ** -22 * dl.abs()
    el = soft + 2.0 ** -8 * (dl.abs() + soft)
    for lo in (0, 1_073_700, v - 300):
        c = slice(lo, lo + 300)
        want = dl[:, c].T @ X
        lim = (el + (t + 2) * 2.0 ** -23 * dl.abs())[:, c].T @ X.abs()
        assert ((dw[c].double() - want).abs() <= lim + 2.0 ** -8 * (want.abs() + lim)).all()
    want, lim, at = 0, 0, 0
    for q in parts:
        c = slice(at, at + len(q))
        want = want + dl[:, c] @ q
        lim = lim + (el + (v + 2) * 2.0 ** -23 * dl.abs())[:, c] @ q.abs()
        at += len(q)
    assert ((dx.double() - want).abs() <= lim + 2.0 ** -8 * (want.abs() + lim)).all()


def test_a_tensor_of_more_than_2_31_parameters():
    n = (1 << 31) + 777
    p, g = rand(n, scale=0.02), rand(n, seed=2, scale=1e-3)
    spans = [(0, 4096), ((1 << 31) - 2048, (1 << 31) + 512), (n - 777 - 256, n)]
    parts = [p[a:b].clone() for a, b in spans]
    opt, small = d.AdamW([p], state_bits=8), d.AdamW(parts, state_bits=8)
    for _ in range(2):
        opt.step([g])
        small.step([g[a:b].clone() for a, b in spans])
    for i, (a, b) in enumerate(spans):
        assert torch.equal(p[a:b], parts[i])
        for k in (0, 2):  # the codes of the moment and of the root
            assert torch.equal(opt.state[k][0][a:b].view(torch.uint8),
                               small.state[k][i].view(torch.uint8))


def test_two_threads_at_once():
    def work(seed, out, stream):
        x, w = rand(100, 512, seed=seed), rand(300, 512, seed=seed + 1, scale=0.05)
        tg = torch.arange(100, device="cuda") * 2
        torch.cuda.current_stream().synchronize()
        got = []
        for _ in range(20):
            y = d.mx4_gemm_dev(d.mx4_quantize_dev(P, x, stream=stream),
                               d.mx4_quantize_dev(P, w, stream=stream), stream=stream)
            got.append((y, *d.linear_xent_mean_dev(x, w, tg, stream=stream)[:3]))
        stream.synchronize()
        out[seed] = got

    alone, both = {}, {}
    for seed in (1, 5):
        work(seed, alone, torch.cuda.Stream())
    pair = [threading.Thread(target=work, args=(s, both, torch.cuda.Stream())) for s in (1, 5)]
    for th in pair:
        th.start()
    for th in pair:
        th.join()
    for seed in (1, 5):
        for got in both[seed]:
            assert all(torch.equal(a, b) for a, b in zip(got, alone[seed][0]))
