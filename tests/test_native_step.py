"""One training step of a small language model on the native operators together:
4-bit linear layer with its backward products, output layer's cross entropy,
AdamW; eager, captured, and with moments in 32 and in 8 bits."""
import pytest

import drift_b200 as d
from drift_b200.mlp import Net

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FWD = d.policies.by_name("mxfp4")
BATCH = 64


class Model:
    """The MLP's embedding, one hidden layer and its output layer."""

    def __init__(self, bits, seed=3, policy=FWD):
        n = Net(96, 8, 16, 256, seed)
        g = lambda a, *s: torch.from_numpy(a.reshape(*s)).float().cuda()  # noqa: E731
        self.embed, self.w1, self.b1 = g(n.embed, 96, 16), g(n.w1, 256, 128), g(n.b1, 256)
        self.w3, self.b3 = g(n.w3, 96, 256), g(n.b3, 96)
        self.low = self.w3.bfloat16()
        self.params = [self.embed, self.w1, self.b1, self.w3, self.b3]
        self.opt = d.AdamW(self.params, state_bits=bits, copies=[None, None, None, self.low, None])
        self.rng = torch.tensor([12345], dtype=torch.int64, device="cuda")
        self.p = policy

    def step(self, contexts, targets):
        p, rm = self.p, self.p.grad_cast_rounding()
        hot = torch.nn.functional.one_hot(contexts, 96).float()          # B, 8, 96
        x0 = (hot @ self.embed).view(BATCH, 128)
        x, xt = d.mx4_quantize_dev(p, x0, axis=None)
        w, wt = d.mx4_quantize_dev(p, self.w1, axis=None)
        h = torch.tanh(d.mx4_gemm_dev(x, w, bias=self.b1))
        hb = h.bfloat16()
        loss, dh, dw3, db3 = d.linear_xent_mean_dev(hb, self.low, targets, bias=self.b3)
        dz = dh.float() * (1 - h * h)
        g, gt = d.mx4_quantize_dev(p, dz, rm, axis=None, d_rng_state=self.rng)
        dx0 = d.mx4_gemm_dev(g, wt)
        dw1 = d.mx4_gemm_dev(gt, xt)
        de = hot.view(-1, 96).T @ dx0.view(-1, 16)
        grads = [de, dw1, dz.sum(0), dw3, db3]
        self.opt.step(grads)
        self.kept = dict(x0=x0, h=h, hb=hb, dz=dz, x=x, xt=xt, w=w, wt=wt, g=g, gt=gt, dh=dh)
        return loss, grads


def tokens(k):
    g = torch.Generator().manual_seed(k)
    t = torch.randint(0, 96, (BATCH,), generator=g)
    t[k % BATCH] = -100
    return torch.randint(0, 96, (BATCH, 8), generator=g).cuda(), t.cuda()


def values(q):
    return d.mx4_dequantize_dev(q)


def test_losses_and_gradients_follow_the_formulas():
    """Each stage in double from the stage before's own values. Products: fp32 sums,
    one unit an addition; the loss and d: as the operator's own tests bound them,
    here with logits below 8 over 256 elements."""
    m = Model(32)
    ctx, tg = tokens(0)
    before = [p.clone() for p in m.params]
    low = m.low.double()
    loss, (de, dw1, db1, dw3, db3) = m.step(ctx, tg)
    k = m.kept
    z = values(k["x"]) @ values(k["w"]).T + before[2].double()
    mag = values(k["x"]).abs() @ values(k["w"]).abs().T
    assert ((k["h"].double() - torch.tanh(z)).abs() <= (130 * mag + 4) * 2.0 ** -23 + 2.0 ** -21).all()
    logits = k["hb"].double() @ low.T + before[4].double()
    on = tg >= 0
    n = int(on.sum())
    lse = torch.logsumexp(logits, 1)
    want = (lse - logits.gather(1, tg.clamp(min=0)[:, None])[:, 0])[on].sum() / n
    assert abs(float(loss) - float(want)) <= 258 * 2.0 ** -23 * float(
        (k["hb"].double().abs() @ low.abs().T).max()) + 2.0 ** -17
    dl = torch.softmax(logits, 1)
    dl[on, tg[on]] -= 1
    dl = dl * on[:, None] / n
    err = 2.0 ** -8 * dl.abs() + 2.0 ** -13 * (dl.abs() + on[:, None] * 2.0 ** -13 / n)
    for got, ref, lim in ((k["dh"], dl @ low, err @ low.abs()),
                          (dw3, dl.T @ k["hb"].double(), err.T @ k["hb"].double().abs())):
        assert ((got.double() - ref).abs() <= 2 * lim + 2.0 ** -8 * ref.abs()).all()
    for got, a, b in ((dw1, k["gt"], k["xt"]),):
        ref, lim = values(a) @ values(b).T, values(a).abs() @ values(b).abs().T
        assert ((got.double() - ref).abs() <= 66 * 2.0 ** -23 * lim).all()
    # the two directions of a cast hold the same matrix, each to its own blocks
    assert (values(k["gt"]).T.sign() * values(k["g"]).sign() >= 0).all()
    for p, q in zip(m.params, before):
        assert torch.isfinite(p).all() and not torch.equal(p, q)
    assert torch.equal(m.low, m.w3.bfloat16())
    d.check_dev()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("name", ["mxfp4", "mxfp4-sr-bwd"])
def test_a_captured_step_replays_as_the_next(bits, name):
    """Three steps of a captured graph equal three eager ones bit for bit, stochastic
    gradient casts (their Rng on the device) included, while another model's eager
    step runs between."""
    p = d.policies.by_name(name)
    a, b, other = Model(bits, policy=p), Model(bits, policy=p), Model(bits, seed=9, policy=p)
    ctx, tg = (t.clone() for t in tokens(0))
    other.step(ctx, tg)  # first use of every kernel
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = a.step(ctx, tg)
    for k in range(3):
        for held, fresh in zip((ctx, tg), tokens(k)):
            held.copy_(fresh)
        graph.replay()
        other.step(*tokens(k + 7))
        want, _ = b.step(*tokens(k))
        assert torch.equal(loss, want)
        for x, y in zip(a.params, b.params):
            assert torch.equal(x, y)
        assert torch.equal(a.low, b.low) and torch.equal(a.rng, b.rng)
    d.check_dev()
