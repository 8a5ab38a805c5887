"""Measured cases of the native training-step operators.

Three operators, each with its plain form in elementary torch operations and
the framework's call:

* microscaled 4-bit floating point (e2m1 elements, one power-of-two scale per
  32 along the contraction): the cast, the product, and a linear layer's
  forward and backward products;
* a linear layer with softmax cross entropy over a vocabulary, with its
  gradients;
* AdamW over a list of tensors, with moments in 32 or in 8 bits.
"""
import math

import torch

own = False

BLOCK = 32        # elements that share one scale of a 4-bit cast
ADAM_BLOCK = 256  # elements that share one scale of an 8-bit moment
IGNORE = -100
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # The cast of one 2048 x 2048 weight matrix held in double, packed and read
        # back as effective values: what a numerics study does with it.
        dict(name="mx4_cast_weight_f64", op="mx4_cast", rows=2048, cols=2048, dtype="f64"),
        # Serving, one token through a large projection: the weights' bytes count.
        dict(name="mx4_linear_one_token", op="mx4_linear", m=1, n=8192, k=8192, dtype="bf16", bias=False),
        # The MLP's hidden layer at its batch of 64: small, launch latency counts.
        dict(name="mx4_linear_mlp_batch", op="mx4_linear", m=64, n=2048, k=2048, dtype="f32", bias=True),
        # A ragged batch through an odd-sized layer.
        dict(name="mx4_linear_odd", op="mx4_linear", m=1001, n=5000, k=4104, dtype="bf16", bias=True),
        # The block-scaled GEMM study's shape: both operands cast, then multiplied.
        dict(name="mx4_product_4096", op="mx4_product", m=4096, n=4096, k=4096, dtype="f32"),
        # Training a large linear: y, dx and dW, every operand cast along its contraction.
        dict(name="mx4_train_linear", op="mx4_train", m=8192, n=8192, k=4096, dtype="bf16"),
        # The MLP's output layer: batch 64, vocabulary 96.
        dict(name="xent_mlp", op="xent_train", t=64, d=2048, v=96, bias=True, ignored=0.0),
        # Evaluation: per-token losses of an odd batch over an odd vocabulary.
        dict(name="xent_eval_odd", op="xent_eval", t=1001, d=1024, v=50021, bias=False, ignored=0.1),
        # Training over a large vocabulary with padded positions.
        dict(name="xent_train_large", op="xent_train", t=4096, d=4096, v=131072, bias=False, ignored=0.05),
        # The MLP's seven tensors, moments in 32 bits.
        dict(name="adamw_mlp", op="adamw", shape="mlp", total=0, count=7, bits=32, p="f32", g="f32"),
        # Many small odd tensors, moments in 8 bits: launch count counts.
        dict(name="adamw_small_odd", op="adamw", shape="odd", total=300000, count=201, bits=8, p="f32", g="bf16"),
        # A large model's share of one GPU, moments in 8 bits.
        dict(name="adamw_large_8bit", op="adamw", shape="odd", total=400000000, count=60, bits=8, p="bf16", g="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["mx4_cast", "mx4_linear", "mx4_linear", "mx4_product", "mx4_train", "xent_eval", "xent_train",
                     "xent_train", "adamw", "adamw"])
    if op == "mx4_cast":
        return dict(op=op, rows=_log(rng, 1, 4096), cols=_log(rng, 1, 4096), dtype=rng.choice(["f64", "f32", "bf16"]))
    if op == "mx4_linear":
        return dict(op=op, m=_log(rng, 1, 4096), n=_log(rng, 32, 8192), k=_log(rng, 32, 8192),
                    dtype=rng.choice(["f32", "bf16"]), bias=rng.random() < 0.5)
    if op == "mx4_product":
        return dict(op=op, m=_log(rng, 16, 4096), n=_log(rng, 16, 4096), k=_log(rng, 16, 4096),
                    dtype=rng.choice(["f64", "f32", "bf16"]))
    if op == "mx4_train":
        return dict(op=op, m=_log(rng, 32, 8192), n=_log(rng, 32, 8192), k=_log(rng, 32, 4096), dtype="bf16")
    if op == "adamw":
        return dict(op=op, shape="odd", total=_log(rng, 10000, 100000000), count=_log(rng, 1, 300),
                    bits=rng.choice([32, 8]), p=rng.choice(["f32", "bf16"]), g=rng.choice(["f32", "bf16"]))
    return dict(op=op, t=_log(rng, 1, 4096), d=8 * _log(rng, 8, 512), v=_log(rng, 16, 131072), bias=rng.random() < 0.5,
                ignored=rng.choice([0.0, 0.1]))


# ------------------------------------------------------------------ inputs

def _adam_sizes(case):
    if case["shape"] == "mlp":  # embedding, then three linears with their biases
        return [96 * 64, 2048 * 2048, 2048, 2048 * 2048, 2048, 96 * 2048, 96]
    # Shares of the total that fall off as 1/(i+1), each made odd.
    n, total = case["count"], case["total"]
    h = sum(1.0 / (i + 1) for i in range(n))
    return [max(1, int(total / h / (i + 1)) | 1) for i in range(n)]


def _flat(parts):
    """One zeroed buffer that holds the parts, each from a multiple of 64 elements on, and the parts as views of it."""
    at = [0]
    for x in parts:
        at.append(at[-1] + -(-x.numel() // 64) * 64)
    buf = torch.zeros(at[-1], dtype=parts[0].dtype, device=parts[0].device)
    views = [buf[a:a + x.numel()] for a, x in zip(at, parts)]
    for to, x in zip(views, parts):
        to.copy_(x)
    return buf, views


def _cast_plain(x, headroom=0):
    """Element codes (0..15) of shape [rows, blocks, 32] and scale exponents [rows, blocks, 1], in the input's precision
    for doubles and in 32 bits otherwise. Blocks run along the last axis and are padded with zeros."""
    x = x if x.dtype == torch.float64 else x.float()
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax).exponent - 1 - 2 + headroom
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-127, 127)
    a = (x * _pow2(-e, x.dtype)).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(x.dtype)
    a = (torch.round(a / step) * step).clamp(max=6.0)
    code = (a >= 0.5).to(torch.uint8)  # magnitudes 0 .5 1 1.5 2 3 4 6 are the codes 0..7
    code = code + (a >= 1) + (a >= 1.5) + (a >= 2) + (a >= 3) + (a >= 4) + (a >= 6)
    return code | (torch.signbit(x) & (amax > 0)).to(torch.uint8) << 3, e


def _pow2(e, dtype):
    """2^e, built from its bits."""
    if dtype == torch.float64:
        return ((e.long() + 1023) << 52).view(torch.float64)
    return torch.where(e > -127, (e.int() + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _values(code, e, k, dtype=torch.float32):
    """The values that codes and exponents stand for, [rows, k]."""
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=code.device)
    return (lut[code.int()] * _pow2(e, dtype)).reshape(code.shape[0], -1)[:, :k]


def _fake(x, dtype=torch.float32):
    """The values of x's cast along its last axis."""
    return _values(*_cast_plain(x), x.shape[1], dtype)


def _unpack(parts, k, dtype=torch.float32):
    codes, scales = parts
    code = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1, BLOCK)
    return _values(code, scales.int()[..., None] - 127, k, dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def heavy(*shape, dtype=torch.float32):  # N(0,1) x lognormal(0,1), the sweeps' distribution
        return (torch.randn(*shape, device="cuda", generator=g) * torch.randn(*shape, device="cuda", generator=g).exp()).to(dtype)

    op = case["op"]
    s = {"op": op}
    if op.startswith("mx4"):
        dt = DTYPES[case["dtype"]]
        if op == "mx4_cast":
            s["x"] = heavy(case["rows"], case["cols"], dtype=dt)
        elif op == "mx4_product":
            s["a"], s["b"] = heavy(case["m"], case["k"], dtype=dt), heavy(case["n"], case["k"], dtype=dt)
        elif op == "mx4_linear":
            m, n, k = case["m"], case["n"], case["k"]
            s["x"] = normal(m, k, dtype=dt)
            # The weights as a checkpoint holds them: two codes a byte, one scale byte a block.
            code, e = _cast_plain(normal(n, k, scale=k ** -0.5))
            code = code.reshape(n, -1)
            s["w"] = (code[:, 0::2] | code[:, 1::2] << 4, (e[..., 0] + 127).to(torch.uint8))
            s["bias"] = normal(n) if case["bias"] else None
            s["k"] = k
        else:
            m, n, k = case["m"], case["n"], case["k"]
            s["x"], s["w"], s["dy"] = (normal(m, k, dtype=dt), normal(n, k, scale=k ** -0.5, dtype=dt),
                                       heavy(m, n, dtype=dt) * 1e-3)
        if own:
            import drift_b200
            s["policy"] = drift_b200.policies.by_name("mxfp4")
            if op == "mx4_linear":  # laid out once, as a server keeps them
                s["packed"] = drift_b200.Mx4.from_parts(*s["w"], cols=case["k"])
    elif op.startswith("xent"):
        t, d, v = case["t"], case["d"], case["v"]
        s["x"], s["w"] = normal(t, d, dtype=torch.bfloat16), normal(v, d, scale=2 * d ** -0.5, dtype=torch.bfloat16)
        s["bias"] = normal(v, scale=0.1) if case["bias"] else None
        tg = torch.randint(0, v, (t,), device="cuda", generator=g)
        drop = torch.rand(t, device="cuda", generator=g) < case["ignored"]
        s["targets"] = torch.where(drop, IGNORE, tg)
    else:
        sizes, pt, gt = _adam_sizes(case), DTYPES[case["p"]], DTYPES[case["g"]]
        s["bits"], s["flat"] = case["bits"], {}

        def keep(key, parts):  # one buffer for all tensors, each starting on a multiple of 64 elements
            s["flat"][key], s[key] = _flat(parts)

        keep("p", [normal(n, scale=0.02, dtype=pt) for n in sizes])
        s["g"] = [normal(n, scale=1e-3, dtype=gt) for n in sizes]
        m = [normal(n, scale=1e-3) for n in sizes]
        v = [normal(n, scale=1e-3).square() for n in sizes]
        if s["bits"] == 8:
            for key, x in (("m", m), ("r", [z.sqrt() for z in v])):
                code, scale = zip(*[_to8(z) for z in x])
                keep(key, code)
                keep(key + "s", scale)
        else:
            keep("m", m)
            keep("v", v)
        s["step"] = torch.full((1,), 10, dtype=torch.int64, device="cuda")
        if own:
            import drift_b200
            kept = ([s["m"], s["ms"], s["r"], s["rs"]] if s["bits"] == 8 else [s["m"], s["v"]])
            s["opt"] = drift_b200.AdamW(s["p"], state_bits=s["bits"], state=kept, d_step=s["step"], **HYPER)
    return s


# ------------------------------------------------------------------ plain forms

def _to8(x):
    """8-bit codes of x in blocks of 256 and one 32-bit scale a block: code = e4m3(x * (448 / amax)), scale = amax / 448."""
    n = x.numel()
    b = torch.nn.functional.pad(x, (0, -n % ADAM_BLOCK)).reshape(-1, ADAM_BLOCK)
    amax = b.abs().amax(1, keepdim=True)
    tiny = amax < 2.0 ** -100
    code = (b * torch.where(tiny, 1.0, 448.0 / amax)).clamp(-448, 448)
    code = torch.where(tiny, 0.0, code).to(torch.float8_e4m3fn)
    return code.reshape(-1)[:n].clone(), torch.where(tiny, 1.0, amax / 448.0)[:, 0].clone()


def _from8(code, scale):
    n = code.numel()
    b = torch.nn.functional.pad(code.float(), (0, -n % ADAM_BLOCK)).reshape(-1, ADAM_BLOCK)
    return (b * scale[:, None]).reshape(-1)[:n]


def _xent_plain(s, grads):
    x, w, t = s["x"].float(), s["w"].float(), s["targets"]
    logits = x @ w.T
    if s["bias"] is not None:
        logits += s["bias"]
    keep = t != IGNORE
    at = torch.where(keep, t, 0)[:, None]
    top = logits.amax(1, keepdim=True)
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    loss = torch.where(keep, (lse - logits.gather(1, at))[:, 0], 0.0)
    if not grads:
        return {"loss": loss, "lse": lse[:, 0]}
    count = keep.sum().clamp(min=1)
    dl = (logits - lse).exp_()
    dl.scatter_add_(1, at, torch.full_like(lse, -1.0))
    dl *= (keep / count)[:, None]
    out = {"loss": loss.sum() / count, "dx": (dl @ w).to(s["x"].dtype), "dw": (dl.T @ x).to(s["w"].dtype)}
    if s["bias"] is not None:
        out["db"] = dl.sum(0)
    return out


def _adam_factors(step):
    """The step's scalars, computed in 64 bits and rounded to 32."""
    t = step.double()
    c1, c2 = 1 - HYPER["betas"][0] ** t, 1 - HYPER["betas"][1] ** t
    return (HYPER["lr"] / c1).float(), (1 / c2.sqrt()).float()


def _adam_update(p, g, m, v, a1, rc2):
    (b1, b2), f = HYPER["betas"], torch.float32
    b1, b2, c1, c2, eps, wd = (torch.tensor(z, dtype=f, device=p.device) for z in (
        b1, b2, 1 - b1, 1 - b2, HYPER["eps"], 1 - HYPER["lr"] * HYPER["weight_decay"]))
    g = g.float()
    m = b1 * m + c1 * g
    v = b2 * v + (c2 * g) * g
    r = v.sqrt()
    p.copy_(wd * p.float() - (a1 * m) / (r * rc2 + eps))
    return m, v, r


def _adam_one32(p, g, m, v, a1, rc2):
    m2, v2, _ = _adam_update(p, g, m, v, a1, rc2)
    m.copy_(m2)
    v.copy_(v2)


def _adam_one8(p, g, m, ms, r, rs, a1, rc2):
    m2, _, r2 = _adam_update(p, g, _from8(m, ms), _from8(r, rs).square(), a1, rc2)
    for to, new in zip((m, ms, r, rs), (*_to8(m2), *_to8(r2))):
        to.copy_(new)


def _plain(s):
    op = s["op"]
    if op == "mx4_cast":
        x = s["x"]
        code, e = _cast_plain(x)
        return _values(code, e, x.shape[1], x.dtype if x.dtype == torch.float64 else torch.float32).to(x.dtype)
    if op == "mx4_product":
        return _fake(s["a"]) @ _fake(s["b"]).T
    if op == "mx4_linear":
        y = _fake(s["x"]) @ _unpack(s["w"], s["k"]).T
        return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)
    if op == "mx4_train":
        x, w, dy = s["x"], s["w"], s["dy"]
        y = _fake(x) @ _fake(w).T
        dx = _fake(dy) @ _fake(w.T).T
        dw = _fake(dy.T) @ _fake(x.T).T
        return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(x.dtype)}
    if op == "xent_eval":
        return _xent_plain(s, False)
    if op == "xent_train":
        return _xent_plain(s, True)
    s["step"] += 1
    a1, rc2 = _adam_factors(s["step"])
    if s["bits"] == 8:
        _ = [_adam_one8(*z, a1, rc2) for z in zip(s["p"], s["g"], s["m"], s["ms"], s["r"], s["rs"])]
    else:
        _ = [_adam_one32(*z, a1, rc2) for z in zip(s["p"], s["g"], s["m"], s["v"])]
    return s["flat"]  # parameters and moments, all updated in place


# ------------------------------------------------------------------ the framework's calls

def _own(s):
    import drift_b200 as d

    op = s["op"]
    if op == "mx4_cast":
        return d.mx4_dequantize_dev(d.mx4_quantize_dev(s["policy"], s["x"]), dtype=s["x"].dtype)
    if op == "mx4_product":
        p = s["policy"]
        return d.mx4_gemm_dev(d.mx4_quantize_dev(p, s["a"]), d.mx4_quantize_dev(p, s["b"]), dtype=torch.float32)
    if op == "mx4_linear":
        return d.mx4_gemm_dev(d.mx4_quantize_dev(s["policy"], s["x"]), s["packed"], bias=s["bias"], dtype=s["x"].dtype)
    if op == "mx4_train":
        p, dt = s["policy"], s["x"].dtype
        x, xt = d.mx4_quantize_dev(p, s["x"], axis=None)
        w, wt = d.mx4_quantize_dev(p, s["w"], axis=None)
        dy, dyt = d.mx4_quantize_dev(p, s["dy"], axis=None)
        return {"y": d.mx4_gemm_dev(x, w, dtype=dt), "dx": d.mx4_gemm_dev(dy, wt, dtype=dt),
                "dw": d.mx4_gemm_dev(dyt, xt, dtype=dt)}
    if op == "xent_eval":
        loss, lse = d.linear_xent_dev(s["x"], s["w"], s["targets"], bias=s["bias"], ignore_index=IGNORE)
        return {"loss": loss, "lse": lse}
    if op == "xent_train":
        loss, dx, dw, db = d.linear_xent_mean_dev(s["x"], s["w"], s["targets"], bias=s["bias"], ignore_index=IGNORE)
        out = {"loss": loss, "dx": dx, "dw": dw}
        if db is not None:
            out["db"] = db
        return out
    s["opt"].step(s["g"])
    return s["flat"]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    size = {"f64": 8, "f32": 4, "bf16": 2}
    packed = 17 / 32  # half a byte an element, one byte a block
    if op == "mx4_cast":
        n = case["rows"] * case["cols"]
        return {"bytes": n * 2 * size[case["dtype"]], "flops": 0}
    if op.startswith("mx4"):
        m, n, k, b = case["m"], case["n"], case["k"], size[case["dtype"]]
        if op == "mx4_product":
            return {"bytes": (m + n) * k * b + 4 * m * n, "flops": 2 * m * n * k}
        if op == "mx4_linear":
            return {"bytes": m * k * b + n * k * packed + m * n * b, "flops": 2 * m * n * k}
        return {"bytes": 2 * b * (m * k + n * k + m * n), "flops": 6 * m * n * k}
    if op.startswith("xent"):
        t, d, v = case["t"], case["d"], case["v"]
        train = op == "xent_train"
        return {"bytes": 2 * d * (t + v) * (2 if train else 1) + 8 * t, "flops": 2 * t * d * v * (3 if train else 1)}
    n = sum(_adam_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / ADAM_BLOCK
    return {"bytes": n * (2 * size[case["p"]] + size[case["g"]] + state), "flops": 16 * n}


# ------------------------------------------------------------------ the definitions in 64 bits

def _cast64(x):
    """The nearest of the fifteen values (ties to the even code), scaled by the block's power of two, by search."""
    x = x.double()
    rows, k = x.shape
    nb = -(-k // BLOCK)
    z = torch.zeros(rows, nb * BLOCK, dtype=torch.float64, device=x.device)
    z[:, :k] = x
    z = z.view(rows, nb, BLOCK)
    amax = z.abs().max(-1, keepdim=True).values
    scale = torch.exp2(torch.floor(torch.log2(amax)) - 2)  # amax is far from the borders of the exponent's range
    scale = torch.where(amax > 0, scale, 1.0)
    a = z.abs() / scale
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    up = torch.bucketize(a, mid)                # first code whose upper midpoint is not below a
    up2 = torch.bucketize(a, mid, right=True)   # differs on ties alone
    pick = torch.where(up % 2 == 0, up, up2)
    return (grid[pick] * z.sign() * scale).view(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "mx4_cast":
        return _cast64(s["x"])
    if op == "mx4_product":
        return _cast64(s["a"]) @ _cast64(s["b"]).T
    if op == "mx4_linear":
        y = _cast64(s["x"]) @ _unpack(s["w"], s["k"], torch.float64).T
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "mx4_train":
        x, w, dy = s["x"], s["w"], s["dy"]
        return {"y": _cast64(x) @ _cast64(w).T, "dx": _cast64(dy) @ _cast64(w.T.contiguous()).T,
                "dw": _cast64(dy.T.contiguous()) @ _cast64(x.T.contiguous()).T}
    if op.startswith("xent"):
        x, w, t = s["x"].double(), s["w"].double(), s["targets"]
        bias = 0.0 if s["bias"] is None else s["bias"].double()
        rows = 1024
        loss, lses, dx, n = [], [], [], int((t != IGNORE).sum())
        dw, db = torch.zeros_like(w), torch.zeros(case["v"], dtype=torch.float64, device="cuda")
        for a in range(0, case["t"], rows):
            xa, ta = x[a:a + rows], t[a:a + rows]
            logits = xa @ w.T + bias
            lse = torch.logsumexp(logits, 1)
            valid = (ta != IGNORE).nonzero()[:, 0]
            li = torch.zeros_like(lse)
            li[valid] = lse[valid] - logits[valid, ta[valid]]
            loss.append(li)
            lses.append(lse)
            if op == "xent_train":
                dl = torch.zeros_like(logits)
                dl[valid] = torch.softmax(logits[valid], 1)
                dl[valid, ta[valid]] -= 1.0
                dl /= max(1, n)
                dx.append(dl @ w)
                dw += dl.T @ xa
                db += dl.sum(0)
        loss = torch.cat(loss)
        if op == "xent_eval":
            return {"loss": loss, "lse": torch.cat(lses)}
        out = {"loss": loss.sum() / max(1, n), "dx": torch.cat(dx), "dw": dw}
        if s["bias"] is not None:
            out["db"] = db
        return out
    # AdamW: parameters and moments; an 8-bit moment is its nearest code.
    t = 11
    (b1, b2), lr, eps, wd = HYPER["betas"], HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
    got = {}

    def read(code, scale):
        return code.double() * scale.double().repeat_interleave(ADAM_BLOCK)[:code.numel()]

    for i in range(len(s["p"])):
        p, g = s["p"][i].double(), s["g"][i].double()
        if s["bits"] == 8:
            m, v = read(s["m"][i], s["ms"][i]), read(s["r"][i], s["rs"][i]) ** 2
        else:
            m, v = s["m"][i].double(), s["v"][i].double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        got.setdefault("p", []).append(p - lr * wd * p - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps))
        if s["bits"] == 8:
            for key, x in (("m", m), ("r", torch.sqrt(v))):
                n = x.numel()
                nb = -(-n // ADAM_BLOCK)
                z = torch.zeros(nb * ADAM_BLOCK, dtype=torch.float64, device=x.device)
                z[:n] = x
                top = z.view(nb, -1).abs().max(1).values
                got.setdefault(key + "s", []).append(top / 448)
                q = z.view(nb, -1) / (top / 448)[:, None]
                e = torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6)))
                u = torch.exp2(e - 3)
                got.setdefault(key, []).append((torch.round(q / u) * u).view(-1)[:n])
        else:
            got.setdefault("m", []).append(m)
            got.setdefault("v", []).append(v)
    return {key: _flat(parts)[0] for key, parts in got.items()}
