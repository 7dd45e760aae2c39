"""What the token operators are timed on: the calls a training or serving program makes of them, over the range it makes them.

``linear``  the product of 8-bit integers with a scale for each token and each output channel.  ``serve``: tokens through a
            layer whose weight codes are kept; ``train``: forward and backward with the weight quantised in the step.
``act``     an activation function whose backward pass reads an 8-bit copy of its input, forward and backward;
``glu``     the gated form, ``f(gate) * up`` of the two halves of the last dimension;
``norm``    group norm with an activation on channels-last tensors: ``train`` (forward and backward, the input kept in 8 bits)
            or ``serve`` (forward only).

With ``own`` false, ``run`` computes the definitions in 32 bits with elementary torch operations; with ``own`` true it makes the
calls of this framework.  ``exact`` computes them in 64 bits.

Definitions.  A code is ``rint(x * (127 / a))`` with ``a`` the largest magnitude of its row (linear) or of its 256 consecutive
elements (act, glu), at least 1e-30, and stands for ``code * (a / 127)``.  Group norm centres its codes on the middle of the range
of each (sample, group).  Products and derivatives that the backward pass takes of a saved input use the values the codes stand for.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = 256                      # consecutive elements that share a scale in the checkpoint of an activation
TINY = 1e-30                     # the smallest magnitude a scale is made of
EPS = 1e-5
MOST_FLOPS = 2 * 16384 * 4096 * 8192
MOST_ELEMENTS = 16384 * 8192


def listed():
    return [
        # one token through a layer: the call of a serving loop, paced by latency
        dict(name="linear_token_f16", kind="linear", mode="serve", t=1, k=2048, n=4096, dtype="f16"),
        # a few tokens, odd sizes: rows that no vector load fits, a head of 1000 classes
        dict(name="linear_odd_bf16", kind="linear", mode="serve", t=23, k=1001, n=1000, dtype="bf16"),
        # a batch of requests: weights are still most of what is read
        dict(name="linear_batch_bf16", kind="linear", mode="serve", t=200, k=4096, n=4096, dtype="bf16"),
        # a long prompt or a training batch, the largest product
        dict(name="linear_large_bf16", kind="linear", mode="serve", t=16384, k=4096, n=8192, dtype="bf16"),
        # a training step of a layer: product, gradients of input, weight and bias
        dict(name="linear_train_bf16", kind="linear", mode="train", t=8192, k=2048, n=4096, dtype="bf16"),
        # a small activation without autocast, odd sizes
        dict(name="act_gelu_odd_f32", kind="act", f="gelu", t=77, c=1001, dtype="f32"),
        # an ordinary one under autocast
        dict(name="act_gelu_tanh_f16", kind="act", f="gelu_tanh", t=8192, c=4096, dtype="f16"),
        # the gated activation of a feed-forward block, the largest elementwise case
        dict(name="glu_silu_bf16", kind="glu", f="silu", t=16384, c=4096, dtype="bf16"),
        # one small image at inference, paced by latency
        dict(name="norm_silu_small_f16", kind="norm", mode="serve", f="silu", b=1, c=64, h=14, w=14, groups=8, dtype="f16"),
        # odd maps and six channels a group
        dict(name="norm_silu_odd_bf16", kind="norm", mode="train", f="silu", b=100, c=192, h=35, w=35, groups=32, dtype="bf16"),
        # the activation of the benchmark, the largest norm
        dict(name="norm_silu_large_f16", kind="norm", mode="train", f="silu", b=512, c=256, h=28, w=28, groups=32, dtype="f16"),
        # float32 training without an activation behind the norm
        dict(name="norm_none_f32", kind="norm", mode="train", f="none", b=64, c=64, h=56, w=56, groups=8, dtype="f32"),
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm, odd as often as even."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "act", "glu", "norm", "norm"])
    if kind == "linear":
        mode = rng.choice(["serve", "serve", "train"])
        t, k, n = _size(rng, 1, 16384), _size(rng, 48, 8192), _size(rng, 32, 16384)
        if rng.random() < 0.6:                           # most layers' widths are whole 16-byte vectors
            k, n = (k + 15) // 16 * 16, (n + 15) // 16 * 16
        t = max(1, min(t, MOST_FLOPS // (2 * k * n * (3 if mode == "train" else 1))))
        return dict(kind=kind, mode=mode, t=t, k=k, n=n,
                    dtype=rng.choice(["f16", "bf16"] if mode == "train" else ["f16", "bf16", "bf16", "f32"]))
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    most = MOST_ELEMENTS * 2 // BYTES[dtype]
    if kind in ("act", "glu"):
        c, t = _size(rng, 32, 16384), _size(rng, 1, 65536)
        if rng.random() < 0.6:
            c = (c + 15) // 16 * 16
        t = max(1, min(t, most // (c * (2 if kind == "glu" else 1))))
        return dict(kind=kind, f=rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), t=t, c=c, dtype=dtype)
    groups = rng.choice([1, 4, 8, 16, 32, 32])
    c, h = groups * _size(rng, 1, 2048 // groups), _size(rng, 4, 96)
    w = max(1, h - rng.choice([0, 0, 1, 3]))
    b = max(1, min(_size(rng, 1, 512), most // (c * h * w)))
    return dict(kind=kind, mode=rng.choice(["train", "train", "serve"]), f=rng.choice(["silu", "silu", "gelu", "relu", "none"]),
                b=b, c=c, h=h, w=w, groups=groups, dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case=case)
    if case["kind"] == "linear":
        t, k, n = case["t"], case["k"], case["n"]
        # tokens of different magnitude, a few channels that stand out, as hidden states have
        outlier = 1 + 7 * (torch.rand(k, generator=g, device="cuda") < 0.01)
        s["x"] = (randn(t, k).mul_(torch.exp(0.5 * randn(t, 1))).mul_(outlier)).to(dt)
        w = randn(n, k).mul_(torch.exp(0.3 * randn(n, 1))).div_(math.sqrt(k))
        s["bias"] = (0.1 * randn(n)).to(dt)
        if case["mode"] == "train":
            s["w"] = w.to(dt)
            s["dy"] = randn(t, n).to(dt)
        else:                    # the codes a serving program keeps: rows of a whole number of 16 bytes, zero behind the end
            a = w.abs().amax(1).clamp_min_(TINY)
            codes = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
            codes[:, :k] = (w * (127 / a)[:, None]).round_().to(torch.int8)
            s["codes"], s["scale"] = codes[:, :k], a / 127
    elif case["kind"] in ("act", "glu"):
        t, c = case["t"], case["c"]
        s["x"] = randn(t, c * (2 if case["kind"] == "glu" else 1)).mul_(1.5).to(dt)
        s["dy"] = randn(t, c).to(dt)
    else:
        b, c, h, w = case["b"], case["c"], case["h"], case["w"]
        # channels with means of their own, in channels-last memory
        x = randn(b, h, w, c).mul_(torch.exp(0.3 * randn(c))).add_(0.5 * randn(c)).to(dt)
        s["x"] = x.permute(0, 3, 1, 2)
        s["gamma"], s["beta"] = 1 + 0.2 * randn(c), 0.2 * randn(c)
        if case["mode"] == "train":
            s["dy"] = randn(b, h, w, c).to(dt).permute(0, 3, 1, 2)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import group_norm, int8
    case = s["case"]
    if case["kind"] == "linear":
        if case["mode"] == "serve":
            return int8.linear(s["x"], s["codes"], s["scale"], s["bias"])
        x, w, bias = (v.detach().requires_grad_() for v in (s["x"], s["w"], s["bias"]))
        y = ops.int8_linear.apply(x, w, bias)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, bias), s["dy"])
    if case["kind"] in ("act", "glu"):
        x = s["x"].detach().requires_grad_()
        y = (ops.glu if case["kind"] == "glu" else ops.activation).apply(x, case["f"])
        return (y.detach(),) + torch.autograd.grad(y, (x,), s["dy"])
    if case["mode"] == "serve":
        return group_norm.inference(s["x"], case["groups"], s["gamma"], s["beta"], EPS, case["f"])
    x, gamma, beta = (v.detach().requires_grad_() for v in (s["x"], s["gamma"], s["beta"]))
    y = ops.group_norm.apply(x, case["groups"], gamma, beta, EPS, case["f"])
    return (y.detach(),) + torch.autograd.grad(y, (x, gamma, beta), s["dy"])


def _f(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return torch.where(z > 0, z, torch.zeros_like(z)) if name == "relu" else z


def _df(name, z):
    if name == "silu":
        sig = torch.sigmoid(z)
        return sig * (1 + z * (1 - sig))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if name == "gelu_tanh":
        th = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return (z > 0).to(z.dtype) if name == "relu" else torch.ones_like(z)


def _row_codes(x):
    a = x.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return (x * (127 / a)).round(), a / 127


def _saved(x):
    """What the codes of blocks of 256 consecutive elements stand for."""
    flat = x.reshape(-1)
    pad = -flat.numel() % BLOCK
    codes, scale = _row_codes(torch.cat([flat, flat.new_zeros(pad)]).view(-1, BLOCK))
    return (codes * scale).view(-1)[:flat.numel()].view(x.shape)


def _run_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x = s["x"].float()
    if case["kind"] == "linear":
        cx, sx = _row_codes(x)
        bias = s["bias"].float()
        if case["mode"] == "serve":
            return ((cx @ s["codes"].float().t()) * sx * s["scale"] + bias).to(dt)
        cw, sw = _row_codes(s["w"].float())
        y, dy = (cx @ cw.t()) * sx * sw.t() + bias, s["dy"].float()
        return y.to(dt), (dy @ (cw * sw)).to(dt), (dy.t() @ (cx * sx)).to(dt), dy.sum(0).to(dt)
    if case["kind"] == "act":
        return _f(case["f"], x).to(dt), (s["dy"].float() * _df(case["f"], _saved(x))).to(dt)
    if case["kind"] == "glu":
        gate, up = x.chunk(2, -1)
        y, dy = _f(case["f"], gate) * up, s["dy"].float()
        gate, up = _saved(gate), _saved(up)
        return y.to(dt), torch.cat([dy * up * _df(case["f"], gate), dy * _f(case["f"], gate)], -1).to(dt)
    b, c, h, w = x.shape
    groups = case["groups"]

    def split(v):                # [b, h, w, c] values as [b, pixels, groups, channels of a group]
        return v.permute(0, 2, 3, 1).reshape(b, h * w, groups, c // groups)

    def back(v):
        return v.reshape(b, h, w, c).permute(0, 3, 1, 2)

    x, gamma, beta = split(x), s["gamma"].view(groups, -1), s["beta"].view(groups, -1)
    mean = x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + EPS)
    y = back(_f(case["f"], (x - mean) * rstd * gamma + beta).to(dt))
    if case["mode"] == "serve":
        return y
    hi, lo = x.amax((1, 3), keepdim=True), x.amin((1, 3), keepdim=True)
    mid, half = 0.5 * hi + 0.5 * lo, (0.5 * hi - 0.5 * lo).clamp_min(TINY)
    xhat = (mid + ((x - mid) * (127 / half)).round() * (half / 127) - mean) * rstd
    dz = split(s["dy"].float()) * _df(case["f"], xhat * gamma + beta)
    dgamma, dbeta, dn = (dz * xhat).sum((0, 1)).view(-1), dz.sum((0, 1)).view(-1), dz * gamma
    dx = rstd * (dn - dn.mean((1, 3), keepdim=True) - xhat * (dn * xhat).mean((1, 3), keepdim=True))
    return y, back(dx.to(dt)), dgamma, dbeta


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "linear":
        t, k, n = case["t"], case["k"], case["n"]
        if case["mode"] == "serve":
            return {"bytes": e * (t * k + t * n + n) + n * k + 4 * n, "flops": 2 * t * k * n}
        return {"bytes": e * (2 * t * k + 2 * t * n + 2 * n * k + 2 * n), "flops": 6 * t * k * n}
    if case["kind"] in ("act", "glu"):       # input and gradient in, output and gradient out, the codes out and in
        ins = case["t"] * case["c"] * (2 if case["kind"] == "glu" else 1)
        outs = case["t"] * case["c"]
        return {"bytes": 2 * e * ins + 2 * e * outs + 2 * ins * (1 + 4 / BLOCK), "flops": 20 * outs}
    count, params = case["b"] * case["c"] * case["h"] * case["w"], 4 * case["c"]
    if case["mode"] == "serve":
        return {"bytes": 2 * e * count + 2 * params, "flops": 10 * count}
    return {"bytes": 4 * e * count + 2 * count + 5 * params, "flops": 40 * count}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_f(name, z):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.clamp(z, min=0), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return z * e, e + z * e * (1 - e)
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    u = math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)          # (1 + tanh(u / 2)) / 2 is the logistic function of u
    e = 1 / (1 + torch.exp(-u))
    return z * e, e + z * e * (1 - e) * math.sqrt(8 / math.pi) * (1 + 0.134145 * z * z)


def _exact_decoded(x, dims):
    """x rounded to 127 steps each way of its largest magnitude along dims."""
    step = x.abs().amax(dims, keepdim=True).clamp(min=TINY) / 127
    return torch.round(x / step) * step


def _exact_blocks(x):
    n = x.numel()
    out = x.new_zeros((n + BLOCK - 1) // BLOCK * BLOCK)
    out[:n] = x.reshape(-1)
    return _exact_decoded(out.view(-1, BLOCK), (1,)).reshape(-1)[:n].reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "linear":
        bias, xq = s["bias"].double(), _exact_decoded(x, (1,))
        if case["mode"] == "serve":
            return torch.addmm(bias, xq, (s["codes"].double() * s["scale"].double()[:, None]).t())
        wq, dy = _exact_decoded(s["w"].double(), (1,)), s["dy"].double()
        return torch.addmm(bias, xq, wq.t()), dy @ wq, dy.t() @ xq, dy.sum(0)
    if case["kind"] == "act":
        return _exact_f(case["f"], x)[0], s["dy"].double() * _exact_f(case["f"], _exact_blocks(x))[1]
    if case["kind"] == "glu":
        c, dy = case["c"], s["dy"].double()
        y = _exact_f(case["f"], x[:, :c])[0] * x[:, c:]
        f, df = _exact_f(case["f"], _exact_blocks(x[:, :c].contiguous()))
        return y, torch.cat([dy * df * _exact_blocks(x[:, c:].contiguous()), dy * f], 1)
    b, c, h, w = x.shape
    groups = case["groups"]
    rows = x.reshape(b, groups, -1)                                # a row for each sample and group
    gamma, beta = (s[v].double().view(1, c, 1, 1) for v in ("gamma", "beta"))
    var, mean = torch.var_mean(rows, 2, correction=0, keepdim=True)
    std = torch.sqrt(var + EPS)
    y = _exact_f(case["f"], ((rows - mean) / std).view(x.shape) * gamma + beta)[0]
    if case["mode"] == "serve":
        return y
    mid = (rows.amax(2, keepdim=True) + rows.amin(2, keepdim=True)) / 2
    norm = (mid + _exact_decoded(rows - mid, (2,)) - mean) / std
    norm4 = norm.view(x.shape)
    dz = s["dy"].double() * _exact_f(case["f"], norm4 * gamma + beta)[1]
    dn = (dz * gamma).reshape(rows.shape)
    dx = (dn - dn.mean(2, keepdim=True) - norm * (dn * norm).mean(2, keepdim=True)) / std
    return y, dx.view(x.shape), (dz * norm4).sum((0, 2, 3)), dz.sum((0, 2, 3))
