"""What the operators of a residual branch are timed on: the calls a training or serving program makes of them, over the range it
makes them.

``linear``   the product in 8-bit floating point with a power-of-two scale for each block of 128.  ``serve``: tokens through a layer
             whose weight codes are kept; ``train``: forward and backward, all three products on codes.
``norm``     the norms before and after a block with its gate and residual scale: ``train`` (forward and backward, the inputs kept
             in 8 bits) or ``serve`` (forward only).
``dropout``  dropout whose mask is drawn again in the backward pass, forward and backward.

With ``own`` false, ``run`` computes the definitions in 32 bits with elementary torch operations; with ``own`` true it makes the
calls of this framework.  ``exact`` computes them in 64 bits.

Definitions.  *Block codes*: e is the least integer, at least -126, with max|block| <= 448 * 2^e; a code is x * 2^-e rounded to e4m3
and stands for code * 2^e.  Blocks are 128 consecutive values of the reduction, of one row for tokens and gradients, of 128 rows for
weights; the products of the backward pass reduce over output channels and over tokens, and code their operands along those.
Scales are bytes e + 127, kept in the order of ``tile_order``.
*Byte codes* (what the norms keep): rint(x * (127 * (1 / a))) with a the largest magnitude, at least 1e-30, of 256 consecutive
channels of a row; they stand for code * (a * (1 / 127)).  As everywhere in this framework the codes and their scales are defined by
these steps, each one rounded float32 operation.
*Norms*: r = scale * x + gate * drop(norm(branch) * w1 + b1), h = norm(r) * w2 + b2, ``rms`` (no means, no biases) or ``layer``; the
first norm may be absent.  The backward pass uses the statistics of the forward pass and the values that the codes stand for.
*Dropout*: element i of the flattened tensor has the 16-bit field i % 8 (words and halves upwards) of the Philox4x32-10 output for key
(seed) and counter (i / 8, offset); it is kept where field + 1 > 65536 p, and divided by 1 - p.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = 128                      # values that share a scale in the product
CHANNELS = 256                   # channels that share a scale in what the norms keep
TINY = 1e-30
EPS = 1e-5
MOST_FLOPS = 2 * 16384 * 4096 * 8192
MOST_ELEMENTS = 16384 * 8192


def listed():
    return [
        # one token through a layer: the call of a serving loop, paced by latency
        dict(name="linear_token_f16", kind="linear", mode="serve", t=1, k=2048, n=4096, dtype="f16"),
        # a few tokens, odd sizes: rows that no vector load fits, blocks that end early, a head of 1000 classes
        dict(name="linear_odd_bf16", kind="linear", mode="serve", t=23, k=1001, n=1000, dtype="bf16"),
        # a batch of requests: weights are still most of what is read
        dict(name="linear_batch_bf16", kind="linear", mode="serve", t=200, k=4096, n=4096, dtype="bf16"),
        # a long prompt, the largest product
        dict(name="linear_large_bf16", kind="linear", mode="serve", t=16384, k=4096, n=8192, dtype="bf16"),
        # a training step of a layer: codes both ways, product, gradients of input, weight and bias
        dict(name="linear_train_bf16", kind="linear", mode="train", t=8192, k=2048, n=4096, dtype="bf16"),
        # one token between two blocks of a serving loop
        dict(name="norm_token_f16", kind="norm", mode="serve", norm="rms", post=True, gate="channel", p=0.0, scale=1.0,
             b=1, s=1, c=2048, dtype="f16"),
        # samples with gates of their own (conditioned blocks), odd channels, layer norm with dropout
        dict(name="norm_odd_bf16", kind="norm", mode="train", norm="layer", post=True, gate="sample", p=0.1, scale=1.0,
             b=7, s=143, c=1001, dtype="bf16"),
        # an ordinary training step with dropout and a learned gate for each channel
        dict(name="norm_train_bf16", kind="norm", mode="train", norm="rms", post=True, gate="channel", p=0.1, scale=1.0,
             b=4, s=2048, c=4096, dtype="bf16"),
        # wide rows without dropout, a scaled residual, the largest norm
        dict(name="norm_large_f16", kind="norm", mode="train", norm="rms", post=True, gate="channel", p=0.0, scale=0.75,
             b=2, s=8192, c=8192, dtype="f16"),
        # image patches in float32, layer norm before the block only
        dict(name="norm_patches_f32", kind="norm", mode="train", norm="layer", post=False, gate="none", p=0.0, scale=1.0,
             b=64, s=197, c=768, dtype="f32"),
        # a small activation without autocast, odd sizes
        dict(name="dropout_odd_f32", kind="dropout", t=77, c=1001, p=0.2, dtype="f32"),
        # the activations of a long batch, the largest elementwise case
        dict(name="dropout_large_bf16", kind="dropout", t=16384, c=8192, p=0.1, dtype="bf16"),
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm, odd as often as even."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "norm", "norm", "norm", "dropout"])
    if kind == "linear":
        mode = rng.choice(["serve", "serve", "train"])
        t, k, n = _size(rng, 1, 16384), _size(rng, 48, 8192), _size(rng, 32, 16384)
        if rng.random() < 0.6:                           # most layers' widths are whole 16-byte vectors
            k, n = (k + 15) // 16 * 16, (n + 15) // 16 * 16
        t = max(1, min(t, MOST_FLOPS // (2 * k * n * (3 if mode == "train" else 1))))
        return dict(kind=kind, mode=mode, t=t, k=k, n=n, dtype=rng.choice(["f16", "bf16", "bf16"]))
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    most = MOST_ELEMENTS * 2 // BYTES[dtype]
    if kind == "dropout":
        c, t = _size(rng, 32, 16384), _size(rng, 1, 65536)
        return dict(kind=kind, t=max(1, min(t, most // c)), c=c, p=rng.choice([0.05, 0.1, 0.3, 0.5]), dtype=dtype)
    c, b, s = _size(rng, 32, 16384), _size(rng, 1, 64), _size(rng, 1, 8192)
    if rng.random() < 0.6:
        c = (c + 15) // 16 * 16
    b = max(1, min(b, most // c))
    s = max(1, min(s, most // (b * c)))
    return dict(kind=kind, mode=rng.choice(["train", "train", "serve"]), norm=rng.choice(["rms", "rms", "layer"]),
                post=rng.random() < 0.7, gate=rng.choice(["none", "channel", "channel", "sample"]), p=rng.choice([0.0, 0.0, 0.1]),
                scale=rng.choice([1.0, 1.0, 0.5]), b=b, s=s, c=c, dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def tile_order(scales):
    """Bytes [rows, blocks] as [ceil(blocks / 4), ceil(rows / 128), 512]: of 128 rows and four blocks, the byte of row r and block j
    lies at (r % 32) * 16 + (r / 32) * 4 + j."""
    rows, blocks = scales.shape
    full = scales.new_zeros((rows + 127) // 128 * 128, (blocks + 3) // 4 * 4)
    full[:rows, :blocks] = scales
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(3, 0, 2, 1, 4).reshape(full.shape[1] // 4, -1, 512).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case=case, key=(1000003 * int(seed) + 17, 4 * (int(seed) % 1000)))
    if case["kind"] == "linear":
        t, k, n = case["t"], case["k"], case["n"]
        # tokens of different magnitude, a few channels that stand out, as hidden states have
        outlier = 1 + 7 * (torch.rand(k, generator=g, device="cuda") < 0.01)
        s["x"] = (randn(t, k).mul_(torch.exp(0.5 * randn(t, 1))).mul_(outlier)).to(dt)
        w = randn(n, k).mul_(torch.exp(0.3 * randn(n, 1))).div_(math.sqrt(k))
        s["bias"] = (0.1 * randn(n)).to(dt)
        if case["mode"] == "train":
            s["w"] = w.to(dt)
            s["dy"] = randn(t, n).mul_(torch.exp(0.5 * randn(t, 1))).to(dt)
        else:                    # the codes a serving program keeps: rows of a whole number of 16 bytes, zero behind the end
            rows, blocks = (n + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK
            full = torch.zeros(rows * BLOCK, blocks * BLOCK, device="cuda")
            full[:n, :k] = w
            e = _exponent(full.view(rows, BLOCK, blocks, BLOCK).abs().amax((1, 3)))
            codes = (full.view(rows, BLOCK, blocks, BLOCK) * _two(-e)[:, None, :, None]).view(full.shape).to(torch.float8_e4m3fn)
            s["codes"] = codes.view(torch.uint8)[:n, :(k + 15) // 16 * 16].contiguous().view(torch.float8_e4m3fn)[:, :k]
            s["scales"] = tile_order((e + 127).to(torch.uint8).repeat_interleave(BLOCK, 0)[:n])
    elif case["kind"] == "norm":
        b, rows, c = case["b"], case["s"], case["c"]
        # a residual stream with a few channels that stand out, and what a block adds to it
        outlier = 1 + 15 * (torch.rand(c, generator=g, device="cuda") < 0.01)
        s["x"] = randn(b, rows, c).mul_(outlier).to(dt)
        s["branch"] = randn(b, rows, c).mul_(torch.exp(0.5 * randn(b, rows, 1))).add_(0.2 * randn(c)).to(dt)
        s["weight"] = (1 + 0.2 * randn(c)).to(dt)
        if case["post"]:
            s["post_weight"] = (1 + 0.2 * randn(c)).to(dt)
        if case["norm"] == "layer":
            s["bias"] = (0.2 * randn(c)).to(dt)
            if case["post"]:
                s["post_bias"] = (0.2 * randn(c)).to(dt)
        if case["gate"] != "none":
            s["gate"] = (0.5 + 0.3 * randn(*((c,) if case["gate"] == "channel" else (b, 1, c)))).to(dt)
        if case["mode"] == "train":
            s["dr"], s["dh"] = randn(b, rows, c).to(dt), randn(b, rows, c).to(dt)
    else:
        s["x"], s["dy"] = randn(case["t"], case["c"]).to(dt), randn(case["t"], case["c"]).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ one pass
PARAMETERS = ("weight", "bias", "post_weight", "post_bias", "gate")


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import fp8, residual_norm
    case = s["case"]
    if case["kind"] == "linear":
        if case["mode"] == "serve":
            return fp8.linear(s["x"], s["codes"], s["scales"], s["bias"])
        x, w, bias = (v.detach().requires_grad_() for v in (s["x"], s["w"], s["bias"]))
        y = ops.fp8_linear.apply(x, w, bias)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, bias), s["dy"])
    if case["kind"] == "dropout":
        x = s["x"].detach().requires_grad_()
        y = ops.seeded_dropout.apply(x, case["p"], s["key"])
        return (y.detach(),) + torch.autograd.grad(y, (x,), s["dy"])
    if case["mode"] == "serve":
        return residual_norm.inference(s["x"], s["branch"], *(s.get(v) for v in PARAMETERS), scale=case["scale"], eps=EPS,
                                       kind=case["norm"], post=case["post"])
    leaves = {v: s[v].detach().requires_grad_() for v in ("x", "branch") + PARAMETERS if v in s}
    r, h = ops.residual_norm.apply(leaves["x"], leaves["branch"], *(leaves.get(v) for v in PARAMETERS), scale=case["scale"],
                                   p=case["p"], eps=EPS, kind=case["norm"], post=case["post"], key=s["key"])
    return (r.detach(), h.detach()) + torch.autograd.grad((r, h), tuple(leaves.values()), (s["dr"], s["dh"]))


def _exponent(a):
    """The least e of at least -126 with a <= 448 * 2^e."""
    m, e = torch.frexp(a)
    return torch.where(a > 0, (e - 9 + (m > 0.875)).clamp_min(-126), -126).int()


def _two(e):
    """2^e for e from -126 to 127, from its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _block_codes(x):
    """What the codes of rows stand for."""
    rows, k = x.shape
    full = torch.nn.functional.pad(x, (0, -k % BLOCK)).view(rows, -1, BLOCK)
    e = _exponent(full.abs().amax(-1, keepdim=True))
    return ((full * _two(-e)).to(torch.float8_e4m3fn).float() * _two(e)).view(rows, -1)[:, :k]


def _square_codes(w):
    """The same in blocks of 128 x 128."""
    n, k = w.shape
    full = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    tiles = full.view(full.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    e = _exponent(tiles.abs().amax((1, 3), keepdim=True))
    return ((tiles * _two(-e)).to(torch.float8_e4m3fn).float() * _two(e)).view(full.shape)[:n, :k]


def _decoded(codes, scales):
    n, k = codes.shape
    groups, tiles, _ = scales.shape
    e = scales.view(groups, tiles, 32, 4, 4).permute(1, 3, 2, 0, 4).reshape(tiles * 128, groups * 4)[:n].int() - 127
    return codes.float() * _two(e.clamp_min(-126)).repeat_interleave(BLOCK, 1)[:, :k]


def _kept(x):
    """What the byte codes of the last dimension stand for."""
    full = torch.nn.functional.pad(x, (0, -x.shape[-1] % CHANNELS))
    parts = full.view(x.shape[:-1] + (-1, CHANNELS))
    a = parts.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return ((parts * (a.reciprocal() * 127)).round() * (a * (1 / 127))).view(full.shape)[..., :x.shape[-1]]


def _low32(v):
    return v & 0xFFFFFFFF


def _round(c, k0, k1):
    p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
    return _low32(p1 >> 32) ^ c[1] ^ k0, _low32(p1), _low32(p0 >> 32) ^ c[3] ^ k1, _low32(p0)


def _fields(count, key, device):
    """The 16-bit fields of `count` elements."""
    calls = torch.arange((count + 7) // 8, device=device)
    seed, offset = key
    c = (_low32(calls), calls >> 32, torch.full_like(calls, offset & 0xFFFFFFFF), torch.full_like(calls, offset >> 32))
    for r in range(10):
        c = _round(c, (seed + r * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
    return torch.stack([(v >> shift) & 0xFFFF for v in c for shift in (0, 16)], -1).view(-1)[:count]


def _keep(x, p, key):
    """1 / (1 - p) where an element is kept, 0 elsewhere."""
    return ((_fields(x.numel(), key, x.device) + 1).float() > 65536 * p).float().mul_(1 / (1 - p)).view(x.shape)


def _statistics(v, layer):
    """Mean (zero without) and reciprocal deviation of the last dimension."""
    mean = v.mean(-1, keepdim=True) if layer else torch.zeros_like(v[..., :1])
    return mean, torch.rsqrt((v - mean).square().mean(-1, keepdim=True) + EPS)


def _norm_gradient(dn, n, rstd, layer):
    m = dn.mean(-1, keepdim=True) if layer else 0
    return rstd * (dn - m - n * (dn * n).mean(-1, keepdim=True))


def _run_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x = s["x"].float()
    if case["kind"] == "linear":
        bias, xq = s["bias"].float(), _block_codes(x)
        if case["mode"] == "serve":
            return (xq @ _decoded(s["codes"], s["scales"]).t() + bias).to(dt)
        w, dy = _square_codes(s["w"].float()), s["dy"].float()
        dw = _block_codes(dy.t().contiguous()) @ _block_codes(x.t().contiguous()).t()
        return (xq @ w.t() + bias).to(dt), (_block_codes(dy) @ w).to(dt), dw.to(dt), dy.sum(0).to(dt)
    if case["kind"] == "dropout":
        keep = _keep(x, case["p"], s["key"])
        return (x * keep).to(dt), (s["dy"].float() * keep).to(dt)

    layer, scale = case["norm"] == "layer", case["scale"]
    f = s["branch"].float()
    w, b, pw, pb, gate = (s[v].float() if v in s else None for v in PARAMETERS)
    gate = 1.0 if gate is None else gate
    keep = _keep(x, case["p"], s["key"]) if case["p"] and case["mode"] == "train" else 1.0
    mean1, rstd1 = _statistics(f, layer) if case["post"] else (0.0, 1.0)

    def affine(n, weight, bias):
        n = n if weight is None else n * weight
        return n if bias is None else n + bias

    d = affine((f - mean1) * rstd1, pw, pb) * keep
    r = scale * x + gate * d
    mean2, rstd2 = _statistics(r, layer)
    h = affine((r - mean2) * rstd2, w, b)
    if case["mode"] == "serve":
        return r.to(dt), h.to(dt)
    dr, dh = s["dr"].float(), s["dh"].float()
    n1 = (_kept(f) - mean1) * rstd1
    d = affine(n1, pw, pb) * keep
    n2 = (scale * _kept(x) + gate * d - mean2) * rstd2
    t = dr + _norm_gradient(dh * w, n2, rstd2, layer)
    du = t * gate * keep
    df = _norm_gradient(du * pw, n1, rstd1, layer) if case["post"] else du
    grads = {"weight": (dh * n2).sum((0, 1)), "bias": dh.sum((0, 1))}
    if case["post"]:
        grads.update(post_weight=(du * n1).sum((0, 1)), post_bias=du.sum((0, 1)))
    if case["gate"] != "none":
        grads["gate"] = (t * d).sum((0, 1) if case["gate"] == "channel" else (1,), keepdim=case["gate"] == "sample")
    return (r.to(dt), h.to(dt), (scale * t).to(dt), df.to(dt)) + tuple(grads[v].to(dt) for v in PARAMETERS if v in s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "linear":
        t, k, n = case["t"], case["k"], case["n"]
        if case["mode"] == "serve":
            return {"bytes": e * (t * k + t * n + n) + n * k + n * k // BLOCK, "flops": 2 * t * k * n}
        return {"bytes": e * (2 * t * k + 2 * t * n + 2 * n * k + 2 * n), "flops": 6 * t * k * n}
    if case["kind"] == "dropout":            # input and gradient in, output and gradient out
        return {"bytes": 4 * e * case["t"] * case["c"], "flops": 4 * case["t"] * case["c"]}
    count = case["b"] * case["s"] * case["c"]
    if case["mode"] == "serve":              # two tensors in, two out
        return {"bytes": 4 * e * count, "flops": 12 * count}
    return {"bytes": 8 * e * count + 4 * int(count * (1 + 4 / CHANNELS)), "flops": 45 * count}      # and the codes out and in


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_e4m3(v):
    """v, of magnitude 448 at most, to the nearest number of three bits behind the leading one, from 2^-6 down in steps of 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_blocks(x, high, wide):
    """x coded in blocks of high x wide."""
    out = torch.empty_like(x)
    rows, cols = x.shape
    whole = x.new_zeros((rows + high - 1) // high * high, (cols + wide - 1) // wide * wide)
    whole[:rows, :cols] = x
    tiles = whole.unfold(0, high, high).unfold(1, wide, wide)             # [.., .., high, wide]
    most = tiles.abs().amax((2, 3), keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2((most / 448).clamp(min=2.0 ** -126))))
    unit = torch.where(most <= 224 * unit, unit.clamp(min=2.0 ** -125) / 2, unit)      # where the logarithm came out a step too high
    unit = torch.where(most > 448 * unit, unit * 2, unit)                              # or too low
    out.copy_((_exact_e4m3(tiles / unit) * unit).transpose(1, 2).reshape(whole.shape)[:rows, :cols])
    return out


def _exact_bytes(x):
    """The codes by the steps that define them, what they stand for in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[-1], CHANNELS):
        part = x[..., c:c + CHANNELS].float()
        a = torch.clamp(torch.linalg.vector_norm(part, math.inf, -1, keepdim=True), min=TINY)
        factor = torch.mul(torch.div(torch.ones_like(a), a), 127.0)
        step = torch.mul(a, torch.full_like(a, 1 / 127))
        out[..., c:c + CHANNELS] = torch.round(torch.mul(part, factor)).double() * step.double()
    return out


def _exact_keep(x, p, key):
    return torch.where(_fields(x.numel(), key, x.device).view(x.shape) >= math.floor(65536 * p), 1 / (1 - p), 0.0).double()


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "dropout":
        keep = _exact_keep(x, case["p"], s["key"])
        return x * keep, s["dy"].double() * keep
    if case["kind"] == "linear":
        bias, xq = s["bias"].double(), _exact_blocks(x, 1, BLOCK)
        if case["mode"] == "serve":
            scales = torch.empty((case["n"] + 127) // 128 * 128, s["scales"].shape[0] * 4, dtype=torch.float64, device="cuda")
            for i in range(4):               # 32 rows at a time, as they lie
                scales.view(-1, 4, 32, s["scales"].shape[0], 4)[:, i] = \
                    s["scales"].view(s["scales"].shape[0], -1, 32, 4, 4)[:, :, :, i].permute(1, 2, 0, 3).double()
            wq = s["codes"].double() * torch.pow(2.0, scales[:case["n"]] - 127).repeat_interleave(BLOCK, 1)[:, :case["k"]]
            return torch.addmm(bias, xq, wq.t())
        wq, dy = _exact_blocks(s["w"].double(), BLOCK, BLOCK), s["dy"].double()
        dw = _exact_blocks(dy, BLOCK, 1).t() @ _exact_blocks(x, BLOCK, 1)
        return torch.addmm(bias, xq, wq.t()), _exact_blocks(dy, 1, BLOCK) @ wq, dw, dy.sum(0)
    c, centred = case["c"], case["norm"] == "layer"
    f = s["branch"].double()
    one, zero = torch.ones(c, dtype=torch.float64, device="cuda"), torch.zeros(c, dtype=torch.float64, device="cuda")
    w, b, pw, pb, gate = (s[v].double() if v in s else d for v, d in zip(PARAMETERS, (one, zero, one, zero, one)))
    keep = _exact_keep(x, case["p"], s["key"]) if case["mode"] == "train" and case["p"] else one

    def moments(v):
        if centred:
            var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
            return mean, torch.sqrt(var + EPS)
        return torch.zeros_like(v[..., :1]), torch.sqrt((v * v).sum(-1, keepdim=True) / c + EPS)

    mean1, dev1 = moments(f) if case["post"] else (zero[:1], one[:1])
    r = case["scale"] * x + gate * keep * (pw * ((f - mean1) / dev1) + pb)
    mean2, dev2 = moments(r)
    h = w * ((r - mean2) / dev2) + b
    if case["mode"] == "serve":
        return r, h
    dr, dh = s["dr"].double(), s["dh"].double()
    n1 = (_exact_bytes(s["branch"]) - mean1) / dev1
    d = keep * (pw * n1 + pb)
    n2 = (case["scale"] * _exact_bytes(s["x"]) + gate * d - mean2) / dev2

    def through(dn, n, dev):                 # the gradient of what was normalised: without its parts along n and along ones
        dn = dn - n * torch.einsum("bsc,bsc->bs", dn, n)[..., None] / c - (dn.sum(-1, keepdim=True) / c if centred else 0)
        return dn / dev

    t = dr + through(dh * w, n2, dev2)
    du = t * gate * keep
    df = through(du * pw, n1, dev1) if case["post"] else du
    grads = dict(weight=torch.einsum("bsc,bsc->c", dh, n2), bias=torch.einsum("bsc->c", dh),
                 post_weight=torch.einsum("bsc,bsc->c", du, n1), post_bias=torch.einsum("bsc->c", du))
    grads["gate"] = torch.einsum("bsc,bsc->c", t, d) if case["gate"] == "channel" else torch.einsum("bsc,bsc->bc", t, d)[:, None]
    return (r, h, case["scale"] * t, df) + tuple(grads[v] for v in PARAMETERS if v in s)
