"""The norms around a residual branch against their formulas in 64 bits: statistics, codes, both results, and every gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
EPS, SCALE, KEY = 1e-5, 0.75, (17, 8)
NAMES = "x branch weight bias post_weight post_bias gate".split()

# A result is made of sums of products of float32.  Whatever the order, it is off by at most (roundings on the longest way) * 2^-24 of what the
# same formula gives with every term positive.  On the way are a row's sums, twice one after the other (a thread's 64 values, 5 + 5 steps
# of a warp and a block) and some 60 products and sums; down a column the rows besides.
STEPS = 256


def randn(*shape, dtype=torch.float32, seed=0, at=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) + at).to(dtype).cuda()


def formula(x, f, w, b, pw, pb, g, keep, st, layer, post, dr, dh, each, sign=-1):
    """All results in 64 bits, of given statistics; sign 1, for arguments without signs: what the terms add up to."""
    m1, p1, m2, p2 = (st[:, i:i + 1] for i in range(4))
    c = x.shape[-1]
    n1 = (f + sign * m1) * p1
    d = keep * (n1 * pw + pb) if post else keep * f
    r = SCALE * x + g * d
    n2 = (r + sign * m2) * p2

    def through(dn, n, p):
        return p * (dn + sign * (layer * dn.mean(-1, keepdim=True) + n * (dn * n).mean(-1, keepdim=True)))

    t = dr + through(dh * w, n2, p2)
    du = keep * g * t
    out = {"r": r, "h": n2 * w + b, "x": SCALE * t, "branch": through(du * pw, n1, p1) if post else du, "weight": (dh * n2).sum(0),
           "bias": dh.sum(0), "post_weight": (du * n1).sum(0), "post_bias": du.sum(0), "gate": (t * d).view(-1, each, c).sum(1)}
    return out


def near(got, want, mag, steps, what=""):
    room = steps * 2.0 ** -24 * mag
    room = room + UNIT[got.dtype] * (want.abs() + room) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126)
    value = got.double().view_as(want)
    over = (want.abs() + room >= torch.finfo(got.dtype).max) & (value == want.sign() * float("inf"))
    bad = ~(((value - want).abs() <= room) | over)
    assert not bad.any(), "%s: %d of %d, %g where %g, room %g" % (what, bad.sum(), bad.numel(), got.view_as(want)[bad][0], want[bad][0], room[bad][0])


class Case:
    """Leaves of a call, and its results in 64 bits."""

    def __init__(self, lead, c, gate, kind, post, p, dtype, params=None, gtype=None, at=0.0):
        params, gtype = params or dtype, gtype or dtype
        self.layer, self.post, self.p, self.kind, self.c = kind == "layer", post, p, kind, c
        self.rows = torch.Size(lead).numel()
        shape = tuple(lead) + (c,)
        self.x, self.branch = randn(*shape, dtype=dtype, seed=1, at=at), randn(*shape, dtype=dtype, seed=2, at=at)
        if self.rows > 4:
            self.branch.view(-1, c)[1] = 0
            self.x.view(-1, c)[2] = 0
            self.branch.view(-1, c)[2] = 0
        self.dr, self.dh = randn(*shape, dtype=dtype, seed=3), randn(*shape, dtype=dtype, seed=4)
        self.weight, self.post_weight = randn(c, dtype=params, seed=5), randn(c, dtype=params, seed=6) if post else None
        self.bias = randn(c, dtype=params, seed=7) if self.layer else None
        self.post_bias = randn(c, dtype=params, seed=8) if self.layer and post else None
        self.gate = None if gate is None else randn(*gate, c, dtype=gtype, seed=9)
        lead_of_gate = () if gate is None else (1,) * (len(lead) - len(gate)) + tuple(gate)
        self.units = 1 if gate is None else torch.Size(lead_of_gate).numel()
        self.each = max(1, self.rows // max(1, self.units))
        self.options = dict(scale=SCALE, p=p, eps=EPS, kind=kind, post=post, key=KEY)

    def leaves(self):
        return [getattr(self, n) for n in NAMES]

    def want(self, x, f, st, sign):
        from actnn_b200.cpp_extension import seeded_dropout
        a = torch.abs if sign == 1 else lambda v: v
        wide = lambda v, none: torch.tensor(none, dtype=torch.float64, device="cuda") if v is None else a(v.double())
        flat = lambda v: a(v.double().reshape(-1, self.c))
        keep = flat(seeded_dropout.apply_mask(torch.ones(self.rows, self.c, device="cuda"), self.p, KEY)) if self.p else 1.0
        g = wide(self.gate, 1.0)
        if self.gate is not None:
            g = g.reshape(self.units, 1, self.c).expand(self.units, self.each, self.c).reshape(-1, self.c)
        return formula(flat(x), flat(f), wide(self.weight, 1.0), wide(self.bias, 0.0), wide(self.post_weight, 1.0), wide(self.post_bias, 0.0), g, keep,
                       a(st.double()), self.layer, self.post, flat(self.dr), flat(self.dh), self.each, sign)

    def check_statistics(self, st):
        """Means and reciprocal deviations against exact ones; what they are off by is what their sums are, through the root."""
        x, f, e = self.x.double().view(-1, self.c), self.branch.double().view(-1, self.c), STEPS * 2.0 ** -24

        def check(v, mag, mean, rec):
            m = v.mean(-1) if self.layer else torch.zeros_like(mean).double()
            p = 1 / torch.sqrt(((v - m[:, None]) ** 2).mean(-1) + EPS)
            assert bool(((mean.double() - m).abs() <= e * mag.mean(-1)).all())
            off = e * (1 + p ** 2 * ((v - m[:, None]).abs() * (mag + mag.mean(-1, keepdim=True))).mean(-1))
            assert bool(((rec.double() / p - 1).abs() <= off * (1 + off)).all())

        if self.post:
            check(f, f.abs(), st[:, 0], st[:, 1])
        r, mag = (self.want(self.x, self.branch, st, s)["r"] for s in (-1, 1))
        check(r, mag, st[:, 2], st[:, 3])

    def decoded(self, codes, scales, x):
        """What the codes stand for; each within half a step of the value, a step being the block's largest magnitude, or 1e-30, over 127."""
        x, pad = x.double().view(-1, self.c), -self.c % 256
        step = torch.nn.functional.pad(x.abs(), (0, pad)).view(x.shape[0], -1, 256).amax(-1).clamp_min(1e-30) / 127
        assert bool(((scales.double() - step).abs() <= 3 * 2.0 ** -24 * step).all())
        wide = scales.double().repeat_interleave(256, 1)[:, :self.c]
        value = codes.double() * wide
        assert bool(((value - x).abs() <= wide * (0.5 + 127 * 2.0 ** -22)).all())
        return value

    def check_gradients(self, grads, x, f, st):
        want, mag = (self.want(x, f, st, s) for s in (-1, 1))
        for name, got in zip(NAMES, grads):
            if got is not None:
                assert got.dtype == getattr(self, name).dtype and got.shape == getattr(self, name).shape
                near(got, want[name], mag[name], STEPS + (0 if name in ("x", "branch") else self.rows), name)


CASES = [((1,), 1, None, "rms", True, 0.0), ((3,), 1, (), "layer", True, 0.1), ((1,), 32, (), "rms", True, 0.0), ((5,), 300, (), "layer", True, 0.1),
         ((10, 10), 256, (10, 1), "layer", True, 0.0), ((100,), 2048, None, "rms", False, 0.3), ((7, 11), 40, (7, 11), "layer", False, 0.2),
         ((700,), 100, None, "rms", True, 0.1), ((7, 143), 1001, (7, 1), "layer", True, 0.1), ((2, 3, 50), 768, (2, 1, 1), "layer", True, 0.1),
         ((2, 3, 50), 768, (2, 3, 1), "rms", True, 0.1), ((300, 2), 264, (300, 1), "rms", True, 0.0), ((64,), 4096, (), "rms", True, 0.1),
         ((37,), 4097, (), "rms", True, 0.1), ((8,), 8192, None, "layer", True, 0.1), ((5, 4), 9000, (5, 1), "layer", True, 0.1),
         ((30,), 16384, (), "layer", True, 0.1), ((9,), 20000, None, "rms", True, 0.0), ((2, 2), 32768, (2, 2), "layer", True, 0.1),
         ((2000,), 520, (), "layer", True, 0.1), ((4000,), 8, (), "rms", True, 0.1), ((3000,), 7, (), "layer", True, 0.1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,c,gate,kind,post,p", CASES)
def test_values_and_gradients(cuda_device, lead, c, gate, kind, post, p, dtype):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import residual_norm as rn
    case = Case(lead, c, gate, kind, post, p, dtype)
    r, h, (cx, sx, cf, sf), st = rn.run(*case.leaves(), **case.options, codes=True)
    case.check_statistics(st)
    want, mag = (case.want(case.x, case.branch, st, s) for s in (-1, 1))
    near(r, want["r"], mag["r"], STEPS, "r")
    near(h, want["h"], mag["h"], STEPS, "h")
    leaves = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
    out = ops.residual_norm.apply(*leaves, **case.options)
    assert torch.equal(out[0], r) and torch.equal(out[1], h)
    asked = [v for v in leaves if v is not None]
    grads = iter(torch.autograd.grad(out, asked, (case.dr, case.dh), retain_graph=True))
    grads = [None if v is None else next(grads) for v in leaves]
    case.check_gradients(grads, case.decoded(cx, sx, case.x), case.decoded(cf, sf, case.branch), st)
    again = iter(torch.autograd.grad(out, asked, (case.dr, case.dh), retain_graph=True))
    assert all(torch.equal(g, next(again)) for g in grads if g is not None)                     # sums in one order
    # one of the two results alone: the other's gradient is zero
    for i in (0, 1):
        both = [case.dr, case.dh]
        both[1 - i] = torch.zeros_like(both[i])
        full = torch.autograd.grad(out, asked, both, retain_graph=True)
        only = torch.autograd.grad(out[i], asked, both[i], retain_graph=True, allow_unused=True)
        assert all(torch.equal(a, b if b is not None else torch.zeros_like(a)) for a, b in zip(full, only))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,c,gate,kind,post,p", [CASES[i] for i in (3, 5, 6, 8, 12, 15)])
def test_gradients_of_inputs_kept_as_they_are(cuda_device, lead, c, gate, kind, post, p, dtype):
    """Against the formula of the inputs themselves, and against differences of the forward pass in 64 bits."""
    import actnn_b200 as actnn
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import residual_norm as rn
    actnn.set_optimization_level("L0")
    case = Case(lead, c, gate, kind, post, p, dtype)
    st = rn.run(*case.leaves(), **case.options, stats=True)[3]
    leaves = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
    asked = [v for v in leaves if v is not None]
    grads = iter(torch.autograd.grad(ops.residual_norm.apply(*leaves, **case.options), asked, (case.dr, case.dh)))
    grads = [None if v is None else next(grads) for v in leaves]
    case.check_gradients(grads, case.x, case.branch, st)

    want, mag = (case.want(case.x, case.branch, st, s) for s in (-1, 1))
    start = [None if v is None else v.detach().double() for v in leaves]

    def loss(values):
        from actnn_b200.cpp_extension import seeded_dropout
        x, f, w, b, pw, pb, g = values
        keep = seeded_dropout.apply_mask(torch.ones(case.rows, c, device="cuda"), p, KEY).double().view_as(x)

        def norm(v):
            m = v.mean(-1, keepdim=True) if case.layer else 0.0
            return (v - m) / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + EPS)
        u = f if not post else norm(f) * pw + (0.0 if pb is None else pb)
        r = SCALE * x + (1.0 if g is None else g) * (keep * u)
        h = norm(r) * w + (0.0 if b is None else b)
        return ((r * case.dr.double()).sum() + (h * case.dh.double()).sum()).item()

    for i, (name, grad) in enumerate(zip(NAMES, grads)):
        if grad is None:
            continue
        way, size = randn(*start[i].shape, seed=30 + i).double(), 1e-8
        sides = []
        for s in (-size, size):
            moved = list(start)
            moved[i] = start[i] + s * way
            sides.append(loss(moved))
        steps = STEPS + (0 if name in ("x", "branch") else case.rows)
        room = ((steps * 2.0 ** -24 + UNIT[dtype]) * 2 * mag[name].view_as(way) * way.abs()).sum().item()
        # the differences' own: the cube of the way, and what the loss is rounded to
        terms = (mag["r"] * case.dr.double().abs().view_as(mag["r"])).sum().item() + (mag["h"] * case.dh.double().abs().view_as(mag["h"])).sum().item()
        room += 2.0 ** -50 * terms / size + size * terms
        value = torch.where(grad.isfinite(), grad.double(), want[name].view_as(way))             # beyond fp16's range, as checked above
        assert abs((sides[1] - sides[0]) / (2 * size) - (value * way).sum().item()) <= room, name


@pytest.mark.parametrize("params,gtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_parameters_of_other_types(cuda_device, dtype, params, gtype):
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import residual_norm as rn
    case = Case((3, 40), 520, (3, 1), "layer", True, 0.1, dtype, params, gtype, at=20.0)              # a large mean besides
    r, h, (cx, sx, cf, sf), st = rn.run(*case.leaves(), **case.options, codes=True)
    case.check_statistics(st)
    want, mag = (case.want(case.x, case.branch, st, s) for s in (-1, 1))
    near(r, want["r"], mag["r"], STEPS, "r")
    near(h, want["h"], mag["h"], STEPS, "h")
    leaves = [v.clone().requires_grad_() for v in case.leaves()]
    grads = torch.autograd.grad(ops.residual_norm.apply(*leaves, **case.options), leaves, (case.dr, case.dh))
    case.check_gradients(grads, case.decoded(cx, sx, case.x), case.decoded(cf, sf, case.branch), st)
    case.bias = case.bias.double().to(torch.bfloat16)                # four of two types: computed in float32, gradients in their own
    leaves = [v.clone().requires_grad_() for v in case.leaves()]
    grads = torch.autograd.grad(ops.residual_norm.apply(*leaves, **case.options), leaves, (case.dr, case.dh))
    assert [g.dtype for g in grads] == [v.dtype for v in leaves]


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("level", ["L3", "L0"])
@pytest.mark.parametrize("which", [("x",), ("branch",), ("gate",), ("weight", "post_bias"), ("x", "post_weight"), ("bias", "gate")])
def test_gradients_of_some(cuda_device, monkeypatch, which, level, half):
    import actnn_b200 as actnn
    from actnn_b200 import _lib, ops
    actnn.set_optimization_level(level)
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    case = Case((4, 33), 264, (4, 1), "layer", True, 0.1, torch.bfloat16)
    every = [v.clone().requires_grad_() for v in case.leaves()]
    full = dict(zip(NAMES, torch.autograd.grad(ops.residual_norm.apply(*every, **case.options), every, (case.dr, case.dh))))
    some = [v.clone().requires_grad_(n in which) for n, v in zip(NAMES, case.leaves())]
    out = ops.residual_norm.apply(*some, **case.options)
    grads = torch.autograd.grad(out, [v for v in some if v.requires_grad], (case.dr, case.dh))
    for name, got in zip([n for n in NAMES if n in which], grads):
        if name in ("x", "branch"):
            assert torch.equal(got, full[name])
        else:                                # with another set of sums the rows may be cut in another way
            a, b = got.double(), full[name].double()
            assert bool(((a - b).abs() <= 2 * UNIT[got.dtype] * b.abs() + 1e-3).all())


def test_one_tensor_as_both_inputs(cuda_device):
    from actnn_b200 import ops
    x, dr, dh = (randn(50, 96, seed=i) for i in (1, 2, 3))
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(ops.residual_norm.apply(leaf, leaf), (leaf,), (dr, dh))
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    want = torch.autograd.grad(ops.residual_norm.apply(a, b), (a, b), (dr, dh))
    assert torch.equal(got, want[0] + want[1])


@pytest.mark.parametrize("level", ["L3", "L0"])
def test_strides_alignment_and_types_of_inputs(cuda_device, level):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    actnn.set_optimization_level(level)
    case = Case((6, 20), 64, (), "layer", True, 0.1, torch.float16)
    base = [v.clone().requires_grad_() for v in case.leaves()]
    want = ops.residual_norm.apply(*base, **case.options)
    want_g = torch.autograd.grad(want, base, (case.dr, case.dh), retain_graph=True)

    def forms(t):
        yield t.transpose(0, 1).contiguous().transpose(0, 1)
        yield torch.cat([t, t], -1)[..., t.shape[-1]:]
        yield torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    for x, f, dr, dh in zip(forms(case.x), forms(case.branch), forms(case.dr), forms(case.dh)):
        leaves = [x.detach().requires_grad_(), f.detach().requires_grad_()] + [v.clone().requires_grad_() for v in case.leaves()[2:]]
        got = ops.residual_norm.apply(*leaves, **case.options)
        got_g = torch.autograd.grad(got, leaves, (dr, dh))
        tight = dict(rtol=2.0 ** -9, atol=2.0 ** -9)                  # unaligned rows add their channels in the same order
        for a, b in zip(got + tuple(got_g), want + tuple(want_g)):
            torch.testing.assert_close(a, b, **tight)
    ones = torch.ones((), dtype=torch.float16, device="cuda").expand(6, 20, 64)
    got = torch.autograd.grad(want, base, (ones, ones), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(want, base, (ones.contiguous(), ones.contiguous()), retain_graph=True)))
    mixed = ops.residual_norm.apply(case.x.float(), case.branch, *case.leaves()[2:], **case.options)
    wide = ops.residual_norm.apply(case.x.float(), case.branch.float(), *case.leaves()[2:], **case.options)
    assert mixed[0].dtype == torch.float32 and all(torch.equal(a, b) for a, b in zip(mixed, wide))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("c", [40, 256, 1000, 4096, 9000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_row_that_is_not_finite_leaves_the_others_alone(cuda_device, kind, c, bad):
    from actnn_b200 import ops
    case = Case((40,), c, None, kind, True, 0.0, torch.bfloat16)
    clean = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
    case.x[7, c // 2] = bad
    case.branch[30, c - 1] = bad
    dirty = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
    outs = [ops.residual_norm.apply(*v, **case.options) for v in (clean, dirty)]
    grads = [torch.autograd.grad(o, v[:2], (case.dr, case.dh)) for o, v in zip(outs, (clean, dirty))]
    others = [i for i in range(40) if i not in (7, 30)]
    for a, b in zip(outs[0] + grads[0], outs[1] + grads[1]):
        assert torch.equal(a[others], b[others])
    assert outs[1][1][30].isnan().all() and not outs[1][1][7].isfinite().all()


@pytest.mark.parametrize("half", ["native", "python"])
@pytest.mark.parametrize("gate", [None, (), (0, 1)])
def test_no_rows(cuda_device, monkeypatch, gate, half):
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    case = Case((0, 5), 24, gate, "layer", True, 0.1, torch.float16)
    leaves = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
    asked = [v for v in leaves if v is not None]
    r, h = ops.residual_norm.apply(*leaves, **case.options)
    assert r.shape == h.shape == (0, 5, 24)
    for v, g in zip(asked, torch.autograd.grad((r, h), asked, (case.dr, case.dh))):
        assert g.shape == v.shape and not g.any()


@pytest.mark.parametrize("half", ["native", "python"])
def test_what_is_kept(cuda_device, monkeypatch, half):
    """Two codes a channel, their scales and four statistics a row; no mask."""
    from actnn_b200 import _lib, ops
    from test_swap_token_inputs_gpu import held
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    rows, c = 512, 2048
    case = Case((rows,), c, None, "rms", True, 0.1, torch.float16)
    leaves = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
    x, f = leaves[0] * 1, leaves[1] * 1
    before = held()
    r, h = ops.residual_norm.apply(x, f, *leaves[2:], **case.options)
    kept = held() - before - r.numel() * 4
    own = rows * (2 * c + 2 * c // 256 * 4 + 16)
    assert own <= kept <= own + 1024
    x = f = None
    assert held() - before - r.numel() * 4 <= own + 1024 - 2 * rows * c * 2
    torch.autograd.grad((r, h), [v for v in leaves if v is not None], (case.dr, case.dh))


def test_a_graph_that_is_replayed(cuda_device):
    """Two graphs with dropout: forward and backward of a replay drop the same elements, replays others; without dropout the results are those
    of a call."""
    from actnn_b200 import ops
    from test_fp8_linear_gpu import captured
    case = Case((3, 50), 264, (3, 1), "layer", True, 0.1, torch.bfloat16)

    def run(p=0.0):
        leaves = [v.detach().requires_grad_() for v in case.leaves()]
        out = ops.residual_norm.apply(*leaves, **{**case.options, "p": p, "key": None})
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, leaves, (case.dr, case.dh))

    graphs = [captured(run) for _ in range(2)]
    for seed in (21, 22):
        case.x.copy_(randn(3, 50, 264, seed=seed))
        case.dh.copy_(randn(3, 50, 264, seed=seed + 2))
        want = run()
        for graph, out in graphs:
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))

    ones = torch.ones(3, 50, 264, device="cuda")

    def dropped():
        branch = ones.detach().requires_grad_()
        r, _ = ops.residual_norm.apply(torch.zeros_like(ones), branch, post=False, p=0.5)
        return r.detach(), torch.autograd.grad(r, branch, ones)[0]

    seen = []
    graphs = [captured(dropped) for _ in range(2)]
    for graph, (r, g) in graphs + graphs:
        graph.replay()
        assert torch.equal(r, g)                          # 2 where kept, of ones and of a gradient of ones
        seen.append(r.clone())
    assert not any(torch.equal(seen[i], seen[j]) for i in range(4) for j in range(i))


def test_calls_on_two_streams_at_once(cuda_device):
    from actnn_b200 import ops
    case = Case((400,), 1024, (), "layer", True, 0.1, torch.bfloat16)
    leaves = [v.clone().requires_grad_() for v in case.leaves()]

    def run():
        out = ops.residual_norm.apply(*leaves, **case.options)
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, leaves, (case.dr, case.dh))

    want, streams, got = run(), [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in got for a, b in zip(out, want))


@pytest.mark.parametrize("level", ["L3", "L0", "L4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,c,gate,kind,post,p", [CASES[i] for i in (3, 5, 6, 10, 15)])
def test_both_halves_of_the_binding_agree(cuda_device, monkeypatch, lead, c, gate, kind, post, p, dtype, level):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    from actnn_b200.cpp_extension import residual_norm as rn
    from test_token_bindings_gpu import both_halves
    actnn.set_optimization_level(level)
    case = Case(lead, c, gate, kind, post, p, dtype)
    rest = {k: v for k, v in case.options.items() if k not in ("p", "key")}
    both_halves(monkeypatch, lambda: rn.inference(*case.leaves(), **rest))

    def drawn(key):
        torch.manual_seed(5)
        leaves = [None if v is None else v.clone().requires_grad_() for v in case.leaves()]
        out = ops.residual_norm.apply(*leaves, **{**case.options, "key": key})
        return [o.detach() for o in out] + list(torch.autograd.grad(out, [v for v in leaves if v is not None], (case.dr, case.dh)))
    both_halves(monkeypatch, lambda: drawn(KEY))
    both_halves(monkeypatch, lambda: drawn(None))


@pytest.mark.parametrize("kind,post,gate", [("rms", True, None), ("layer", True, 0.1), ("layer", False, 0.0), ("rms", False, 1.0)])
def test_layer(cuda_device, kind, post, gate):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    layer = actnn.QResidualNorm(96, kind=kind, post=post, gate=gate, scale=0.5, p=0.1).cuda()
    names = [n for n, there in (("weight", True), ("bias", kind == "layer"), ("post_weight", post), ("post_bias", post and kind == "layer"),
                                ("gate", gate is not None)) if there]
    assert sorted(n for n, _ in layer.named_parameters()) == sorted(names)
    x, f = (randn(4, 20, 96, dtype=torch.bfloat16, seed=i).requires_grad_() for i in (1, 2))
    torch.manual_seed(1)
    r, h = layer(x, f)
    torch.manual_seed(1)
    want = ops.residual_norm.apply(x, f, layer.weight, layer.bias, layer.post_weight, layer.post_bias, layer.gate, 0.5, 0.1, 1e-5, kind, post)
    assert torch.equal(r, want[0]) and torch.equal(h, want[1])
    (r.float().sum() + h.float().square().sum()).backward()
    assert all(p.grad is not None and p.grad.dtype == p.dtype for p in layer.parameters()) and x.grad is not None and f.grad is not None
    layer.eval()
    with torch.no_grad():
        a, b = layer(x, f), layer(x, f)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        given = randn(4, 1, 96, seed=5)
        if gate is None:
            want = ops.residual_norm.apply(x, f, layer.weight, layer.bias, layer.post_weight, layer.post_bias, given, 0.5, 0.0, 1e-5, kind, post)
            assert all(torch.equal(u, v) for u, v in zip(layer(x, f, given), want))
        else:
            with pytest.raises(RuntimeError, match="learned gate"):
                layer(x, f, given)


@pytest.mark.parametrize("half", ["native", "python"])
def test_refusals(cuda_device, monkeypatch, half):
    from actnn_b200 import _lib, ops
    if half == "python":
        monkeypatch.setattr(_lib, "_native", False)
    x, v = randn(2, 3, 16), randn(16)
    apply = ops.residual_norm.apply
    for call, word in ((lambda: apply(x, x[:1]), "same shape"), (lambda: apply(x, x, v[:8]), "each of the 16"), (lambda: apply(x, x, v, v), "layer"),
                       (lambda: apply(x, x, v, None, v, v), "layer"), (lambda: apply(x, x, post_weight=v, post=False), "belongs"),
                       (lambda: apply(x, x, gate=randn(3, 16)), "gate"), (lambda: apply(x, x, gate=randn(2, 1, 8)), "gate"),
                       (lambda: apply(x, x, gate=randn(1, 2, 1, 16)), "gate"), (lambda: apply(x, x, v.cpu()), "CUDA"), (lambda: apply(x, x, p=1.0), "below 1"),
                       (lambda: apply(x, x, kind="batch"), "kind"), (lambda: apply(x, x, key=3), "key"), (lambda: apply(x.double(), x.double()), "type"),
                       (lambda: apply(randn(1, 32769), randn(1, 32769)), "channels"), (lambda: apply(x[..., :0], x[..., :0]), "channels")):
        with pytest.raises(RuntimeError, match=word):
            call()
        with pytest.raises(RuntimeError, match=word), torch.no_grad():
            call()


@pytest.mark.parametrize("kind,post", [("rms", True), ("layer", True), ("layer", False)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [1, 30, 96, 257, 1024, 5000, 8192, 20000])
def test_what_is_not_given_is_ones_and_zeros(cuda_device, c, dtype, kind, post):
    from actnn_b200 import ops
    x, f, dr, dh = (randn(3, 5, c, dtype=dtype, seed=i) for i in range(4))
    ones, zeros = torch.ones(c, dtype=dtype, device="cuda"), torch.zeros(c, dtype=dtype, device="cuda")
    layer = kind == "layer"
    given = (ones, zeros if layer else None, ones if post else None, zeros if layer and post else None, ones)
    results = []
    for params in (given, (None,) * 5):
        leaves = [v.clone().requires_grad_() for v in (x, f)]
        out = ops.residual_norm.apply(*leaves, *params, scale=SCALE, p=0.2, kind=kind, post=post, key=KEY)
        results.append([o.detach() for o in out] + list(torch.autograd.grad(out, leaves, (dr, dh))))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("c", [96, 1024, 8192])
def test_parameters_that_are_not_on_16_bytes(cuda_device, c):
    from actnn_b200 import ops
    case = Case((3, 7), c, (3, 1), "layer", True, 0.1, torch.bfloat16)

    def off(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    results = []
    for leaves in (case.leaves(), case.leaves()[:2] + [off(v) for v in case.leaves()[2:]]):
        leaves = [v.detach().requires_grad_() for v in leaves]
        out = ops.residual_norm.apply(*leaves, **case.options)
        results.append([o.detach() for o in out] + list(torch.autograd.grad(out, leaves, (case.dr, case.dh))))
    for a, b in zip(*results):                           # the same sums in the same order; fused or not where the compiler chose
        near(b, a.double(), a.double().abs() + 1, STEPS)
