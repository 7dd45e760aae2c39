"""Norms around a residual branch, a row with a value that is not finite: where the formulas take it, of each kind, and no further."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, BAD, SCALE = 6, 2, 0.75


@pytest.mark.parametrize("level", ["L3", "L0"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [40, 256, 1000, 4096, 9000, 20000])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["x", "branch"])
@pytest.mark.parametrize("kind,post", [("rms", True), ("layer", True), ("rms", False), ("layer", False)])
def test_one_row(cuda_device, kind, post, where, value, c, dtype, level):
    import actnn_b200 as actnn
    from actnn_b200 import ops
    actnn.set_optimization_level(level)
    g = torch.Generator().manual_seed(c)
    x, f, dr, dh = (torch.randn(ROWS, c, generator=g).to(dtype).cuda() for _ in range(4))
    weight = torch.randn(c, generator=g).to(dtype).cuda()
    at = c // 2

    def run(x, f):
        leaves = [v.clone().requires_grad_() for v in (x, f)]
        r, h = ops.residual_norm.apply(*leaves, weight, scale=SCALE, kind=kind, post=post)
        return (r.detach(), h.detach()) + torch.autograd.grad((r, h), leaves, (dr, dh))

    want = run(x, f)
    (x if where == "x" else f)[BAD, at] = value
    got = run(x, f)
    with torch.no_grad():
        served = ops.residual_norm.apply(x, f, weight, scale=SCALE, kind=kind, post=post)
    for a, b in zip(served, got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    others, rest = [i for i in range(ROWS) if i != BAD], [i for i in range(c) if i != at]
    for a, b in zip(got, want):
        assert torch.equal(a[others], b[others])
    r, h, dx, df = (v[BAD] for v in got)
    infinite = abs(value) == float("inf")

    # the first norm, then what it adds to the stream
    if where == "branch" and post:
        if kind == "rms" and infinite:                       # 1 / inf: zero, and inf times it
            assert r[at].isnan() and torch.equal(r[rest], (SCALE * x[BAD].float()).to(dtype)[rest])
        else:
            assert r.isnan().all()
        assert h.isnan().all()
    else:
        assert torch.equal(r[rest], want[0][BAD][rest])
        if infinite:
            assert r[at] == value
        else:
            assert r[at].isnan()
        if kind == "rms" and infinite:
            assert h[at].isnan() and not h[rest].any()
        else:
            assert h.isnan().all()
    assert dx.isnan().all() and df.isnan().all()


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_a_value_that_is_dropped(cuda_device, kind):
    """A factor of zero leaves no number of what is not finite."""
    from actnn_b200 import ops
    x, f = torch.randn(3, 64, device="cuda"), torch.randn(3, 64, device="cuda")
    key = (3, 4)
    dropped = ops.residual_norm.apply(torch.zeros_like(x), torch.ones_like(f), kind=kind, post=False, p=0.5, key=key)[0] == 0
    at = int(dropped[1].nonzero()[0])
    f[1, at] = float("inf")
    r, h = ops.residual_norm.apply(x, f, kind=kind, post=False, p=0.5, key=key)
    assert r[1, at].isnan() and int(r.isnan().sum()) == 1 and h[1].isnan().all() and h[[0, 2]].isfinite().all()
