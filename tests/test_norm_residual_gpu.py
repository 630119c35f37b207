"""rms_norm_residual (csrc/irx_rmsnorm.hip) against the formula in 64 bits, within bounds counted from its roundings."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["cpp", "py"])
def backend(request, monkeypatch):
    """the C++ autograd node and the Python one"""
    from instancerefer_amd import dense, _nodes
    if request.param == "cpp":
        assert _nodes.load() is not None
    monkeypatch.setattr(dense, "NORM_BACKEND", "py" if request.param == "py" else "auto")


HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24


def inputs(rows, cols, dt, wt, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda s: (torch.randn(rows, cols, generator=g) * s).to(dt)  # noqa: E731
    x, res, dy, dh = r(1.0), r(2.0), r(1.0), r(0.5)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wt)
    return x, res if residual else None, w, dy, dh


def expected(x, res, w, dy, dh, eps):
    """{name: (value, bound)}: 32-bit arithmetic (sums of n terms: n half steps of the sum of magnitudes at most) and one rounding of a result"""
    dt, cols, rows = x.dtype, x.shape[1], x.shape[0]
    h = x if res is None else (x.float() + res.float()).to(dt)          # one rounding, the same in the operator: equal bit by bit
    H, W, G = h.double(), w.double(), dy.double()
    ms = H.square().mean(1, keepdim=True) + eps
    rs = 1 / ms.sqrt()
    e_rs = (cols + 8) * U32                                             # relative: mean square, root, quotient
    hat = H * rs
    y = hat * W
    gw = G * W
    mean = (gw * hat).mean(1, keepdim=True)
    amean = (gw * hat).abs().mean(1, keepdim=True)
    dx = rs * (gw - hat * mean) + (dh.double() if dh is not None else 0)
    big = rs * (gw.abs() + hat.abs() * amean) + (dh.double().abs() if dh is not None else 0)
    dw = (G * hat).sum(0)
    adw = (G * hat).abs().sum(0)
    low = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -133
    # without a residual h IS x: autograd adds dh to the operator's gradient itself, so that value is rounded once as the operator's result
    # (|dx - dh| half steps) and once as the sum
    twice = HALF[dt] * (dx - dh.double()).abs() + low if res is None and dh is not None else 0
    got = {"y": (y, (e_rs + 4 * U32 + HALF[dt]) * y.abs() + low), "dx": (dx, (3 * e_rs + 8 * U32) * big + HALF[dt] * (1 + HALF[dt]) * dx.abs() + twice + low),
           "dw": (dw, (e_rs + (rows + 8) * U32) * adw + HALF[w.dtype] * dw.abs() + low)}
    return h, got


def check(name, got, want):
    off = (got.double().cpu() - want[0]).abs()
    assert torch.isfinite(got).all() and (off <= want[1]).all(), "%s: %.3g of its bound" % (name, float((off / want[1].clamp(min=1e-300)).max()))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (480, 256), (5, 511), (33, 512), (9, 1024), (130, 2048), (17, 4096), (7, 8192), (3, 20000), (2500, 64), (300, 33)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward_and_gradients(kind, rows, cols, residual):
    from instancerefer_amd.dense import rms_norm_residual
    print("case", rows, cols, kind, residual, flush=True)
    for wt in {torch.float32, kind}:
        x, res, w, dy, dh = inputs(rows, cols, kind, wt, rows + cols, residual)
        h, want = expected(x, res, w, dy, dh, 1e-6)
        xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
        rd = res.to(DEV).requires_grad_(True) if residual else None
        y, s = rms_norm_residual(xd, rd, wd)
        assert torch.equal(s.detach().cpu(), h)
        check("y", y, want["y"])
        leaves = [xd, wd] + ([rd] if residual else [])
        grads = torch.autograd.grad((y, s), leaves, (dy.to(DEV), dh.to(DEV)))
        check("dx", grads[0], want["dx"])
        check("dw", grads[1], want["dw"])
        if residual:
            assert torch.equal(grads[2], grads[0])
        with torch.no_grad():
            y2, s2 = rms_norm_residual(xd, rd, wd)
        assert torch.equal(y, y2) and torch.equal(s, s2)


def test_one_output_used_alone(backend):
    from instancerefer_amd.dense import rms_norm_residual
    x, res, w, dy, dh = inputs(20, 96, torch.float32, torch.float32, 3)
    _, want = expected(x, res, w, dy, None, 1e-5)
    xd, rd, wd = (t.to(DEV).requires_grad_(True) for t in (x, res, w))
    y, h = rms_norm_residual(xd, rd, wd, eps=1e-5)
    check("dx", torch.autograd.grad(y, xd, dy.to(DEV), retain_graph=True)[0], want["dx"])
    assert torch.equal(torch.autograd.grad(h, xd, dh.to(DEV))[0].cpu(), dh)


def test_shapes_strides_and_empty(backend):
    from instancerefer_amd.dense import rms_norm_residual
    x, res, w, _, _ = inputs(12, 64, torch.bfloat16, torch.float32, 5)
    want = rms_norm_residual(x.to(DEV), res.to(DEV), w.to(DEV))
    xt = x.to(DEV).t().contiguous().t()
    odd = torch.empty(12 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(3, 4, 64)
    odd.copy_(res.to(DEV).view(3, 4, 64))
    got = rms_norm_residual(xt.view(12, 64), odd.view(12, 64), w.to(DEV))
    assert got[0].shape == (12, 64)
    # another order of addition (one element per lane): the mean square differs by at most 64 half steps, y by one rounding more
    assert float((got[0].float() - want[0].float()).abs().max()) <= 2 * 2.0 ** -8 * float(want[0].float().abs().max()) and torch.equal(got[1], want[1])
    y, h = rms_norm_residual(x.to(DEV).view(3, 4, 64), odd, w.to(DEV))
    assert y.shape == (3, 4, 64) and h.shape == (3, 4, 64)
    y, h = rms_norm_residual(x.to(DEV)[0], None, w.to(DEV))
    assert y.shape == (64,) and torch.equal(y, rms_norm_residual(x.to(DEV), None, w.to(DEV))[0][0])
    z = torch.zeros(0, 64, device=DEV, requires_grad=True)
    wd = w.to(DEV).requires_grad_(True)
    y, h = rms_norm_residual(z, z.detach(), wd)
    dz, dw = torch.autograd.grad(y, (z, wd), torch.zeros_like(y))
    assert dz.shape == (0, 64) and float(dw.abs().max()) == 0
    y, _ = rms_norm_residual(torch.zeros(2, 64, device=DEV), None, wd, eps=1e-6)
    assert float(y.abs().max()) == 0


def test_against_differences():
    from instancerefer_amd.dense import rms_norm_residual
    x, res, w, dy, dh = inputs(6, 40, torch.float32, torch.float32, 8)
    f = lambda a, b, c: sum(float((o.double() * g.to(DEV).double()).sum()) for o, g in zip(rms_norm_residual(a.to(DEV), b.to(DEV), c.to(DEV)), (dy, dh)))  # noqa: E731
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, res, w)]
    grads = torch.autograd.grad(rms_norm_residual(*leaves), leaves, (dy.to(DEV), dh.to(DEV)))
    for n in range(3):
        way = torch.randn(leaves[n].shape, generator=torch.Generator().manual_seed(n))
        up, down = [x, res, w], [x, res, w]
        up[n], down[n] = up[n] + 1e-2 * way, down[n] - 1e-2 * way
        want, have = (f(*up) - f(*down)) / 2e-2, float((grads[n].double().cpu() * way.double()).sum())
        assert abs(want - have) <= 1e-2 * max(1.0, abs(have)), (n, want, have)       # third order: 1e-4; rounding of f: 1e-5 / 2e-2


def test_captured_and_on_another_stream(backend):
    from instancerefer_amd.dense import rms_norm_residual
    x, res, w, dy, dh = (t.to(DEV) for t in inputs(700, 512, torch.bfloat16, torch.float32, 9))
    for t in (x, res, w):
        t.requires_grad_(True)

    def step():
        y, h = rms_norm_residual(x, res, w)
        return [y, h] + list(torch.autograd.grad((y, h), (x, res, w), (dy, dh)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        with torch.no_grad():
            x.mul_(1.1)


@pytest.mark.parametrize("rows,cols,kind", [(2 ** 24 + 5, 1, torch.float32), (2 ** 26 + 3, 8, torch.bfloat16)])
def test_more_rows_than_one_launch(rows, cols, kind, backend):
    from instancerefer_amd.dense import rms_norm_residual
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn((rows, cols), generator=g, device=DEV).to(kind)
    w = torch.linspace(0.5, 1.5, cols, device=DEV)
    y, h = rms_norm_residual(x, x, w)
    trained = torch.nn.Parameter(w)                                     # (a call with gradients keeps one more value per row)
    y2, _ = rms_norm_residual(x, x, trained)
    assert torch.equal(y, y2.detach())
    half = torch.finfo(kind).eps / 2
    for lo in list(range(0, rows, 1 << 22)):
        xs = x[lo:lo + (1 << 22)].double()
        assert torch.equal(h[lo:lo + (1 << 22)].double(), 2 * xs)       # doubling is exact
        want = 2 * xs / (4 * xs.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
        # sum of 8 squares, the mean, eps, the inverse root (2 half steps) and two products in 32 bits, then the type's rounding
        assert ((y[lo:lo + (1 << 22)].double() - want).abs() <= (half + 16 * 2.0 ** -24) * want.abs() + 1e-40).all()


@pytest.mark.parametrize("leaf", ["x", "x transposed", "residual"])
def test_capture_beside_a_living_eager_graph_of_other_leaves(leaf, backend):
    """a leaf that the operator views or copies first is found too"""
    from instancerefer_amd.dense import rms_norm_residual
    x, res, w, dy, dh = (t.to(DEV) for t in inputs(6, 64, torch.float32, torch.float32, 12))
    if leaf == "x transposed":
        x = x.t().contiguous().t()
    (res if leaf == "residual" else x).requires_grad_(True)
    alive = rms_norm_residual(x, res, w)
    assert rms_norm_residual(x, None, w)[1] is x
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            rms_norm_residual(x, res, w)
    torch.cuda.synchronize()
    assert alive[0].requires_grad


def test_capture_beside_a_living_eager_graph_is_refused(backend):
    from instancerefer_amd.dense import rms_norm_residual
    x, res, w, dy, dh = (t.to(DEV) for t in inputs(7, 64, torch.float32, torch.float32, 10))
    w.requires_grad_(True)
    alive = rms_norm_residual(x, res, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            rms_norm_residual(x, res, w)
    torch.cuda.synchronize()
    assert math.isfinite(float(torch.autograd.grad(alive[0], w, dy)[0].sum()))
