"""What rms_norm_residual keeps between its two directions: h, the weight and a value per row — not its inputs, on either backend."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["cpp", "py"])
def backend(request, monkeypatch):
    from instancerefer_amd import _nodes, dense
    assert _nodes.load() is not None
    monkeypatch.setattr(dense, "NORM_BACKEND", "py" if request.param == "py" else "auto")


def inputs(rows=33, cols=96, dt=torch.bfloat16):
    g = torch.Generator().manual_seed(rows + cols)
    x, r, dy, dh = (torch.randn(rows, cols, generator=g).to(dt).to(DEV) for _ in range(4))
    return x, r, torch.rand(cols, generator=g).to(DEV), dy, dh


def test_inputs_may_change_in_place_after_the_call(backend):
    from instancerefer_amd.dense import rms_norm_residual
    x, r, w, dy, dh = inputs()
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    want = torch.autograd.grad(rms_norm_residual(*leaves), leaves, (dy, dh))
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    a, b = leaves[0] * 1, leaves[1] * 1                                 # (results of other operations: a leaf may not change in place)
    out = rms_norm_residual(a, b, leaves[2])
    with torch.no_grad():
        a.zero_()
        b.fill_(7.0)
    got = torch.autograd.grad(out, leaves, (dy, dh))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_what_the_gradient_needs_may_not_change(backend):
    from instancerefer_amd.dense import rms_norm_residual
    x, r, w, dy, _ = inputs()
    leaf = x.clone().requires_grad_(True)
    a = leaf * 1
    y, h = rms_norm_residual(a, r, w)
    with torch.no_grad():
        h.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, dy)
    y, _ = rms_norm_residual(a, None, w)                                # h is x itself
    with torch.no_grad():
        a.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, dy)


def test_inputs_are_released(backend):
    from instancerefer_amd.dense import rms_norm_residual
    x, r, w, dy, dh = inputs(2048, 1024)
    leaf, size = x.clone().requires_grad_(True), x.numel() * x.element_size()
    a, b = leaf * 1, leaf * 2
    before = torch.cuda.memory_allocated()
    y, h = rms_norm_residual(a, b, w)
    del a, b
    # y and h come, the two inputs go, 4 bytes a row stay (blocks of 512 bytes)
    assert torch.cuda.memory_allocated() - before <= 4 * x.shape[0] + 512
    (dx,) = torch.autograd.grad((y, h), leaf, (dy, dh))
    assert dx.shape == x.shape and size == 2048 * 1024 * 2
