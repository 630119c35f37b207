"""A captured backward of an eager forward, beside an older eager graph of the same leaves on another stream: refused before the operator
records anything, also where the operator (or the caller) padded, copied or viewed the leaf first. Which leaves are asked is tested without
a GPU in test_capture_leaves_cpu.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["cpp", "py"])
def backend(request, monkeypatch):
    """the C++ autograd nodes and the Python ones"""
    from instancerefer_amd import _nodes, attention, dense
    assert _nodes.load() is not None
    monkeypatch.setattr(attention, "BACKEND", "py" if request.param == "py" else "auto")
    monkeypatch.setattr(dense, "NORM_BACKEND", "py" if request.param == "py" else "auto")


def refused(call, leaf, grad):
    alive = call()                                                      # keeps the leaf's accumulator on this stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph, stream=side):
            torch.autograd.grad(out, leaf, grad)
    torch.cuda.synchronize()
    # eagerly both graphs work
    want = torch.autograd.grad(alive, leaf, grad)[0]
    with torch.cuda.stream(side):
        got = torch.autograd.grad(call(), leaf, grad)[0]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and float(want.float().abs().max()) > 0


@pytest.mark.parametrize("how", ["itself", "padded", "copied", "viewed", "table"])
def test_attention(how, backend):
    from instancerefer_amd.attention import attention_packed, relative_buckets
    print("case", how, flush=True)
    dim = 40 if how == "padded" else 64
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (torch.randn(40, 2, dim, generator=g).to(DEV) for _ in range(4))
    cu, args, leaf = torch.tensor([0, 40], dtype=torch.int32, device=DEV), {}, q
    if how == "copied":                                                 # not on 16 bytes
        leaf = q = torch.empty(q.numel() + 1, device=DEV)[1:].copy_(q.reshape(-1)).view(q.shape)
    if how == "table":
        leaf = torch.randn(2, 8, generator=g).to(DEV).t()               # (8, 2), not contiguous
        args = {"bias": leaf, "buckets": relative_buckets(8, 16, device=DEV)}
    if how == "viewed":
        leaf = q.reshape(40, 2 * dim)
    leaf.requires_grad_(True)
    refused(lambda: attention_packed(leaf.view(40, 2, dim) if how == "viewed" else q, k, v, cu, **args), leaf, do)


@pytest.mark.parametrize("how", ["x", "x transposed", "residual", "weight"])
def test_norm(how, backend):
    from instancerefer_amd.dense import rms_norm_residual
    print("case", how, flush=True)
    g = torch.Generator().manual_seed(6)
    x, r, dy = (torch.randn(6, 64, generator=g).to(DEV) for _ in range(3))
    w = torch.rand(64, generator=g).to(DEV)
    if how == "x transposed":
        x = x.t().contiguous().t()
    leaf = {"residual": r, "weight": w}.get(how, x).requires_grad_(True)
    refused(lambda: rms_norm_residual(x, r, w)[0], leaf, dy)
