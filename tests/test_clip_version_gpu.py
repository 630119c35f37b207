"""clip_grads_ writes in place: autograd has to know."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_gradient_that_a_later_backward_needs():
    """clipping it in place is an error there, not a silently different result"""
    from instancerefer_amd.optim import clip_grads_
    for view in (lambda t: t, lambda t: t[:, 1:]):                      # written by the kernel, and copied back by torch
        x = torch.randn(40, 30, generator=torch.Generator().manual_seed(7)).to(DEV).requires_grad_(True)
        (g,) = torch.autograd.grad((x * x * x).sum(), x, create_graph=True)
        again, before = (g * g).sum(), g._version
        clip_grads_([view(g)], 1.0)
        assert g._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            again.backward()


def test_in_inference_mode():
    from instancerefer_amd.optim import clip_grads_
    with torch.inference_mode():
        g = torch.full((4,), 3.0, device=DEV)
        assert abs(float(clip_grads_([g], 1.0)) - 6.0) < 1e-5 and abs(float(g[0]) - 0.5) < 1e-5
