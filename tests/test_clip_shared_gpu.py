"""clip_grads_ on tensors that share memory in ways that no contiguous range shows: refused before anything is written; pieces of one base that
do not meet are clipped. The decision itself is tested without a GPU in test_clip_shared_cpu.py."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def base(rows=40, cols=30):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(7)).to(DEV)


@pytest.mark.parametrize("pieces", [
    lambda b: [b[:, :5], b[:, 3:8]], lambda b: [b, b[:, 2:4]], lambda b: [b[:, 2:4], b], lambda b: [b[:, 1:5], b[:, 1:5]], lambda b: [b[::2], b[::3]],
    lambda b: [b.t()[2:9], b[7]], lambda b: [b[:, :5], b.view(-1)[33:36]]])
def test_refused(pieces):
    from instancerefer_amd.optim import clip_grads_
    b = base()
    keep = b.clone()
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grads_(pieces(b), 1.0)
    assert torch.equal(b, keep)


def test_a_tensor_over_itself_is_refused():
    from instancerefer_amd.optim import clip_grads_
    b = base()
    keep = b.clone()
    for t in (b.view(-1).unfold(0, 8, 4), b.view(-1).as_strided((5, 4), (3, 1)), b[:1].expand(4, 30)):
        with pytest.raises(ValueError, match="in place"):
            clip_grads_([t], 1.0)
    assert torch.equal(b, keep)


@pytest.mark.parametrize("pieces", [
    lambda b: [b[:, :5], b[:, 5:8], b[:, 8:]], lambda b: [b[::2], b[1::2]], lambda b: [b[:, :5], b.view(-1)[35:60]], lambda b: [b[:, ::2], b[:, 1::2]],
    lambda b: [b[:20, 3:9].t(), b[20:, 3:9]], lambda b: [b.view(-1).as_strided((3, 2), (2, 3)), b[2:, ::2]]])
def test_pieces_that_do_not_meet(pieces):
    from instancerefer_amd.optim import clip_grads_
    b = base()
    keep = b.clone()
    ps = pieces(b)
    inside = torch.zeros_like(b, dtype=torch.bool)
    for mask in pieces(inside):
        mask.fill_(True)
    norm = math.sqrt(float(keep[inside].double().square().sum()))
    assert abs(float(clip_grads_(ps, 1.0)) - norm) <= 1e-6 * norm
    want = torch.where(inside, keep.double() / (norm + 1e-6), keep.double())
    assert float((b.double() - want).abs().max()) <= 4 * 2.0 ** -24 * float(keep.abs().max())
