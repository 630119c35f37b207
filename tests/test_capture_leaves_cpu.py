"""Which leaves a node's backward will feed: what the refusal of a captured backward beside a living eager graph asks, without a GPU."""
import pytest
import torch

from instancerefer_amd import _nodes


class Probe(torch.autograd.Function):
    """an identity whose backward notes the leaves behind it"""
    seen = None

    @staticmethod
    def forward(ctx, *ts):
        return sum(t.sum() for t in ts)

    @staticmethod
    def backward(ctx, g):
        Probe.seen = _nodes.load().leaves_behind()
        return tuple(g.expand(shape) if need else None for shape, need in zip(Probe.shapes, ctx.needs_input_grad))


def behind(*ts, wrt=None):
    Probe.seen, Probe.shapes = None, [t.shape for t in ts]
    out = Probe.apply(*ts)
    if wrt is None:
        out.backward()
    else:
        torch.autograd.grad(out, wrt)
    return Probe.seen


def leaf(*shape):
    return torch.randn(*(shape or (3, 4))).requires_grad_(True)


MAKES = {"itself": lambda x: x, "padded": lambda x: torch.nn.functional.pad(x, (0, 3)), "copied": lambda x: x.clone(),
         "transposed and copied": lambda x: x.t().contiguous(), "viewed": lambda x: x.view(-1), "sliced": lambda x: x[:, 1:], "one row": lambda x: x[1],
         "cast": lambda x: x.to(torch.bfloat16), "split": lambda x: x.split((1, 3), 1)[1], "expanded": lambda x: x.expand(2, 3, 4),
         "sliced, padded, copied": lambda x: torch.nn.functional.pad(x[:, :2], (0, 1)).clone()}


@pytest.mark.parametrize("how", sorted(MAKES))
def test_a_leaf_behind_copies_and_views_is_found(how):
    x = leaf()
    seen = behind(MAKES[how](x))
    assert len(seen) == 1 and seen[0].data_ptr() == x.data_ptr()


def test_every_input_is_asked_and_results_of_other_operations_are_not_followed():
    x, y, z = leaf(), leaf(), torch.randn(3, 4)
    seen = behind(x * 2, y.t(), z, x)
    assert [t.data_ptr() for t in seen] == [y.data_ptr(), x.data_ptr()]
    assert behind(x @ y.t()) == []


def test_only_what_the_pass_feeds_is_named():
    x, y = leaf(), leaf()
    assert [t.data_ptr() for t in behind(x, y, wrt=[y])] == [y.data_ptr()]
    copied = y.clone()
    assert behind(x, copied, wrt=[copied]) == []                          # the pass ends at the copy
    assert [t.data_ptr() for t in behind(x, copied, wrt=[y, x])] == [x.data_ptr(), y.data_ptr()]


def test_outside_a_backward_there_is_nothing():
    assert _nodes.load().leaves_behind() == [] and _nodes.load().foreign_behind() == -1
