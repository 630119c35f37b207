"""clip_grads_ and FlatAdam's clipping (csrc/irx_optim.hip) against the formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
KINDS = [torch.float32, torch.bfloat16, torch.float16]


def make(sizes, seed=0, scale=1.0, kinds=KINDS):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


def compare(grads, max_norm, norm_type=2.0):
    from instancerefer_amd.optim import clip_grads_
    if norm_type == 2.0:
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    else:
        norm = max([float(g.double().abs().max()) for g in grads if g.numel()] + [0.0])
    factor = min(1.0, max_norm / (norm + 1e-6))
    dev = [g.to(DEV) for g in grads]
    got = clip_grads_(dev, max_norm, norm_type)
    assert abs(float(got) - norm) <= 2 * 2.0 ** -24 * norm + 1e-45
    for g, d in zip(grads, dev):
        want = g.double() * factor
        if factor == 1.0:
            assert torch.equal(d.cpu(), g)
        low = 2.0 ** -25 if g.dtype == torch.float16 else 2.0 ** -133
        # the factor's and the product's roundings in 32 bits, the value's own
        assert ((d.double().cpu() - want).abs() <= (2 * 2.0 ** -24 + HALF[g.dtype]) * want.abs() + low).all()


@pytest.mark.parametrize("sizes", [[1], [3, 1, 17], [4096, 4097, 8191, 5], [100000, 1, 333, 70001], [0, 5, 0], [2500000, 12, 1300001]])
def test_list_of_mixed_types(sizes):
    for max_norm in (0.5, 1e9, 0.0):
        compare(make(sizes, len(sizes)), max_norm)
    compare(make(sizes, 7), 0.25, math.inf)


def test_more_tensors_than_one_table_and_more_sums_than_one_fold():
    compare(make([37 + i % 11 for i in range(161)], 1), 1.0)
    compare(make([1 + i % 5 for i in range(2400)], 2), 1.0)
    compare(make([1 + i % 5 for i in range(2400)], 2), 0.1, math.inf)


def test_no_overflow_and_tiny_values():
    compare(make([1000, 50], 3, 1e25, [torch.float32]), 1.0)
    compare(make([1000, 50], 3, 1e-25, [torch.float32]), 1e-26)


def test_values_that_are_not_numbers():
    from instancerefer_amd.optim import clip_grads_
    for nt in (2.0, math.inf):
        g = [t.to(DEV) for t in make([100, 5000], 4)]
        g[0][7] = math.nan
        assert math.isnan(float(clip_grads_(g, 1.0, nt))) and all(torch.isnan(t).all() for t in g)
        g = [t.to(DEV) for t in make([100, 5000], 4)]
        g[0][7] = -math.inf
        assert float(clip_grads_(g, 1.0, nt)) == math.inf
        assert math.isnan(float(g[0][7])) and float(g[1].float().abs().max()) == 0.0


def test_views_orders_none_and_empty():
    from instancerefer_amd.optim import clip_grads_
    base = torch.randn(40, 30, generator=torch.Generator().manual_seed(5)).to(DEV)
    parts = [base.t()[:, :20], base[20:, 1:9]]                                  # a dense transpose, a strided piece
    flat = torch.randn(101, generator=torch.Generator().manual_seed(6)).to(DEV)
    parts += [flat[1:], None]                                                   # not on 16 bytes
    keep = [p.clone() for p in parts if p is not None]
    norm = math.sqrt(sum(float(k.double().square().sum()) for k in keep))
    first, untouched = float(flat[0]), base[20:, 9:].clone()
    got = clip_grads_(parts, 1.0)
    assert abs(float(got) - norm) <= 1e-6 * norm
    for p, k in zip(parts, keep):
        assert float((p.double() - k.double() / (norm + 1e-6)).abs().max()) <= 4 * 2.0 ** -24 * float(k.abs().max())
    assert float(flat[0]) == first and torch.equal(base[20:, 9:], untouched)
    assert float(clip_grads_([], 1.0)) == 0.0 and float(clip_grads_([None], 1.0)) == 0.0
    assert float(clip_grads_([torch.zeros(0, device=DEV)], 1.0)) == 0.0 and float(clip_grads_(torch.zeros(4, device=DEV), 1.0)) == 0.0


def test_refuses_shared_memory():
    from instancerefer_amd.optim import clip_grads_
    t = torch.ones(100, device=DEV)
    for pair in ([t, t], [t, t[50:]], [t[:60], t[59:]]):
        with pytest.raises(RuntimeError, match="share memory"):
            clip_grads_(pair, 1.0)
    assert float(t.min()) == 1.0
    assert abs(float(clip_grads_([t[:50], t[50:]], 1.0)) - 10.0) <= 1e-5


def test_captured_and_replayed():
    from instancerefer_amd.optim import clip_grads_
    fresh = [t.to(DEV) for t in make([70000, 33, 5000], 8)]
    work = [torch.empty_like(t) for t in fresh]

    def step():
        for w, f in zip(work, fresh):
            w.copy_(f)
        return clip_grads_(work, 2.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(3):
        want = float(step())
        expect = [w.clone() for w in work]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert float(held) == want and all(torch.equal(a, b) for a, b in zip(work, expect))
        for f in fresh:
            f.mul_(0.5)


def params_of(shapes, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(DEV)) for s in shapes]


SHAPES = [(300, 256), (256,), (1,), (7, 9), (1000, 33)]


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_optimizer_step_with_clipping(norm_type):
    """three steps against Adam in 64 bits on gradients clipped in 64 bits"""
    from instancerefer_amd.optim import FlatAdam
    ps = params_of(SHAPES, 1)
    ref = [p.detach().double().clone() for p in ps]
    m, v = [torch.zeros_like(r) for r in ref], [torch.zeros_like(r) for r in ref]
    b1, b2, lr, eps, wd = 0.875, 1 - 2.0 ** -10, 1e-2, 1e-8, 1e-2      # 1 - b is exact in 32 bits
    opt = FlatAdam(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
    for step in range(1, 4):
        g = torch.Generator().manual_seed(step)
        grads = [torch.randn(p.shape, generator=g).to(DEV) for p in ps]
        opt.zero_grad()
        for p, x in zip(ps, grads):
            p.grad = x
        got = opt.backward_step(max_norm=0.5, norm_type=norm_type)
        all_g = torch.cat([x.double().reshape(-1) for x in grads])
        norm = float(all_g.norm()) if norm_type == 2.0 else float(all_g.abs().max())
        assert abs(float(got) - norm) <= 2 * 2.0 ** -24 * norm
        f = min(1.0, 0.5 / (norm + 1e-6))
        for i, x in enumerate(grads):
            gr = x.double() * f + wd * ref[i]
            m[i] = b1 * m[i] + (1 - b1) * gr
            v[i] = b2 * v[i] + (1 - b2) * gr * gr
            ref[i] -= lr / (1 - b1 ** step) * m[i] / (v[i].sqrt() / math.sqrt(1 - b2 ** step) + eps)
            # lr * m / sqrt(v) is at most lr in size per step; its relative error is a few half steps plus the state's
            assert float((ps[i].double() - ref[i]).abs().max()) <= step * (lr * 64 * 2.0 ** -24 + float(ref[i].abs().max()) * 2.0 ** -23) + 1e-6
        assert torch.equal(opt._slots[0], grads[0])                     # the gradients stay as they are


def test_a_large_limit_is_the_unclipped_step():
    from instancerefer_amd.optim import FlatAdam
    one, two = params_of(SHAPES, 2), params_of(SHAPES, 2)
    a, b = FlatAdam(one, lr=1e-3, weight_decay=1e-5), FlatAdam(two, lr=1e-3, weight_decay=1e-5)
    for step in range(3):
        g = torch.Generator().manual_seed(step)
        for p, q in zip(one, two):
            p.grad = torch.randn(p.shape, generator=g).to(DEV)
            q.grad = p.grad.clone()
        assert a.backward_step() is None
        assert float(b.backward_step(max_norm=1e9)) > 0
    assert torch.equal(a.flat_p, b.flat_p) and torch.equal(a.exp_avg_sq, b.exp_avg_sq)


def test_parameters_without_gradients_and_none_at_all():
    from instancerefer_amd.optim import FlatAdam
    ps = params_of(SHAPES, 3)
    opt = FlatAdam(ps, lr=1e-2)
    ps[1].grad, ps[4].grad = torch.full((256,), 2.0, device=DEV), torch.full((1000, 33), 1.0, device=DEV)
    before = [p.detach().clone() for p in ps]
    norm = opt.backward_step(max_norm=1.0)
    assert abs(float(norm) - math.sqrt(256 * 4 + 33000)) <= 1e-4
    assert torch.equal(ps[0], before[0]) and torch.equal(ps[3], before[3]) and not torch.equal(ps[4], before[4])
    opt.zero_grad()
    before = [p.detach().clone() for p in ps]
    assert float(opt.backward_step(max_norm=1.0)) == 0.0
    assert all(torch.equal(p, b) for p, b in zip(ps, before))


def test_gather_of_gradients_of_every_layout_and_of_many_tensors():
    """transposed, expanded, off 16 bytes, more tensors than one table and more sums than one fold: as if gathered first"""
    from instancerefer_amd.optim import FlatAdam
    for shapes in ([(40, 30), (7, 9), (50,), (3, 5)], [(1 + i % 7,) for i in range(2300)]):
        one, two = params_of(shapes, 5), params_of(shapes, 5)
        a, b = FlatAdam(one, lr=1e-2), FlatAdam(two, lr=1e-2)
        g = torch.Generator().manual_seed(6)
        for i, (p, q) in enumerate(zip(one, two)):
            x = torch.randn(p.shape, generator=g).to(DEV)
            if i == 0 and p.dim() == 2:
                x = x.t().contiguous().t()
            elif i == 1 and p.dim() == 2:
                x = x[:1].expand(p.shape)
            elif i == 2:
                buf = torch.empty(x.numel() + 1, device=DEV)[1:]
                buf.copy_(x)
                x = buf.view(x.shape)
            p.grad, q.grad = x, x.clone()
        a.gather_grads()
        want = a.step(max_norm=0.3)                                     # gathered, then summed over the flat buffer
        got = b.backward_step(max_norm=0.3)                             # summed on the way
        assert torch.equal(a.flat_g, b.flat_g)
        assert abs(float(got) - float(want)) <= 4 * 2.0 ** -24 * float(want)
        assert float((a.flat_p - b.flat_p).abs().max()) <= 1e-2 * 64 * 2.0 ** -24 + 2.0 ** -23 * float(a.flat_p.abs().max())


def test_addresses_read_at_once_or_one_by_one(monkeypatch):
    """the same bits either way; a slot that a producer has filled, and one that has a gradient besides, count once"""
    from instancerefer_amd.optim import FlatAdam
    pair = [params_of(SHAPES, 8), params_of(SHAPES, 8)]
    a, b = (FlatAdam(ps, lr=1e-2) for ps in pair)
    monkeypatch.setattr(b, "_gather_plain", lambda todo, inf_norm: None)
    for step, (filled, besides) in enumerate([((), ()), ((1,), ()), ((1, 3), (3,)), ((), ())]):
        g = torch.Generator().manual_seed(step)
        grads = [torch.randn(p.shape, generator=g).to(DEV) for p in pair[0]]
        for opt, ps in ((a, pair[0]), (b, pair[1])):
            opt.zero_grad()
            for i, p in enumerate(ps):
                if i in filled:
                    opt._slots[i].copy_(grads[i])
                p.grad = grads[i].clone() if i not in filled or i in besides else None
            if filled:                                                  # as a producer of that group reports it
                opt._direct.update(filled)
                opt._direct_groups.add(("group",) + filled)
        norms = [float(opt.backward_step(max_norm=0.5)) for opt in (a, b)]
        want = torch.cat([(x * (2 if i in besides else 1)).double().reshape(-1) for i, x in enumerate(grads)])
        assert abs(norms[0] - float(want.norm())) <= 2 * 2.0 ** -24 * norms[0]
        assert norms[0] == norms[1] and torch.equal(a.flat_g, b.flat_g) and torch.equal(a.flat_p, b.flat_p)


def test_norm_counts_the_mean_over_ranks():
    from instancerefer_amd.optim import FlatAdam
    ps = params_of([(50,)], 4)
    opt = FlatAdam(ps, lr=1e-2, world_size=4)                           # (no process group: the sum over ranks stands in flat_g)
    ps[0].grad = torch.full((50,), 8.0, device=DEV)
    assert abs(float(opt.backward_step(max_norm=1.0)) - 2.0 * math.sqrt(50)) <= 1e-5
