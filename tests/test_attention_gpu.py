"""attention_packed (csrc/irx_attn.hip, csrc/irx_attn_bwd.hip) against the formula in 64 bits, value by value within derived bounds."""
import math

import pytest
import torch

from attention_ref import check, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["cpp", "py"])
def backend(request, monkeypatch):
    """the C++ autograd node and the Python one"""
    from instancerefer_amd import attention, _nodes
    if request.param == "cpp":
        assert _nodes.load() is not None
    monkeypatch.setattr(attention, "BACKEND", "py" if request.param == "py" else "auto")


TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def make(lens, klens, heads, kv, dim, dt, seed=0, extra=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda n, h, s: (torch.randn(n, h, dim, generator=g) * s).to(dt)  # noqa: E731
    tq, tk = sum(lens) + extra, sum(klens) + extra
    return r(tq, heads, spread), r(tk, kv, spread), r(tk, kv, 1.0), r(tq, heads, 1.0)


def run(q, k, v, cu, cuk, dout, causal=False, scale=None, table=None, buckets=None):
    from instancerefer_amd.attention import attention_packed
    ts = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    tb = table.to(DEV).requires_grad_(True) if table is not None else None
    o = attention_packed(*ts, cu.to(DEV), cuk.to(DEV), causal=causal, scale=scale, bias=tb, buckets=buckets.to(DEV) if buckets is not None else None)
    grads = torch.autograd.grad(o, ts + ([tb] if tb is not None else []), dout.to(DEV))
    got = dict(zip(("dq", "dk", "dv", "dtable"), grads))
    got["out"] = o
    return got


def compare(lens, klens, heads, kv, dim, kind, causal=False, table=None, buckets=None, scale=None, seed=0, spread=1.0):
    q, k, v, do = make(lens, klens, heads, kv, dim, TYPES[kind], seed, spread=spread)
    cu, cuk = offsets(lens), offsets(klens)
    print("case", lens[:8], klens[:8], heads, kv, dim, kind, causal, flush=True)
    got = run(q, k, v, cu, cuk, do, causal, scale, table, buckets)
    want = reference(q, k, v, cu, cuk, do, causal, scale, table, buckets)
    return {n: check(got[n], want[n], n) for n in want}


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_forward_and_gradients_of_ragged_sequences(kind, dim, causal):
    compare([1, 33, 64, 130, 5, 200], [1, 33, 64, 130, 5, 200], 4, 2, dim, kind, causal)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 2), (8, 1), (3, 3)])
def test_grouped_heads(kind, heads, kv):
    compare([70, 129], [70, 129], heads, kv, 64, kind, True, seed=3)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
def test_queries_and_keys_of_different_lengths_and_empty_sequences(kind, causal):
    # more queries than keys under a causal mask leaves rows with no key; sequences without queries, without keys, without both
    compare([40, 3, 0, 17, 0, 129, 64], [10, 300, 25, 0, 0, 128, 65], 4, 4, 64, kind, causal, seed=5)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("narrow", [False, True])
def test_position_bias_and_its_gradient(kind, both, narrow):
    from instancerefer_amd.attention import relative_buckets
    dt = TYPES[kind]
    table = (torch.randn(16, 4, generator=torch.Generator().manual_seed(9)) * 1.5).to(dt if narrow else torch.float32)
    compare([1, 40, 150, 333], [1, 40, 150, 333], 4, 2, 64, kind, not both, table=table, buckets=relative_buckets(16, 50, both), seed=7)


def test_position_bias_with_keys_of_their_own_length_and_a_free_map(backend):
    table = torch.randn(5, 2, generator=torch.Generator().manual_seed(1))
    buckets = torch.randint(0, 5, (2 * 512 + 1,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    compare([90, 7, 1], [33, 700, 0], 2, 2, 32, "f32", False, table=table, buckets=buckets)
    compare([90, 200, 1], [33, 700, 0], 2, 1, 128, "f32", True, table=table, buckets=buckets)
    compare([90, 7, 1], [33, 700, 5], 2, 2, 128, "bf16", True, table=table[:, :2], buckets=torch.zeros(1, dtype=torch.int32))


def test_position_bias_that_forbids_buckets():
    from instancerefer_amd.attention import relative_buckets
    buckets = relative_buckets(8, 20, True)
    table = torch.randn(8, 2, generator=torch.Generator().manual_seed(4))
    table[5] = -math.inf                       # keys right behind the query
    table[1:4, 1] = torch.finfo(torch.float32).min
    compare([60, 1], [60, 1], 2, 1, 64, "f32", False, table=table, buckets=buckets)
    table[:] = torch.finfo(torch.float32).min  # every key equally forbidden: the formula's softmax is the mean
    q, k, v, do = make([50], [50], 2, 1, 64, torch.float32, 3, spread=0.1)
    cu = offsets([50])
    got = run(q, k, v, cu, cu, do, False, None, table, buckets)
    mean = v.double().mean(0, keepdim=True).expand(50, 1, 64).repeat(1, 2, 1)
    assert float((got["out"].detach().double().cpu() - mean).abs().max()) <= 50 * 2.0 ** -24 * float(v.abs().max())
    table[:] = -math.inf                       # no key at all: zeros, no gradient
    got = run(q, k, v, cu, cu, do, False, None, table, buckets)
    for n, t in got.items():
        assert float(t.abs().max()) == 0.0, n


@pytest.mark.parametrize("kind,heads,kv,dim,causal", [("bf16", 16, 4, 32, False), ("f16", 9, 3, 64, True), ("f32", 4, 4, 128, True), ("f32", 60, 20, 32, True)])
def test_key_axis_in_parts_with_many_rows(kind, heads, kv, dim, causal):
    """parts of the key axis joined row by row, several rows to a workgroup; the last case: two parts although the launch fills the chip"""
    from instancerefer_amd import _lib
    rows = 1101
    code, mask = {"f32": 0, "bf16": 1, "f16": 2}[kind], 2 * causal
    assert _lib.load().irx_attn_packed_fwd_workspace_bytes(rows, rows, 1, heads, kv, dim, code, mask) > 0
    assert rows * heads * (dim // 4) >= 512 * 256
    compare([rows], [rows], heads, kv, dim, kind, causal, seed=16)


@pytest.mark.parametrize("kind,dim,causal", [("bf16", 64, True), ("f32", 128, False), ("f16", 32, True)])
def test_key_axis_in_parts_with_a_bias(kind, dim, causal, backend):
    from instancerefer_amd.attention import relative_buckets
    table = torch.randn(12, 4, generator=torch.Generator().manual_seed(17))
    compare([1300, 40, 1100], [1300, 900, 1100], 4, 2, dim, kind, causal, table=table, buckets=relative_buckets(12, 60, not causal), seed=18)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_bias_gradient_without_keys_and_of_many_buckets(kind, backend):
    table = torch.randn(700, 3, generator=torch.Generator().manual_seed(13))
    buckets = torch.arange(700, dtype=torch.int32)[:2 * 340 + 1]              # a bucket per distance, some that none has
    compare([300, 64], [300, 20], 3, 3, 32, kind, False, table=table, buckets=buckets, seed=14)
    junk = [torch.full((700, 3), math.nan, device=DEV) for _ in range(8)]      # what lies where the result will
    del junk
    q, k, v, do = make([70, 5], [0, 0], 3, 3, 64, TYPES[kind], 15)
    got = run(q, k, v, offsets([70, 5]), offsets([0, 0]), do, False, None, table, buckets)
    for n, t in got.items():
        assert not t.numel() or float(t.abs().max()) == 0.0, n


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_lowest_bias_beyond_the_clipped_distance(kind, dim):
    """every key a row sees is equally forbidden, most of them beyond the clipped distance: the mean, and the mean's gradients"""
    from instancerefer_amd.attention import relative_buckets
    table = torch.full((8, 2), torch.finfo(torch.float32).min)
    compare([40, 1, 130], [200, 170, 400], 2, 1, dim, kind, True, table=table, buckets=relative_buckets(8, 20, False), spread=2.0)
    table[:7] = -math.inf                      # ... and those within it not allowed at all
    compare([40, 1, 130], [200, 170, 400], 2, 1, dim, kind, True, table=table, buckets=relative_buckets(8, 20, False), spread=2.0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_outside_every_sequence_and_other_sequences_never_matter(kind, causal):
    from instancerefer_amd.attention import attention_packed
    lens = [50, 1, 77]
    q, k, v, do = make(lens, lens, 4, 2, 64, TYPES[kind], 11)
    cu = offsets(lens)
    want = run(q, k, v, cu, cu, do, causal)
    bad = lambda t, n: torch.cat((t, torch.full((n,) + t.shape[1:], math.nan).to(t.dtype)))  # noqa: E731
    got = run(bad(q, 40), bad(k, 40), bad(v, 40), cu, cu, bad(do, 40), causal)
    for n in want:
        rows = want[n].shape[0]
        assert torch.equal(got[n][:rows], want[n]), n
        assert float(got[n][rows:].float().abs().max()) == 0.0, n
    # rows in front of the first sequence
    front = lambda t: torch.cat((torch.full((5,) + t.shape[1:], math.nan).to(t.dtype), t))  # noqa: E731
    got = run(front(q), front(k), front(v), cu + 5, cu + 5, front(do), causal)
    for n in want:
        assert torch.equal(got[n][5:], want[n]) and float(got[n][:5].float().abs().max()) == 0.0, n
    # a neighbour of infinities
    k2, v2 = k.clone(), v.clone()
    k2[50:51], v2[50:51] = math.inf, math.nan
    o = attention_packed(q.to(DEV), k2.to(DEV), v2.to(DEV), cu.to(DEV), causal=causal)
    assert torch.equal(o[:50], want["out"][:50]) and torch.equal(o[51:], want["out"][51:])


def test_infinite_keys_behind_the_causal_border_do_not_matter():
    lens = [100]
    q, k, v, do = make(lens, lens, 2, 2, 64, torch.float32, 12)
    cu = offsets(lens)
    want = run(q, k, v, cu, cu, do, True)["out"]
    k[60:] = math.inf
    got = run(q, k, v, cu, cu, do, True)["out"]
    assert torch.equal(got[:60], want[:60])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strided_views_and_other_head_dimensions(kind, backend):
    from instancerefer_amd.attention import attention_packed
    dt, lens = TYPES[kind], [37, 100]
    g = torch.Generator().manual_seed(2)
    cu = offsets(lens).to(DEV)
    fused = torch.randn(137, 8 * 64, generator=g).to(dt).to(DEV).requires_grad_(True)
    q, k, v = fused[:, :256].view(137, 4, 64), fused[:, 256:384].view(137, 2, 64), fused[:, 384:].view(137, 2, 64)
    o = attention_packed(q, k, v, cu, causal=True)
    do = torch.randn(137, 4, 64, generator=g).to(dt).to(DEV)
    (df,) = torch.autograd.grad(o, fused, do)
    qc, kc, vc = (t.detach().contiguous().requires_grad_(True) for t in (q, k, v))
    o2 = attention_packed(qc, kc, vc, cu, causal=True)
    want = torch.autograd.grad(o2, (qc, kc, vc), do)
    assert torch.equal(o, o2) and torch.equal(df, torch.cat([t.reshape(137, -1) for t in want], 1))
    # heads before rows, a shifted view, a gradient with strides of its own
    qt = qc.detach().transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(137 * 2 * 64 + 1, dtype=dt, device=DEV)[1:].view(137, 2, 64)
    odd.copy_(kc.detach())
    wide = torch.zeros(137, 4, 128, dtype=dt, device=DEV)
    wide[..., :64] = do
    qt.requires_grad_(True)
    o3 = attention_packed(qt, odd, vc.detach(), cu, causal=True)
    assert torch.equal(o3, o2)
    (dq3,) = torch.autograd.grad(o3, qt, wide[..., :64])
    assert torch.equal(dq3, want[0])
    (dq4,) = torch.autograd.grad(attention_packed(qt, odd, vc.detach(), cu, causal=True).sum(), qt)       # an expanded gradient
    (dq5,) = torch.autograd.grad(attention_packed(qt, odd, vc.detach(), cu, causal=True), qt, torch.ones_like(o3))
    assert torch.equal(dq4, dq5)
    for dim in (1, 40, 100):
        compare([30, 70], [30, 70], 2, 1, dim, kind, True, seed=dim)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_few_queries_over_many_keys_in_parts(kind, dim):
    from instancerefer_amd import _lib
    lens, klens = [1, 3, 1, 0, 2], [3000, 1, 1500, 700, 0]
    assert _lib.load().irx_attn_packed_fwd_workspace_bytes(sum(lens), sum(klens), 5, 4, 2, dim, 0, 0) > 0
    compare(lens, klens, 4, 2, dim, kind)
    compare([2, 1], [2500, 4000], 2, 2, dim, kind, True, seed=2)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv", [(3, 1), (32, 1), (40, 1), (5, 5), (12, 4)])
def test_few_queries_of_every_grouping(kind, heads, kv):
    """rows of a few-query tile are (token, head of the group): groups that do not divide 32, that fill it, that exceed it; one sequence
    with more queries than a tile holds among short ones; causal with more queries than keys"""
    compare([1, 14, 2, 1, 1, 0], [900, 700, 40, 2500, 1, 33], heads, kv, 32, kind, False, seed=heads)
    compare([1, 14, 5, 1, 1, 0, 1, 1, 1, 1], [900, 700, 3, 2500, 1, 33, 900, 0, 800, 1000], heads, kv, 64, kind, True, seed=heads)


def test_few_queries_with_a_bias_in_parts():
    from instancerefer_amd.attention import relative_buckets
    table = torch.randn(8, 2, generator=torch.Generator().manual_seed(3))
    compare([1, 2], [3000, 2600], 2, 1, 64, "bf16", False, table=table, buckets=relative_buckets(8, 30))


def test_keys_shared_by_many_query_heads_in_parts():
    """few key tiles, many queries: the backward gives each workgroup a part of the queries and joins dk, dv"""
    from instancerefer_amd import _lib
    one = _lib.load().irx_attn_packed_bwd_workspace_bytes
    assert one(1400, 1400, 2, 8, 2, 64, 1, -1) > 8 * 1400 * 4      # more than D alone: the parts
    for kind, dim in (("bf16", 64), ("f16", 128), ("f32", 32)):
        compare([900, 500], [900, 500], 8, 2, dim, kind, True, seed=dim)
    compare([1100, 3], [70, 0], 2, 1, 64, "bf16", False, seed=1)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_scores_of_every_size(kind):
    for spread in (0.01, 6.0):
        compare([150], [150], 2, 1, 64, kind, True, spread=spread, seed=4)
    compare([60], [60], 2, 1, 64, kind, False, scale=0.5, seed=6)


def test_against_differences():
    from instancerefer_amd.attention import attention_packed, relative_buckets
    lens = [9, 30]
    q, k, v, do = make(lens, lens, 2, 1, 32, torch.float32, 21, spread=0.7)
    cu = offsets(lens)
    buckets = relative_buckets(8, 12, False)
    table = torch.randn(8, 2, generator=torch.Generator().manual_seed(5))
    got = run(q, k, v, cu, cu, do, True, None, table, buckets)
    f = lambda a: float((attention_packed(*[t.to(DEV) for t in a[:3]], cu.to(DEV), causal=True, bias=a[3].to(DEV), buckets=buckets.to(DEV)).double()  # noqa: E731
                         * do.to(DEV).double()).sum())
    base = [q, k, v, table]
    for n, name in enumerate(("dq", "dk", "dv", "dtable")):
        way = torch.randn(base[n].shape, generator=torch.Generator().manual_seed(n))
        step = 1e-2
        up, down = list(base), list(base)
        up[n], down[n] = base[n] + step * way, base[n] - step * way
        want = (f(up) - f(down)) / (2 * step)
        have = float((got[name].double().cpu() * way.double()).sum())
        # central difference: third-order term about step^2 times the value, rounding of f about 1e-6 / step
        assert abs(want - have) <= 2e-3 * max(1.0, abs(have)) * 10, (name, want, have)


def test_rows_beyond_32_bit_offsets():
    """key rows 2^20 elements apart: the last ones lie behind 2^31 elements (and 2^32 bytes)"""
    from instancerefer_amd.attention import attention_packed
    n, stride = 2200, 1 << 20
    room = torch.empty(n * stride, dtype=torch.bfloat16, device=DEV)
    far = room.as_strided((n, 2, 64), (stride, 64, 1))
    q, k, v, do = (t.to(DEV) for t in make([n], [n], 2, 2, 64, torch.bfloat16, 31))
    far.copy_(k)
    cu = offsets([n]).to(DEV)
    a = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = attention_packed(*a, cu, causal=True)
    want = torch.autograd.grad(o, a, do)
    b = [q.clone().requires_grad_(True), far.requires_grad_(True), v.clone().requires_grad_(True)]
    o2 = attention_packed(*b, cu, causal=True)
    got = torch.autograd.grad(o2, b, do)
    assert torch.equal(o, o2) and all(torch.equal(x, y) for x, y in zip(want, got))


def test_a_captured_few_query_launch():
    from instancerefer_amd.attention import attention_packed
    q, k, v, _ = (t.to(DEV) for t in make([1, 1, 2], [900, 3000, 700], 8, 2, 128, torch.bfloat16, 81))
    cu, cuk = offsets([1, 1, 2]).to(DEV), offsets([900, 3000, 700]).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_packed(q, k, v, cu, cuk)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = attention_packed(q, k, v, cu, cuk)
    for ends in ([900, 3000, 700], [4600, 0, 0], [1, 2, 3]):
        cuk.copy_(offsets(ends))
        want = attention_packed(q, k, v, cu, cuk)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
        q.mul_(0.7)


def test_two_calls_at_once_on_two_streams():
    from instancerefer_amd.attention import attention_packed
    sets = [make([700, 300], [700, 300], 4, 2, 64, torch.bfloat16, s) for s in (91, 92)]
    sets = [[t.to(DEV) for t in s] for s in sets]
    cu = offsets([700, 300]).to(DEV)
    want = [attention_packed(*s[:3], cu, causal=True) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n in range(2):
            with torch.cuda.stream(streams[n]):
                got[n].append(attention_packed(*sets[n][:3], cu, causal=True))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(x, want[n]) for x in got[n])


def test_same_bits_every_time_and_on_another_stream():
    from instancerefer_amd.attention import relative_buckets
    lens = [300, 64, 111]
    q, k, v, do = make(lens, lens, 4, 2, 64, torch.bfloat16, 41)
    cu = offsets(lens)
    table = torch.randn(32, 4, generator=torch.Generator().manual_seed(8))
    buckets = relative_buckets(32, 128)
    want = run(q, k, v, cu, cu, do, False, None, table, buckets)
    side = torch.cuda.Stream()
    for n in range(4):
        with torch.cuda.stream(side if n % 2 else torch.cuda.current_stream()):
            got = run(q, k, v, cu, cu, do, False, None, table, buckets)
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(got[name], want[name]), name


@pytest.mark.parametrize("kind,dim,far", [("bf16", 64, 40), ("f32", 128, 512), ("f16", 128, 512)])      # up to 160 KB of LDS
def test_captured_forward_and_backward_with_new_offsets(backend, kind, dim, far):
    from instancerefer_amd.attention import attention_packed, relative_buckets
    dt, total = TYPES[kind], 260
    g = torch.Generator().manual_seed(6)
    q, k, v = ((torch.randn(total, h, dim, generator=g)).to(dt).to(DEV).requires_grad_(True) for h in (4, 2, 2))
    do = torch.randn(total, 4, dim, generator=g).to(dt).to(DEV)
    table = torch.randn(16, 4, generator=g).to(DEV).requires_grad_(True)
    buckets = relative_buckets(16, far, False, device=DEV)
    cu = offsets([100, 60, 100]).to(DEV)
    leaves = [q, k, v, table]

    def step():
        o = attention_packed(q, k, v, cu, causal=True, bias=table, buckets=buckets)
        return [o] + list(torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for lens in ([100, 60, 100], [1, 259, 0], [0, 0, 200], [130, 130, 0]):
        cu.copy_(offsets(lens))
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), lens
        with torch.no_grad():
            q.mul_(0.9)


def test_capture_beside_a_living_eager_graph_is_refused(backend):
    """a captured backward would make the eager graph's stream wait inside the capture: refused before anything is recorded, in the forward
    and, where the forward was eager, in the backward"""
    from instancerefer_amd.attention import attention_packed
    q, k, v, do = (t.to(DEV) for t in make([40], [40], 2, 2, 64, torch.float32, 61))
    cu = offsets([40]).to(DEV)
    q.requires_grad_(True)
    alive = attention_packed(q, k, v, cu)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            attention_packed(q, k, v, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with torch.no_grad():
            held = attention_packed(q, k, v, cu)              # without gradients there is nothing to refuse
    graph.replay()
    assert torch.equal(held, alive)
    torch.cuda.synchronize()
    assert float(torch.autograd.grad(alive, q, do)[0].abs().max()) > 0


@pytest.mark.parametrize("how", ["padded", "copied", "table"])
def test_capture_beside_a_living_eager_graph_of_copied_leaves(how, backend):
    """a leaf that the operator pads or copies before its node sees it is found too"""
    from instancerefer_amd.attention import attention_packed, relative_buckets
    dim = 40 if how == "padded" else 64
    q, k, v, do = (t.to(DEV) for t in make([40], [40], 2, 2, dim, torch.float32, 62))
    cu, args = offsets([40]).to(DEV), {}
    if how == "copied":
        buf = torch.empty(q.numel() + 1, device=DEV)[1:]
        q = buf.copy_(q.reshape(-1)).view(q.shape)
    if how == "table":
        leaf = torch.zeros((2, 8), device=DEV).t()                      # (8, 2), not contiguous
        args = {"bias": leaf, "buckets": relative_buckets(8, 16, device=DEV)}
    else:
        leaf = q
    leaf.requires_grad_(True)
    alive = attention_packed(q, k, v, cu, **args)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            attention_packed(q, k, v, cu, **args)
    torch.cuda.synchronize()
    assert float(torch.autograd.grad(alive, leaf, do)[0].abs().max()) > 0


def test_second_derivative_is_refused(backend):
    from instancerefer_amd.attention import attention_packed
    q, k, v, do = (t.to(DEV) for t in make([9], [9], 2, 2, 32, torch.float32, 71))
    q.requires_grad_(True)
    o = attention_packed(q, k, v, offsets([9]).to(DEV))
    (dq,) = torch.autograd.grad((o * o).sum(), q, create_graph=True)      # a gradient that depends on q itself
    with pytest.raises(RuntimeError, match="differentiable once|once_differentiable"):
        dq.sum().backward()


def test_offsets_are_clamped_to_the_rows():
    """offsets beyond the tensors reach no memory outside them: they are clamped on the device"""
    from instancerefer_amd.attention import attention_packed
    q, k, v, _ = (t.to(DEV) for t in make([64], [64], 2, 2, 64, torch.bfloat16, 51))
    want = attention_packed(q, k, v, offsets([64]).to(DEV))
    got = attention_packed(q, k, v, torch.tensor([-5, 1 << 30], dtype=torch.int32, device=DEV))
    assert torch.equal(got, want)


def test_no_rows_and_no_keys(backend):
    from instancerefer_amd.attention import attention_packed
    z = lambda n, h: torch.zeros(n, h, 64, device=DEV, requires_grad=True)  # noqa: E731
    cu0, cu = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([0, 0], dtype=torch.int32, device=DEV)
    assert attention_packed(z(0, 4), z(0, 2), z(0, 2), cu).shape == (0, 4, 64)
    q = torch.ones(5, 4, 64, device=DEV, requires_grad=True)
    k, v = z(0, 2), z(0, 2)
    o = attention_packed(q, k, v, torch.tensor([0, 5], dtype=torch.int32, device=DEV), cu)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
    assert float(o.abs().max()) == 0 and float(dq.abs().max()) == 0 and dk.shape == (0, 2, 64)
    k, v = z(7, 2), z(7, 2)
    q0 = z(0, 4)
    tb = torch.ones(3, 4, device=DEV, requires_grad=True)
    o = attention_packed(q0, k, v, cu, torch.tensor([0, 7], dtype=torch.int32, device=DEV), bias=tb, buckets=torch.zeros(3, dtype=torch.int32, device=DEV))
    for t in torch.autograd.grad(o, (q0, k, v, tb), torch.ones_like(o)):
        assert t.numel() == 0 or float(t.abs().max()) == 0
    o = attention_packed(q, k.detach() + 1, v.detach() + 1, cu0, cu0.clone())      # no sequence at all: every row is outside
    assert float(o.abs().max()) == 0


def test_offsets_from_lengths():
    from instancerefer_amd.attention import packed_offsets
    lens = torch.tensor([3, 0, 7], device=DEV)
    assert packed_offsets(lens).tolist() == [0, 3, 3, 10] and packed_offsets(lens).dtype == torch.int32
