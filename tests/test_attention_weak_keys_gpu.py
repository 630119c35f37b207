"""Rows whose result comes from weights far below the row's largest: one key takes nearly all the weight and has a value of zero."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


def expected(q, k, v, scale):
    """(rows, heads, dim) over the keys of one sequence, 64 bits, and what may be off: the exponent's 32-bit arithmetic, a rounding of each weight
    to the type (in float16 also half the smallest step, 2^-25, of weights that are 2^7 for the row's largest key), sums, the result's rounding"""
    dt, heads, kv, dim = q.dtype, q.shape[1], k.shape[1], q.shape[2]
    half = torch.finfo(dt).eps / 2
    out, off = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for h in range(heads):
        Q, K, V = q[:, h].double(), k[:, h // (heads // kv)].double(), v[:, h // (heads // kv)].double()
        s = scale * (Q @ K.t())
        es = ((dim + 4) * U32 * scale * (Q.abs() @ K.abs().t()) + 4 * U32 * s.abs()).amax(1, keepdim=True)
        e = torch.exp(s - s.amax(1, keepdim=True))
        l = e.sum(1, keepdim=True)
        A = e @ V.abs() / l
        out[:, h] = e @ V / l
        sub = 2.0 ** -32 / l * V.abs().sum(0, keepdim=True) if dt == torch.float16 else 0
        low = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -133
        off[:, h] = (2 * es + half + (2 * k.shape[0] + 24) * U32) * A + sub + half * out[:, h].abs() + low
    return out, off


# below the largest by e^-14 = 2^-20.2 and e^-17.25 = 2^-24.9: in float16 steps of 2^-24 the first is 14 steps, the second one or none
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("gap", [9.25, 14.0, 17.25])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("rows,keys,heads,kv,dim,bias", [(70, 1000, 2, 1, 64, False), (70, 1000, 2, 1, 128, True), (70, 4003, 2, 1, 64, False), (1, 4003, 4, 1, 128, False),
                                                         (1, 4003, 2, 2, 64, True), (640, 4003, 8, 8, 32, False)])
def test_weights_far_below_the_largest(kind, gap, place, rows, keys, heads, kv, dim, bias):
    from instancerefer_amd.attention import attention_packed, relative_buckets
    print("case", kind, gap, place, rows, keys, heads, kv, dim, bias, flush=True)
    scale = 0.125
    g = torch.Generator().manual_seed(keys + rows)
    q, k = torch.zeros(rows, heads, dim), torch.zeros(keys, kv, dim)
    at = {"first": 0, "middle": keys // 2, "last": keys - 1}[place]
    q[..., 0], k[at, :, 0] = 8.0, gap
    q[..., 1], k[:, :, 1] = 1.0, torch.linspace(0.0, 4.0, keys)[:, None]   # the weak keys differ a little
    v = 30 + torch.rand(keys, kv, dim, generator=g) * 10
    v[at] = 0.0
    q, k, v = (t.to(TYPES[kind]) for t in (q, k, v))
    want, off = expected(q, k, v, scale)
    args = {}
    if bias:
        args = {"bias": torch.zeros(8, heads, device=DEV), "buckets": relative_buckets(8, 16, device=DEV)}
    cu, cuk = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (rows, keys))
    got = attention_packed(q.to(DEV), k.to(DEV), v.to(DEV), cu, cuk, scale=scale, **args)
    far = (got.double().cpu() - want).abs() / off
    assert float(far.max()) <= 1.0, "%.3g of its bound" % float(far.max())
    # with gradients: the same output, and weights that sum to one (every value 1, every output gradient 1: dv is the sum of weights)
    qs, ks, vs = (t.to(DEV).requires_grad_(True) for t in (q, k, torch.ones_like(v)))
    o = attention_packed(qs, ks, vs, cu, cuk, scale=scale, **args)
    (dv,) = torch.autograd.grad(o, vs, torch.ones_like(o))
    total = dv.double().sum(0).cpu()
    half, each = torch.finfo(TYPES[kind]).eps / 2, rows * (heads // kv)    # rows that a key's dv sums over
    # the weak keys' sums of weights may lie where float16 has steps of 2^-24 (2^-25 each), the weights in it are lifted by 2^10
    slack = keys * (2.0 ** -25 + each * 2.0 ** -35) if kind == "f16" else 0.0
    assert float((total - each).abs().max()) <= (2 * half + (3 * keys + 64) * U32) * each + slack
