"""Short 16-bit calls: the output is the 64-bit value rounded once, but for 32-bit arithmetic — the softmax's weights enter the second
product in two terms, so that their own rounding does not reach the output or, through it, the gradients."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("lens,heads,kv,dim", [([20, 57, 3, 130], 4, 2, 32), ([200, 300], 16, 16, 32), ([20, 57, 3, 130], 4, 2, 64), ([33], 2, 1, 128), ([200, 300], 2, 2, 40)])
def test_output_is_rounded_once(kind, causal, bias, lens, heads, kv, dim):
    from instancerefer_amd.attention import attention_packed, relative_buckets
    print("case", kind, causal, bias, lens, heads, kv, dim, flush=True)
    dt, rows = TYPES[kind], sum(lens)
    half = torch.finfo(dt).eps / 2
    g = torch.Generator().manual_seed(rows + dim)
    q, k, v = (torch.randn(rows, h, dim, generator=g).to(dt) for h in (heads, kv, kv))
    table = torch.randn(8, heads, generator=g)
    buckets = relative_buckets(8, 16)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    args = {"bias": table.to(DEV), "buckets": buckets.to(DEV)} if bias else {}
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = attention_packed(*leaves, cu.to(DEV), causal=causal, **args).detach()
    with torch.no_grad():
        assert torch.equal(got, attention_packed(*leaves, cu.to(DEV), causal=causal, **args))
    got = got.double().cpu()
    scale = 1 / math.sqrt(dim)
    low = 2.0 ** -25 if kind == "f16" else 2.0 ** -133
    for r0, r1 in zip(cu.tolist(), cu.tolist()[1:]):
        n = r1 - r0
        away = torch.arange(n)[None, :] - torch.arange(n)[:, None]
        for h in range(heads):
            Q, K, V = q[r0:r1, h].double(), k[r0:r1, h // (heads // kv)].double(), v[r0:r1, h // (heads // kv)].double()
            s = scale * (Q @ K.t())
            es = (dim + 4) * U32 * scale * (Q.abs() @ K.abs().t()) + 4 * U32 * s.abs()
            if bias:
                b = table.double()[buckets.long()[away.clamp(-16, 16) + 16], h]
                s, es = s + b, es + 8 * U32 * b.abs()
            if causal:
                s = torch.where(away <= 0, s, torch.full_like(s, -math.inf))
                es = torch.where(away <= 0, es, torch.zeros_like(es))
            e = torch.exp(s - s.amax(1, keepdim=True))
            l = e.sum(1, keepdim=True)
            A, O = e @ V.abs() / l, e @ V / l
            # of a weight: its exponent's and the row maximum's 32-bit arithmetic, the sums', and the second term's rounding (half a step of half a
            # step; in float16 also 2^-25 where the row's largest weight is 2^7); then the output's own
            sub = 2.0 ** -32 / l * V.abs().sum(0, keepdim=True) if kind == "f16" else 0
            off = (2 * es.amax(1, keepdim=True) + half ** 2 + (2 * n + 24) * U32) * A + sub + half * O.abs() + low
            far = (got[r0:r1, h] - O).abs() / off
            assert float(far.max()) <= 1.0, "%.3g of its bound" % float(far.max())
