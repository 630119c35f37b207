"""Plain 64-bit restatement of the packed-attention formulas (forward, gradients) with a bound on what 32-bit arithmetic, one rounding of
the softmax's weights and of the score gradients, and one rounding of each result may differ from it, value by value."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative
U32 = 2.0 ** -24


def reference(q, k, v, cu_q, cu_k, dout=None, causal=False, scale=None, table=None, buckets=None):
    """CPU tensors of the operator's types -> {name: (64-bit value, bound on |operator - value|)}"""
    dt = q.dtype
    tq, heads, dim = q.shape
    tk, kv, _ = k.shape
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    up, sub = HALF[dt], (2.0 ** -25 if dt == torch.float16 else 0.0)       # float16 below 2^-14: half a step is 2^-25
    low = 2.0 ** -133 if dt != torch.float16 else 2.0 ** -25               # a result below the normal range
    d = lambda t: t.detach().double()  # noqa: E731
    o, eo = torch.zeros(tq, heads, dim, dtype=torch.float64), torch.zeros(tq, heads, dim, dtype=torch.float64)
    g = {n: torch.zeros(t.shape, dtype=torch.float64) for n, t in (("dq", q), ("dk", k), ("dv", v), ("edq", q), ("edk", k), ("edv", v))}
    dtab = etab = None
    if table is not None:
        dtab, etab = torch.zeros(table.shape, dtype=torch.float64), torch.zeros(table.shape, dtype=torch.float64)
        far = (buckets.shape[0] - 1) // 2
    for b in range(cu_q.shape[0] - 1):
        r0, r1, c0, c1 = int(cu_q[b]), int(cu_q[b + 1]), int(cu_k[b]), int(cu_k[b + 1])
        lq, lk = r1 - r0, c1 - c0
        if lq == 0 or lk == 0:
            continue
        i, j = torch.arange(lq)[:, None], torch.arange(lk)[None, :]
        seen = (j <= i + lk - lq) if causal else torch.ones(lq, lk, dtype=torch.bool)
        for h in range(heads):
            hk = h // (heads // kv)
            Q, K, V = d(q[r0:r1, h]), d(k[c0:c1, hk]), d(v[c0:c1, hk])
            s = scale * (Q @ K.t())
            # a dot product of `dim` terms, the scale, log2 e, the bias and the subtraction of the maximum in 32 bits (all in exponent units)
            es = (dim + 4) * U32 * scale * (Q.abs() @ K.abs().t()) + 4 * U32 * s.abs()
            if table is not None:
                kind = buckets.long()[(j - i - (lk - lq)).clamp(-far, far) + far]
                bias = d(table)[kind, h]
                fine = torch.where(bias.abs() == math.inf, torch.zeros_like(bias), bias)
                s, es = s + bias, es + 4 * U32 * fine.abs().clamp(max=1e4) + torch.where(fine.abs() > 1e30, torch.zeros_like(fine), 4 * U32 * fine.abs())
            s = torch.where(seen, s, torch.full_like(s, -math.inf))
            m = s.amax(1, keepdim=True)
            m = torch.where(m == -math.inf, torch.zeros_like(m), m)
            e = torch.exp(s - m)
            l = e.sum(1, keepdim=True)
            P = torch.where(l > 0, e / l.clamp(min=1e-300), torch.zeros_like(e))
            # relative error of a normalised weight: of its exponent, of the row maximum's, of the exponential (2 ulp), of the sum
            E = 2 * torch.where(seen, es, torch.zeros_like(es)).amax(1, keepdim=True) + (lk + 16) * U32
            O = P @ V
            A = P @ V.abs()
            EO = (E + up + (lk + 8) * U32) * A + HALF[dt] * O.abs() + low
            ED = (E + up + (lk + 8) * U32) * A + HALF[dt] ** 2 * O.abs() + low       # ... with what the rounding left over added back
            o[r0:r1, h], eo[r0:r1, h] = O, EO
            if dout is None:
                continue
            G = d(dout[r0:r1, h])
            dP = G @ V.t()
            D = (G * O).sum(1, keepdim=True)
            S = P * (dP - D)
            eS = E * S.abs() + P * ((dim + 4) * U32 * (G.abs() @ V.abs().t()) + (G.abs() * (EO if dt == torch.float32 else ED)).sum(1, keepdim=True)
                                    + (dim + 4) * U32 * (G.abs() * O.abs()).sum(1, keepdim=True)) + 4 * U32 * S.abs()
            eR = eS + up * S.abs() + sub
            g["dq"][r0:r1, h] = scale * (S @ K)
            g["edq"][r0:r1, h] = scale * (eR @ K.abs()) + scale * (lk + 8) * U32 * (S.abs() @ K.abs())
            g["dk"][c0:c1, hk] += scale * (S.t() @ Q)
            g["edk"][c0:c1, hk] += scale * (eR.t() @ Q.abs()) + scale * (lq * heads // kv + 8) * U32 * (S.abs().t() @ Q.abs())
            g["dv"][c0:c1, hk] += P.t() @ G
            g["edv"][c0:c1, hk] += ((E + up) * P + sub / 1024).t() @ G.abs() + (lq * heads // kv + 8) * U32 * (P.t() @ G.abs())
            if table is not None:
                n = table.shape[0]
                flat = kind.reshape(-1)
                dtab[:, h] += torch.zeros(n, dtype=torch.float64).index_add_(0, flat, S.reshape(-1))
                etab[:, h] += torch.zeros(n, dtype=torch.float64).index_add_(0, flat, (eS + (lq + lk) * U32 * S.abs()).reshape(-1))
    got = {"out": (o, eo)}
    if dout is not None:
        for n in ("dq", "dk", "dv"):
            got[n] = (g[n], g["e" + n] + HALF[dt] * g[n].abs() + low)
        if table is not None:
            got["dtable"] = (dtab, etab + HALF[table.dtype] * dtab.abs() + low)
    return got


def check(got, want, name):
    """every value within its bound; the message says the worst"""
    value, bound = want
    x = got.detach().double().cpu()
    assert x.shape == value.shape, (name, x.shape, value.shape)
    assert torch.isfinite(x).all(), "%s: not finite" % name
    off = (x - value).abs()
    worst = float((off / bound.clamp(min=1e-300)).max()) if x.numel() else 0.0
    assert worst <= 1.0, "%s: off by %.3g of its bound (value %.3g, off %.3g)" % (name, worst, float(value.reshape(-1)[(off / bound).argmax()]), float(off.max()))
    return worst
