"""Attention over packed sequences on the irx kernels (csrc/irx_attn.hip, csrc/irx_attn_bwd.hip), with an optional learned relative
position bias by buckets.

Stands beside `dense.gru_packed`: the other way to let the words of a description see each other. Sequences of different lengths lie one
behind the other along the first axis (no padding), `cu` holds their offsets on the device, and no length is ever read by the host.

    cu = packed_offsets(lang_len)                                   # int32 (B + 1,)
    o = attention_packed(q, k, v, cu)                               # q (T, H, D), k / v (T, Hkv, D) -> (T, H, D)
    o = attention_packed(q, k, v, cu, bias=table, buckets=relative_buckets(32, 128, device=q.device))
    o = attention_packed(q, k, v, cu_objects, cu_words)             # queries of one set attending to another

Formula, per sequence and query head h with its key / value head h // (H / Hkv):
    s_ij = scale q_i . k_j (+ bias[buckets[far + clamp(j - (i + Lk - Lq), -far, far)], h]),   o_i = sum_j softmax_j(s_ij) v_j
over every key j of the sequence or, with `causal`, j <= i + Lk - Lq (the last query sees the last key). A query that sees no key gives
zeros and takes no gradient; so do rows outside every sequence (behind cu[-1]).

Types: float32 (products in float32), bfloat16, float16; scores, softmax and sums are float32, the softmax's weights and the score gradients
are rounded to the tensors' type where they enter the second products (in short launches the weights in two terms). In float16 a weight below
2^-21 of its row's largest keeps fewer than 10 bits, one below 2^-32 none; gradients of scores below 6e-8 vanish: scale the loss. In 16 bits a
forward that will be differentiated keeps a second tensor of the output's size, what its rounding left over, for the gradients' sake. An
exponent is good to 2^-22 of its score: weights of scores beyond 1e6 have no digits left, beyond 5e7 a row may come out as NaN or zeros.
Keys of other sequences and rows outside never reach a result, whatever they hold. A NaN or infinity in a later row of the SAME sequence
can reach earlier rows of its tile of 64 under `causal`, as in any matrix product. Head dimensions other than 32, 64 and 128 are padded to the
next of them (a copy), up to 128. Deterministic; captures into a graph (the offsets may change between replays, the shapes may not). A capture
with gradients is refused while an eager graph of the same leaves lives on another stream."""
import math
import os

import torch
from torch.autograd.function import once_differentiable

from . import _lib, _nodes

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_DIMS = (32, 64, 128)
MAX_FAR = 512
BACKEND = os.environ.get("IRX_ATTENTION_BACKEND", "auto")   # "py": the Python autograd.Function below even when the C++ node exists


def packed_offsets(lengths):
    """(B,) whole numbers -> int32 (B + 1,) offsets of the packed sequences, on the same device (no host read)."""
    if lengths.dim() != 1 or lengths.is_floating_point() or lengths.dtype == torch.bool:
        raise ValueError("packed_offsets: lengths must be a vector of whole numbers, got %s of %s" % (tuple(lengths.shape), lengths.dtype))
    cu = torch.zeros(lengths.shape[0] + 1, dtype=torch.int32, device=lengths.device)
    torch.cumsum(lengths, 0, dtype=torch.int32, out=cu[1:])
    return cu


def relative_buckets(num_buckets, max_distance, bidirectional=True, device=None):
    """Bucket of every clipped distance key - query: int32 (2 max_distance + 1,), index distance + max_distance.

    bidirectional: the upper half of the buckets is for keys behind the query (distance > 0), the lower half for the others; else every
    distance >= 0 is bucket 0 and all buckets are for keys before the query. Of a side's n buckets the first n // 2 hold one distance
    each, bucket n // 2 + t the distances from (n // 2) (max_distance / (n // 2))^(t / (n - n // 2)) on; everything from max_distance on is
    in the last one. The borders are found in whole numbers, so no rounding moves a distance across one."""
    num_buckets, max_distance = int(num_buckets), int(max_distance)
    n = num_buckets // 2 if bidirectional else num_buckets
    single = n // 2
    if n < 2 or (bidirectional and num_buckets % 2):
        raise ValueError("relative_buckets: %d buckets%s" % (num_buckets, " for two sides" if bidirectional else ""))
    if not single < max_distance <= MAX_FAR:
        raise ValueError("relative_buckets: max_distance must be above %d and at most %d, got %d" % (single, MAX_FAR, max_distance))
    steps, side, t = n - single, [], 0
    for d in range(max_distance + 1):
        if d < single:
            side.append(d)
            continue
        # d >= single (max / single)^((t + 1) / steps), both sides to the power of `steps`
        while t + 1 < steps and d ** steps * single ** (t + 1) >= max_distance ** (t + 1) * single ** steps:
            t += 1
        side.append(single + t)
    if bidirectional:
        both = side[:0:-1] + [side[0]] + [n + b for b in side[1:]]
    else:
        both = side[:0:-1] + [0] * (max_distance + 1)
    return torch.tensor(both, dtype=torch.int32, device=device)


def _rows(t):
    """The kernels read rows and heads in place from any strides that keep 16-byte alignment; everything else is copied."""
    e = t.element_size()
    if t.stride(2) == 1 and t.stride(0) * e % 16 == 0 and t.stride(0) * e < 1 << 24 and t.stride(1) * e % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)     # (contiguous() would keep a tensor that merely starts off 16 bytes)


def _table_args(table, buckets):
    if table is None:
        return (None, 1, None, 0, -1)
    return (table.data_ptr(), 1 if table.dtype == torch.float32 else 0, buckets.data_ptr(), table.shape[0], (buckets.shape[0] - 1) // 2)


def _forward(q, k, v, table, cu_q, cu_k, causal, scale, buckets, want_stats):
    tq, heads, dim = q.shape
    tk, kv_heads, _ = k.shape
    batch = cu_q.shape[0] - 1
    out = torch.empty((tq, heads, dim), dtype=q.dtype, device=q.device)
    stats = torch.empty((heads, tq, 2), dtype=torch.float32, device=q.device) if want_stats else None
    rest = torch.empty_like(out) if want_stats and q.dtype != torch.float32 else None      # what the output's rounding leaves over
    n = int(_lib.load().irx_attn_packed_fwd_workspace_bytes(tq, tk, batch, heads, kv_heads, dim, _TYPES[q.dtype],
                                                              (table is not None) + (2 if causal else 0)))
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    tb, tb_f32, mp, nb, far = _table_args(table, buckets)
    _lib.call("irx_attn_packed_fwd", q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
              v.stride(0), v.stride(1), cu_q.data_ptr(), cu_k.data_ptr(), batch, tq, tk, heads, kv_heads, dim, _TYPES[q.dtype], scale,
              causal, tb, tb_f32, mp, nb, max(far, 0), out.data_ptr(),
              rest.data_ptr() if rest is not None else None, stats.data_ptr() if want_stats else None,
              ws.data_ptr() if n else None, n, _lib.stream_ptr())
    return out, stats, rest


class AttentionPackedFn(torch.autograd.Function):
    """irx_attn_packed_fwd / irx_attn_packed_bwd as one node: (q, k, v, bias table) -> out."""

    @staticmethod
    def forward(ctx, q, k, v, table, cu_q, cu_k, causal, scale, buckets):
        out, stats, rest = _forward(q, k, v, table, cu_q, cu_k, causal, scale, buckets, True)
        ctx.save_for_backward(q, k, v, table, cu_q, cu_k, buckets, out, stats, rest)
        ctx.cfg = (causal, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, table, cu_q, cu_k, buckets, out, stats, rest = ctx.saved_tensors
        causal, scale = ctx.cfg
        if torch.cuda.is_current_stream_capturing():
            _nodes.refuse_foreign_behind("attention_packed")
        tq, heads, dim = q.shape
        tk, kv_heads, _ = k.shape
        batch = cu_q.shape[0] - 1
        dout = _rows(dout)
        dq = torch.empty((tq, heads, dim), dtype=q.dtype, device=q.device)
        dk = torch.empty((tk, kv_heads, dim), dtype=q.dtype, device=q.device)
        dv = torch.empty((tk, kv_heads, dim), dtype=q.dtype, device=q.device)
        dt = None
        if table is not None:
            dt = torch.empty_like(table) if tq else torch.zeros_like(table)
        tb, tb_f32, mp, nb, far = _table_args(table, buckets)
        n = int(_lib.load().irx_attn_packed_bwd_workspace_bytes(tq, tk, batch, heads, kv_heads, dim, _TYPES[q.dtype], far))
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device=q.device)
        _lib.call("irx_attn_packed_bwd", q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                  v.stride(0), v.stride(1), dout.data_ptr(), dout.stride(0), dout.stride(1), out.data_ptr(),
                  rest.data_ptr() if rest is not None else None, stats.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), batch, tq, tk, heads, kv_heads, dim, _TYPES[q.dtype], scale, causal, tb, tb_f32,
                  mp, nb, max(far, 0), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dt.data_ptr() if dt is not None else None,
                  ws.data_ptr(), n, _lib.stream_ptr())
        return dq, dk, dv, dt, None, None, None, None, None


def _check(q, k, v, cu_q, cu_k, bias, buckets):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError("attention_packed: %s must be (rows, heads, dim), got %s" % (name, tuple(t.shape)))
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("attention_packed: q, k, v must share one of float32, bfloat16, float16, got %s, %s, %s" % (q.dtype, k.dtype, v.dtype))
    if k.shape != v.shape:
        raise ValueError("attention_packed: k is %s, v is %s" % (tuple(k.shape), tuple(v.shape)))
    if k.shape[2] != q.shape[2] or not 1 <= q.shape[2] <= _DIMS[-1]:
        raise ValueError("attention_packed: head dimensions %d and %d (equal, at most %d)" % (q.shape[2], k.shape[2], _DIMS[-1]))
    if q.shape[1] < 1 or k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError("attention_packed: %d query heads over %d key / value heads" % (q.shape[1], k.shape[1]))
    for name, cu in (("cu_q", cu_q), ("cu_k", cu_k)):
        if cu.dim() != 1 or cu.shape[0] < 1 or cu.dtype != torch.int32 or not cu.is_contiguous():
            raise ValueError("attention_packed: %s must be a contiguous int32 vector of offsets (packed_offsets makes one)" % name)
    if cu_q.shape != cu_k.shape:
        raise ValueError("attention_packed: offsets of %d and %d sequences" % (cu_q.shape[0] - 1, cu_k.shape[0] - 1))
    if cu_k is cu_q and k.shape[0] != q.shape[0]:
        raise ValueError("attention_packed: %d query rows and %d key rows need offsets of their own" % (q.shape[0], k.shape[0]))
    if (bias is None) != (buckets is None):
        raise ValueError("attention_packed: a bias table and its bucket map come together")
    ts = [q, k, v, cu_q, cu_k]
    if bias is not None:
        if bias.dim() != 2 or bias.shape[1] != q.shape[1] or bias.shape[0] < 1 or bias.dtype not in (torch.float32, q.dtype):
            raise ValueError("attention_packed: the bias table must be (buckets, %d) in float32 or %s, got %s of %s"
                             % (q.shape[1], q.dtype, tuple(bias.shape), bias.dtype))
        if buckets.dim() != 1 or buckets.dtype != torch.int32 or not buckets.is_contiguous() or buckets.shape[0] % 2 == 0 \
                or buckets.shape[0] > 2 * MAX_FAR + 1:
            raise ValueError("attention_packed: the bucket map must be a contiguous int32 vector of 2 far + 1 values, far <= %d" % MAX_FAR)
        ts += [bias, buckets]
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("irx operators need tensors on a HIP device (got %s); the CPU path exists only as the test oracle "
                               "under /oracle" % t.device)
        if t.device != q.device:
            raise ValueError("attention_packed: tensors on %s and %s" % (q.device, t.device))


def attention_packed(q, k, v, cu_q, cu_k=None, causal=False, scale=None, bias=None, buckets=None):
    """softmax(scale q k^T + bias) v per packed sequence; see the module's text for the formula.

    q (Tq, H, D), k, v (Tk, Hkv, D), H a multiple of Hkv; views with any row and head strides are read in place when they keep 16-byte
    alignment (slices of a fused projection do). cu_q, cu_k int32 (B + 1,) on the device, non-decreasing from 0; cu_k None: cu_q.
    scale: positive, default 1 / sqrt(D). bias (buckets, H): float32 or q's type, `buckets` int32 (2 far + 1,): its map (relative_buckets).
    -> (Tq, H, D) in q's type. Differentiable in q, k, v and bias (once)."""
    if cu_k is None:
        cu_k = cu_q
    _check(q, k, v, cu_q, cu_k, bias, buckets)
    dim = q.shape[2]
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("attention_packed: the scale must be positive and finite, got %r" % scale)
    if q.device.index != torch.cuda.current_device():
        with torch.cuda.device(q.device):
            return attention_packed(q, k, v, cu_q, cu_k, causal, scale, bias, buckets)
    if dim not in _DIMS:
        _nodes.refuse_capture_of_copies("attention_packed", (q, k, v))
        more = next(d for d in _DIMS if d > dim) - dim
        q, k, v = (torch.nn.functional.pad(t, (0, more)) for t in (q, k, v))
        return attention_packed(q, k, v, cu_q, cu_k, causal, scale, bias, buckets)[..., :dim]
    nodes = _nodes.load() if BACKEND != "py" else None
    if nodes is not None:
        return nodes.attention(q, k, v, bias, cu_q, cu_k, buckets, bool(causal), scale, _lib.stream_ptr())
    leaves = (q, k, v, bias)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if bias is not None:
        bias = bias.contiguous()
    causal = 1 if causal else 0
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad)):
        if torch.cuda.is_current_stream_capturing():
            _nodes.refuse_foreign_leaves("attention_packed", leaves)
        return AttentionPackedFn.apply(q, k, v, bias, cu_q, cu_k, causal, scale, buckets)
    return _forward(q, k, v, bias, cu_q, cu_k, causal, scale, buckets, False)[0]
