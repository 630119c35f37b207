"""Refusals and host-side parts of the text encoder's operators, without a GPU."""
import ctypes
import math

import pytest
import torch

from instancerefer_amd import attention as A
from instancerefer_amd.dense import rms_norm_residual
from instancerefer_amd.optim import FlatAdam, clip_grads_


def qkv(tq=6, tk=6, heads=4, kv=2, dim=64, dt=torch.float32):
    return torch.zeros(tq, heads, dim, dtype=dt), torch.zeros(tk, kv, dim, dtype=dt), torch.zeros(tk, kv, dim, dtype=dt)


CU = torch.tensor([0, 6], dtype=torch.int32)


def test_attention_needs_a_device():
    with pytest.raises(RuntimeError, match="HIP device"):
        A.attention_packed(*qkv(), CU)


@pytest.mark.parametrize("make,message", [
    (lambda: (qkv()[0][0], *qkv()[1:], CU), "rows, heads, dim"),
    (lambda: (*qkv(dt=torch.float64), CU), "float32, bfloat16"),
    (lambda: (qkv()[0], qkv()[1].half(), qkv()[2], CU), "share one"),
    (lambda: (qkv()[0], qkv(tk=5)[1], qkv()[2], CU), "k is"),
    (lambda: (qkv(dim=32)[0], *qkv()[1:], CU), "head dimensions"),
    (lambda: (*qkv(dim=129), CU), "head dimensions"),
    (lambda: (*qkv(heads=3), CU), "key / value heads"),
    (lambda: (*qkv(), CU.long()), "int32"),
    (lambda: (*qkv(), CU[:0]), "int32"),
    (lambda: (*qkv(), CU, torch.tensor([0, 2, 6], dtype=torch.int32)), "sequences"),
    (lambda: (*qkv(tk=7), CU), "offsets of their own"),
])
def test_attention_refuses(make, message):
    with pytest.raises(ValueError, match=message):
        A.attention_packed(*make())


def test_attention_refuses_bad_bias_and_scale():
    q, k, v = qkv()
    table, buckets = torch.zeros(8, 4), A.relative_buckets(8, 20)
    for bias, bk in ((table, None), (None, buckets), (table[:, :3], buckets), (table.half(), buckets), (table, buckets[:-1]), (table, buckets.long()),
                     (table, torch.zeros(2 * A.MAX_FAR + 3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            A.attention_packed(q, k, v, CU, bias=bias, buckets=bk)


def test_buckets():
    b = A.relative_buckets(32, 128).tolist()
    assert len(b) == 257 and b[128] == 0 and b[:128] == [x - 16 for x in b[:128:-1]]       # the two sides mirror each other
    right = b[128:]
    assert right[1:9] == [17, 18, 19, 20, 21, 22, 23, 24][:7] + [24] and max(right) == 31 and right[128] == 31
    # the borders of the growing buckets, where a logarithm in floating point rounds either way: 8 * 16^(t / 8)
    assert right[15] == 25 and right[16] == 26 and right[31] == 27 and right[32] == 28 and right[63] == 29 and right[64] == 30
    one = A.relative_buckets(32, 128, bidirectional=False).tolist()
    assert one[128:] == [0] * 129 and one[127] == 1 and one[0] == 31
    for n, far in ((16, 50), (32, 512), (6, 9)):
        m = A.relative_buckets(n, far, False).tolist()
        assert sorted(m, reverse=True) == m and set(m) == set(range(n))
    for bad in ((3, 20, True), (2, 20, True), (1, 20, False), (32, 8, True), (32, A.MAX_FAR + 1, True)):
        with pytest.raises(ValueError):
            A.relative_buckets(*bad)


def test_offsets():
    assert A.packed_offsets(torch.tensor([2, 0, 5])).tolist() == [0, 2, 2, 7]
    for bad in (torch.tensor([1.0]), torch.tensor([[1]]), torch.tensor([True])):
        with pytest.raises(ValueError):
            A.packed_offsets(bad)


def test_norm_refuses():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    with pytest.raises(RuntimeError, match="HIP device"):
        rms_norm_residual(x, x, w)
    for args in ((x, x[:2], w), (x, x.half(), w), (x, None, w[:7]), (x, None, w.half()), (x.double(), None, w), (x.long(), None, w)):
        with pytest.raises(ValueError):
            rms_norm_residual(*args)
    for eps in (-1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="eps"):
            rms_norm_residual(x, None, w, eps)


def test_clip_refuses():
    g = [torch.ones(3)]
    with pytest.raises(RuntimeError, match="HIP device"):
        clip_grads_(g, 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grads_(g, bad)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grads_(g, 1.0, 1.0)
    with pytest.raises(ValueError, match="dense"):
        clip_grads_([torch.ones(3).double()], 1.0)
    with pytest.raises(ValueError, match="dense"):
        clip_grads_([torch.ones(3).to_sparse()], 1.0)
    opt = FlatAdam([torch.nn.Parameter(torch.ones(3))])
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=-2.0)
    with pytest.raises(ValueError, match="norm_type"):
        opt.step(max_norm=2.0, norm_type=3)


def test_c_entries_refuse(lib):
    f = lib.irx_attn_packed_fwd
    one = ctypes.c_void_p(4096)

    def call(dim=64, dtype=0, heads=4, kv=2, scale=0.1, q=one, row=256, far=0, table=None, tq=8, out=one, cu=one):
        return f(q, row, 64, one, 128, 64, one, 128, 64, cu, cu, 1, tq, 8, heads, kv, dim, dtype, scale, 0, table, 1, one, 4, far, out, None, None, None, 0, None)

    for kw in (dict(dim=48), dict(dtype=3), dict(heads=3), dict(kv=0), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf), dict(q=ctypes.c_void_p(4100)),
               dict(row=257), dict(table=one, far=A.MAX_FAR + 1), dict(table=one, far=-1), dict(tq=-1), dict(out=None), dict(cu=None), dict(q=None)):
        assert call(**kw) == -1, kw
        assert b"irx_attn_packed_fwd" in lib.irx_last_error()
    assert call(tq=0) == 0
    assert lib.irx_attn_packed_fwd_workspace_bytes(16, 16, 1, 4, 4, 64, 0, 0) == 0
    need = lib.irx_attn_packed_fwd_workspace_bytes(1, 8000, 1, 4, 2, 64, 0, 0)
    assert need > 0 and need % ((64 + 2) * 4 * 4) == 0
    assert f(one, 256, 64, one, 128, 64, one, 128, 64, one, one, 1, 1, 8000, 4, 2, 64, 0, 0.1, 0, None, 1, None, 0, 0, one, None, None, None, 0, None) == -3
    assert lib.irx_attn_packed_bwd_workspace_bytes(100, 100, 2, 4, 4, 64, 0, -1) == 100 * 4 * 4
    assert lib.irx_attn_packed_bwd_workspace_bytes(100, 100, 2, 4, 4, 64, 0, 8) > 100 * 4 * 4
    assert lib.irx_attn_packed_bwd(one, 256, 64, one, 128, 64, one, 128, 64, one, 256, 64, one, None, one, one, one, 1, 8, 8, 4, 2, 64, 0, 0.1, 0, None, 1, None,
                                   0, 0, one, one, one, None, None, 0, None) == -3
    assert lib.irx_rms_norm_fwd(one, None, one, 1, 4, 0, 0, 1e-6, one, None, None, None) == -1
    assert lib.irx_rms_norm_fwd(one, None, one, 1, 4, 1 << 26, 0, 1e-6, one, None, None, None) == -1
    assert lib.irx_rms_norm_fwd(one, one, one, 1, 4, 8, 0, 1e-6, one, None, None, None) == -1
    assert lib.irx_rms_norm_fwd(None, None, None, 1, 0, 8, 0, 1e-6, None, None, None, None) == 0
    assert lib.irx_rms_norm_bwd(one, None, one, one, 1, one, 4, 8, 0, one, one, None, 0, None) == -3
    counts = (ctypes.c_ulonglong * 2)(10, 10)
    types = (ctypes.c_int * 2)(0, 1)
    same = (ctypes.c_void_p * 2)(4096, 4116)
    assert lib.irx_clip_grads(same, types, counts, 2, 0, 1.0, one, one, 1 << 20, None) == -1 and b"share memory" in lib.irx_last_error()
    apart = (ctypes.c_void_p * 2)(4096, 4136)
    assert lib.irx_clip_grads(apart, types, counts, 2, 0, 1.0, one, None, 0, None) == -3
    assert lib.irx_clip_grads(apart, types, counts, 2, 0, -1.0, one, one, 1 << 20, None) == -1
    types[1] = 3
    assert lib.irx_clip_grads(apart, types, counts, 2, 0, 1.0, one, one, 1 << 20, None) == -1
    assert lib.irx_adam_step_clip(one, one, one, one, 4, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, 1.0, one, 4, 0, 1.0, one, None) == -1
    assert lib.irx_grad_gather_parts(counts, 2) == 2 and lib.irx_grad_gather_parts(None, 0) == 0
    assert lib.irx_grad_gather_norm(apart, apart, counts, 2, 0, None, 0, None) == -3
    odd = (ctypes.c_void_p * 2)(4098, 4136)
    assert lib.irx_grad_gather_norm(odd, apart, counts, 2, 0, one, 1 << 10, None) == -1
    assert lib.irx_grad_gather_norm(None, None, None, 0, 0, None, 0, None) == 0
