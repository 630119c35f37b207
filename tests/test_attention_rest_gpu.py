"""What a 16-bit forward keeps of its output's rounding: output and rest together are the value before it was rounded, also where that lies beside
the middle of two 16-bit values."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U32 = 2.0 ** -24


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("rows,each,heads", [(40, 1, 2), (9, 100, 4), (300, 1, 100), (200, 400, 2), (1, 500, 3)])
def test_output_and_rest(kind, dim, rows, each, heads):
    """equal scores over 3 * each keys: the output is a third of three values, chosen so that it is the middle of two 16-bit values"""
    from instancerefer_amd import attention
    print("case", kind, dim, rows, each, heads, flush=True)
    step = torch.finfo(kind).eps                                         # from 1 to 2; half of it from 0.5 to 1
    g = torch.Generator().manual_seed(dim + rows)
    keys = 3 * each
    # 3 (odd) step / 2 = a + b + c: a, b in whole steps from 1 on, c an odd number of half steps below 1
    last = int(0.9 / step)
    odd = 2 * torch.randint(int(1.05 / step), int(1.2 / step), (heads, dim), generator=g) + 1                         # the middle, in half steps
    c = 2 * torch.randint(int(0.55 / step), last, (heads, dim), generator=g) + 1                                      # ... of half steps: 0.55 .. 0.9
    a = (3 * odd - c) // 4
    b = (3 * odd - c) // 2 - a
    parts = torch.stack([a * step, b * step, c * (step / 2)]).to(kind)                                               # (3, heads, dim)
    assert torch.equal(parts.double().sum(0), 3 * odd * (step / 2)) and float(parts.max()) < 2
    v = parts.repeat(each, 1, 1)
    q, k = torch.zeros(rows, heads, dim).to(kind), torch.randn(keys, heads, dim, generator=g).to(kind)
    cu, cuk = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (rows, keys))
    out, _, rest = attention._forward(q.to(DEV), k.to(DEV), v.to(DEV), None, cu, cuk, 0, 1.0, None, True)
    want = (odd * (step / 2)).double()
    # equal weights are powers of two; sums, the quotient and the product in 32 bits; the rest is rounded in its turn
    off = (out.double() + rest.double()).cpu() - want
    assert float(off.abs().max()) <= (2 * keys + 24) * U32 * 2 + step / 2 * step, float(off.abs().max()) / step
    assert float((out.double().cpu() - want).abs().max()) <= step / 2 + (2 * keys + 24) * U32 * 2
