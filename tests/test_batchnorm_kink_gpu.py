"""BatchNorm + ReLU where pre-activations lie within a rounding of zero: against 64 bits, the incoming gradient zero at those few values, whose side
of the kink 32-bit sums in another order decide either way (test_ops_gpu.test_batchnorm_act compares with torch's float32 result on the
CPU, whose side depends on its number of threads)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


@pytest.mark.parametrize("n,c", [(5000, 32), (777, 64), (260, 128), (1500, 20)])
def test_gradients_beside_the_kink(lib, n, c):
    from instancerefer_amd.sparse import nn as spnn
    torch.manual_seed(n + c)
    x = torch.randn(n, c) * 2 + 0.5
    ref = torch.nn.BatchNorm1d(c)
    ref.weight.data.uniform_(0.5, 1.5)
    ref.bias.data.uniform_(-0.5, 0.5)
    g = torch.randn(n, c)
    bn = spnn.BatchNorm(c).cuda()
    bn.load_state_dict(ref.state_dict())
    X, W, B = x.double(), ref.weight.detach().double(), ref.bias.detach().double()
    mean, rstd = X.mean(0), 1 / (X.var(0, unbiased=False) + ref.eps).sqrt()
    hat = (X - mean) * rstd
    pre = hat * W + B
    # statistics of n values in 32 bits (n + 8 half steps of the sums of magnitudes at most), then a handful of operations
    e = (n + 16) * U32
    e_pre = e * ((X.abs().mean(0) + X.abs()) * rstd * W + 2 * hat.abs() * W + B.abs())
    near = pre.abs() <= e_pre
    assert float(near.double().mean()) < 0.01                            # few: the rest is compared in full
    g[near] = 0.0
    xd = x.cuda().requires_grad_(True)
    y = bn.feats(xd, None, True)
    y.backward(g.cuda())
    G = torch.where(pre > 0, g.double(), torch.zeros_like(X))
    gm, gh = G.mean(0), (G * hat).mean(0)
    dx = W * rstd * (G - gm - hat * gh)
    big = W * rstd * (G.abs() + G.abs().mean(0) + hat.abs() * (G * hat).abs().mean(0))
    assert ((y.detach().double().cpu() - pre.clamp(min=0)).abs() <= e_pre).all()
    e_hat = e * (X.abs().mean(0) + X.abs()) * rstd                        # the normalised value itself, where the statistics are off
    off = (xd.grad.double().cpu() - dx).abs()
    assert (off <= 4 * e * big + W * rstd * (e_hat * (G * hat).abs().mean(0) + hat.abs() * (G.abs() * e_hat).mean(0))).all(), float(off.max())
    assert ((bn.bias.grad.double().cpu() - G.sum(0)).abs() <= e * G.abs().sum(0)).all()
    assert ((bn.weight.grad.double().cpu() - (G * hat).sum(0)).abs() <= (G.abs() * (e * hat.abs() * 2 + e_hat)).sum(0)).all()
