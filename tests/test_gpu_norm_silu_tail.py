"""SiLU far below zero: y * sigmoid(y) = y e^y there, an ordinary number down
to y = -91.9 (fp32, bf16) and a subnormal one below.

Tolerance.  With weights of zero y is the bias itself.  The exponential's
argument is y log2 e, rounded to 24 bits: |y| 2^-23 of the value (two
roundings of half of it each), its own error, the reciprocal and the products
2^-20 together; then one rounding to the type, of half the smallest subnormal
number where the result is below the normal ones."""
import pytest
import torch

from ssla_rt_b200 import ops
from test_gpu_ops import DT, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,p,g", [(3, 1, 4), (2, 2000, 4), (1, 60001, 1)])
def test_silu_tail(dtype, n, p, g):
    c = 96
    x = rand(1, n, p, c, dtype=DT[dtype])
    bias = torch.cat([torch.linspace(-112, -60, 64), torch.tensor([-86.9, -87.3, -87.4, -88.0, -88.8, -91.8, -1000.0, -3e38]),
                      torch.tensor([0.0, -0.5, 0.5, 60.0, 88.0, 89.0, 200.0, 3e4]), torch.linspace(-20, 20, 16)]).cuda()
    y = ops.group_norm(x, g, torch.zeros(c, device="cuda"), bias)
    z = bias.double()
    want = (z * torch.sigmoid(z)).expand_as(y)
    f = torch.finfo(DT[dtype])
    tol = (f.eps / 2 + 2.0 ** -20 + z.abs().clamp(max=200) * 2.0 ** -23) * want.abs() + f.smallest_normal * f.eps
    off = (y.double() - want).abs()
    assert (off <= tol).all(), (off / tol).amax((0, 1))
