"""The type's lowest and largest values are finite values: in a value, a key,
a query or the state they reach nothing but what depends on them, and what
does is the formula's (test_gpu_ops.close's tolerance)."""
import pytest
import torch

from ssla_rt_b200 import ops
from test_gpu_ops import DT, check_attention, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", [(24, 24), (64, 64), (128, 128)], ids=str)
@pytest.mark.parametrize("which", ["q", "k", "v"])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("at", [0, 40, 70])
def test_lowest_value(dtype, dims, which, sign, at):
    n, h = 100, 2
    q, k, v, d, state = inputs(401, n, h, h, h, *dims, DT[dtype], True, slots=1)
    # small enough that no product with the largest number leaves the type's range
    q, k, v, state = q * 0.03, k * 0.03, v * 0.03, state * 0.03
    t = {"q": q, "k": k, "v": v}
    t[which][at, 1, 7] = sign * torch.finfo(DT[dtype]).max
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.1)
    check_attention(q, k, v, d, [(range(n), 0)], before, 0.1, out, state)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])       # (fp16 ends far below)
@pytest.mark.parametrize("dims", [(24, 24), (128, 128)], ids=str)
def test_largest_state(dtype, dims):
    n, h = 70, 1
    q, k, v, d, state = inputs(411, n, h, h, h, *dims, DT[dtype], True, slots=1)
    q = q * 0.03                                          # the sums over dk are held in 32 bits before the scale
    state[0, 0, 3, 5] = -torch.finfo(torch.float32).max
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.1)
    check_attention(q, k, v, d, [(range(n), 0)], before, 0.1, out, state)


def test_an_infinite_state_stays_infinite():
    q, k, v, d, state = inputs(421, 70, 1, 1, 1, 128, 128, torch.bfloat16, True, slots=1)
    state[0, 0, 3, 5] = torch.inf
    out = ops.linear_attention(q, k, v, d, state=state)
    assert not torch.isfinite(out[:, 0, 5].float()).any() and torch.isfinite(out[:, 0, :5].float()).all()
    assert not torch.isfinite(state[0, 0, 3, 5])
