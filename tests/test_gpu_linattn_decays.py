"""A decay that is not a number reaches its own and later tokens, never
earlier ones: what comes before is, bit for bit, as without it."""
import math

import pytest
import torch

from ssla_rt_b200 import ops
from test_gpu_ops import DT, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", [(24, 24), (40, 24), (64, 64), (128, 128)], ids=str)
@pytest.mark.parametrize("bad", [0, 1, 2, 15, 16, 17, 63, 64, 65, 91, 139])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_decay_reaches_no_earlier_token(dtype, dims, bad, value):
    n, h = 140, 2
    q, k, v, d, state = inputs(43, n, h, h, h, *dims, DT[dtype], True, slots=1)
    clean, st = ops.linear_attention(q, k, v, d, state=state.clone()), state.clone()
    d[bad, 1] = value
    out = ops.linear_attention(q, k, v, d, state=st)
    assert torch.equal(out[:bad], clean[:bad]) and torch.equal(out[:, 0], clean[:, 0])
    assert not torch.isfinite(out[bad:, 1].float()).any()
    assert torch.isfinite(st[0, 0]).all() and not torch.isfinite(st[0, 1]).any()


@pytest.mark.parametrize("dims", [(24, 24), (128, 128)], ids=str)
@pytest.mark.parametrize("bad", [2001, 4000])
def test_in_a_divided_sequence(dims, bad):
    q, k, v, d, state = inputs(45, 5003, 1, 1, 1, *dims, torch.bfloat16, True, slots=1)
    clean = ops.linear_attention(q, k, v, d, state=state.clone())
    d[bad] = math.nan
    out = ops.linear_attention(q, k, v, d, state=state)
    assert torch.equal(out[:bad], clean[:bad])
    assert not torch.isfinite(out[bad:].float()).any() and not torch.isfinite(state).any()
