"""A decay of -infinity clears the state before its token, whatever the state
holds: NaN and infinities in the state, the keys, the values or the decays
before a clear reach nothing from it on.

The reference is the recurrence in 64 bits with the state replaced by zero at
a clear.  Where it is finite the result is within test_gpu_ops.close's
tolerance of it, and where it is not the result is not."""
import math

import numpy as np
import pytest
import torch

from ssla_rt_b200 import ops
from test_gpu_ops import DT, inputs

pytestmark = pytest.mark.gpu
DIMS = [(24, 24), (40, 24), (64, 64), (128, 128), (128, 96), (100, 130)]


def recurrence(q, k, v, decay, state, scale, rows=None):
    q, k, v, S = q.double(), k.double(), v.double(), state.double().clone()
    decay = decay.double()
    out = torch.zeros_like(v)
    for r in rows if rows is not None else range(len(v)):
        a = decay[r][:, None, None]
        S = torch.where(a == -math.inf, 0.0, a.exp() * S) + k[r][:, :, None] * v[r][:, None, :]
        out[r] = scale * (q[r][:, :, None] * S).sum(1)
    return out, S


def agree(got, want, size, dtype, steps, dk, what):
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got.double()), finite), f"{what}: {(torch.isfinite(got.double()) != finite).sum()} places"
    split = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -15
    tol = (torch.finfo(dtype).eps / 2 * want.abs() + size * (split + (6 * steps + dk + 32) * 2.0 ** -24) +
           torch.finfo(dtype).smallest_normal)
    off = (got.double() - want).abs()[finite] / tol[finite]
    assert not off.numel() or off.max() <= 1, f"{what}: {off.max().item():.3g} of the tolerance"


def check(q, k, v, d, before, scale, out, state, steps=None):
    want, S = recurrence(q, k, v, d, before, scale)
    size, big = recurrence(q.abs(), k.abs(), v.abs(), d, before.abs(), abs(scale))
    steps = steps or len(v)
    agree(out, want, size, v.dtype, steps, q.shape[2], "out")
    agree(state, S, big, torch.float32, steps, q.shape[2], "state")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", DIMS, ids=str)
@pytest.mark.parametrize("at", [0, 1, 17, 63, 64, 77, 130])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_poisoned_state_is_cleared(dtype, dims, at, value):
    n, h = 140, 2
    q, k, v, d, state = inputs(301, n, h, h, h, *dims, DT[dtype], True, slots=2)
    state[0, 0] = value
    state[0, 1, 3, 5] = value
    d[at] = -math.inf
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.5, offsets=[0, n], slots=[0])
    check(q, k, v, d, before[0], 0.5, out, state[0])
    assert torch.isfinite(state[0]).all() and torch.isfinite(out[at:].float()).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", DIMS, ids=str)
@pytest.mark.parametrize("which", ["q", "k", "v", "decay"])
@pytest.mark.parametrize("bad,at", [(0, 1), (3, 4), (5, 40), (20, 63), (62, 63), (63, 64), (10, 70), (64, 65), (66, 100), (128, 139)])
def test_a_poisoned_token_is_cleared(dtype, dims, which, bad, at):
    n, h = 140, 2
    q, k, v, d, state = inputs(311, n, h, h, h, *dims, DT[dtype], True, slots=1)
    if which == "decay":
        d[bad, 1] = math.nan
    else:
        {"q": q, "k": k, "v": v}[which][bad, 1, [7, 20]] = torch.tensor([math.inf, math.nan], device="cuda").to(DT[dtype])
    d[at, 1] = -math.inf
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.5)
    check(q, k, v, d, before[0], 0.5, out, state[0])
    assert torch.isfinite(state).all() and torch.isfinite(out[at:].float()).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_several_clears_and_poisons(dtype, dims):
    """Packed documents, some of them with bad values before, between and behind the clears of one chunk."""
    n, h = 201, 3
    q, k, v, d, state = inputs(321, n, h, h, h, *dims, DT[dtype], True, slots=1)
    for t in (0, 9, 10, 30, 33, 64, 66, 120, 127, 128, 190, 200):
        d[t, 0] = -math.inf
    d[25::7, 1] = -math.inf
    d[:, 2] = -math.inf                                   # every token by itself
    for t, col in ((2, 1), (12, 2), (31, 3), (65, 4), (125, 5), (191, 6)):
        v[t, :, col] = math.nan
    k[20, :, 3] = math.inf
    k[100, 1, 2] = math.nan
    q[26, 0, 0] = -math.inf
    d[15, 0] = math.nan
    state[0, 0, 2, 2] = math.inf
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.5)
    check(q, k, v, d, before[0], 0.5, out, state[0])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", [(24, 24), (64, 64), (128, 128)], ids=str)
@pytest.mark.parametrize("bad,at", [(700, 1900), (1000, 1010), (2000, 2049), (4990, 5002)])
def test_in_a_divided_sequence(dtype, dims, bad, at):
    n = 5003
    q, k, v, d, state = inputs(331, n, 1, 1, 1, *dims, DT[dtype], True, slots=1)
    state[0, 0, 1] = math.nan
    v[bad, 0, 7] = math.inf
    k[bad + 1, 0, 3] = math.nan
    d[300] = d[at] = -math.inf
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.5)
    # (decays of e^-0.24 on average: what is over 200 tokens back no longer counts)
    check(q, k, v, d, before[0], 0.5, out, state[0], steps=200)
    assert torch.isfinite(state).all() and torch.isfinite(out[at:].float()).all() and torch.isfinite(out[300:bad].float()).all()


@pytest.mark.parametrize("dtype", DT)
def test_an_underflowing_decay_is_no_clear(dtype):
    """A finite decay multiplies, however small its factor: NaN stays."""
    q, k, v, d, state = inputs(341, 70, 1, 1, 1, 64, 64, DT[dtype], True, slots=1)
    state[0, 0, 0, 5] = math.nan
    d[10] = -1e4
    d[20] = torch.finfo(torch.float32).min
    ops.linear_attention(q, k, v, d, state=state)
    assert torch.isnan(state[0, 0, :, 5]).any()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dk,dv", [(24, 24), (33, 17), (128, 128)])
def test_step(dtype, dk, dv):
    rows, h = 6, 2
    q, k, v, d, state = inputs(351, rows, h, h, h, dk, dv, DT[dtype], True, slots=4)
    slots = [0, 1, 2, 1, 3, 2]
    state[0] = math.nan
    state[1, 0, 3, 5] = math.inf
    d[0] = d[1, 0] = d[5] = -math.inf
    v[2, 1, 4] = math.nan                                 # row 2 poisons slot 2, row 5 clears it
    before = state.clone()
    out = ops.linear_attention_step(q, k, v, d, state, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"), scale=0.5)
    for s in range(4):
        mine = [r for r, x in enumerate(slots) if x == s]
        want, S = recurrence(q, k, v, d, before[s], 0.5, mine)
        size, big = recurrence(q.abs(), k.abs(), v.abs(), d, before[s].abs(), 0.5, mine)
        agree(out[mine], want[mine], size[mine], v.dtype, len(mine), dk, "out")
        agree(state[s], S, big, torch.float32, len(mine), dk, "state")
    assert torch.isfinite(state).all() and torch.isfinite(out[[0, 1, 5]].float()).all()


def test_one_decay_for_each_head_can_clear_too():
    """A decay of -infinity for a whole head: every token alone."""
    n, h = 150, 2
    q, k, v, _, state = inputs(361, n, h, h, h, 128, 128, torch.bfloat16, True, slots=1)
    d = torch.tensor([-math.inf, -0.1], device="cuda")
    state[0, 0] = math.nan
    v[40, 0, 3] = math.nan
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, offsets=np.array([0, n], np.int32))
    check(q, k, v, d.expand(n, h), before[0], 1.0, out, state[0])
