"""Counts beyond the other tests': thousands of rows and states a call, and
states the size of an engine's layers.  Tolerances as in test_gpu_ops."""
import numpy as np
import pytest
import torch

from ssla_rt_b200 import ops
from test_gpu_ops import DT, check_attention, close, inputs, quantised, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
def test_step_of_thousands_of_rows(dtype):
    rows, h, dk, dv = 4096, 2, 24, 24
    q, k, v, d, state = inputs(701, rows, h, h, h, dk, dv, DT[dtype], True, slots=rows)
    slots = torch.randperm(rows, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    slots[100] = slots[4000]                              # one slot twice, one not named, two padding rows
    slots[7], slots[3000] = -1, rows
    before = state.clone()
    out = ops.linear_attention_step(q, k, v, d, state, slots=slots.cuda(), scale=0.5)
    alone = [r for r in range(rows) if r not in (7, 100, 3000, 4000)]
    at = slots[alone].long().cuda()
    new = d[alone].double().exp()[:, :, None, None] * before[at].double() + k[alone].double()[..., None] * v[alone].double()[..., None, :]
    want = 0.5 * (q[alone].double()[..., None] * new).sum(2)
    size = (d[alone].double().exp()[:, :, None, None] * before[at].double().abs() +
            k[alone].double().abs()[..., None] * v[alone].double().abs()[..., None, :])
    close(out[alone], want, 0.5 * (q[alone].double().abs()[..., None] * size).sum(2), v.dtype, 1, dk, "out")
    close(state[at], new, size, torch.float32, 1, dk, "state")
    assert (out[[7, 3000]] == 0).all()
    s = int(slots[100])
    two = [t[[100, 4000]] for t in (q, k, v, d)]
    check_attention(*two, [(range(2), 0)], before[s:s + 1], 0.5, out[[100, 4000]], state[s:s + 1])
    named = set(slots.tolist())
    rest = [i for i in range(rows) if i not in named]
    assert rest and torch.equal(state[rest], before[rest])


def test_one_slot_named_by_thousands_of_rows():
    rows, h, d = 3000, 1, 8
    q, k, v, dec, state = inputs(711, rows, h, h, h, d, d, torch.float32, True, slots=2)
    before = state.clone()
    out = ops.linear_attention_step(q, k, v, dec, state, slots=torch.zeros(rows, dtype=torch.int32, device="cuda"))
    chunked = before[:1].clone()
    want = ops.linear_attention(q, k, v, dec, state=chunked)
    # both within the tolerance of the recurrence: decays of e^-0.24 on average, 200 tokens count
    tol = 2 * (6 * 200 + d + 32) * 2.0 ** -24 * 40
    assert (out - want).abs().max() < tol and (state[0] - chunked[0]).abs().max() < tol
    assert torch.equal(state[1], before[1])


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("n,rows,cols,block", [(24, 5120, 12, 12), (12, 1280, 48, 48), (3000, 5, 24, 16), (2, 80, 96, 96)])
def test_states_like_an_engines_layers(fmt, n, rows, cols, block):
    x = rand(n + cols, n, rows, cols)
    slots = torch.randperm(n + 3, generator=torch.Generator().manual_seed(2))[:n].to(torch.int32).cuda()
    codes, scales = ops.state_cache(n + 3, rows, cols, block=block, dtype=fmt)
    ops.state_store(x, codes, scales, block=block, slots=slots)
    want_c, want_s = quantised(x, block, fmt)
    assert np.array_equal(codes.float()[slots.long()].cpu().numpy(), want_c)
    assert np.array_equal(scales[slots.long()].cpu().numpy(), want_s)
    y = ops.state_load(codes, scales, block=block, slots=slots)
    assert torch.equal(y.cpu(), torch.from_numpy(want_c.astype(np.float32) * np.repeat(want_s, block, 2)[:, :, :cols]))


def test_a_store_of_thousands_of_states_keeps_the_last_of_a_slot():
    n = 5000
    x = rand(3, n, 2, 16)
    slots = torch.arange(n, dtype=torch.int32) % 37
    codes, scales = ops.state_cache(37, 2, 16, block=16)
    ops.state_store(x, codes, scales, block=16, slots=slots.cuda())
    last = torch.tensor([max(i for i in range(n - 40, n) if i % 37 == s) for s in range(37)])
    c1, s1 = ops.state_cache(37, 2, 16, block=16)
    ops.state_store(x[last.cuda()].contiguous(), c1, s1, block=16)
    assert torch.equal(codes, c1) and torch.equal(scales, s1)


@pytest.mark.parametrize("dtype", DT)
def test_many_sequences_divided(dtype):
    """Two launch groups, each of them divided into segments."""
    lengths = [3000] + [1] * 300 + [2500]
    off = np.concatenate([[0], np.cumsum(lengths)])
    n = int(off[-1])
    q, k, v, d, state = inputs(721, n, 1, 1, 1, 24, 24, DT[dtype], True, slots=len(lengths))
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, offsets=off)
    for i in (0, 1, 150, 300, 301):
        one = before[i:i + 1].clone()
        part = slice(int(off[i]), int(off[i + 1]))
        o = ops.linear_attention(q[part], k[part], v[part], d[part], state=one)
        # the same sequence in a call of its own, divided elsewhere: twice the tolerance of either
        size = 60 * (2.0 ** -22 if dtype == "fp32" else 2.0 ** -15) + 60 * (6 * 200 + 24 + 32) * 2.0 ** -24
        assert (o.double() - out[part].double()).abs().max() <= 2 * size + 2 * torch.finfo(DT[dtype]).eps * o.double().abs().max()
        assert (one[0] - state[i]).abs().max() <= 2 * 60 * (2.0 ** -22 + (6 * 200 + 56) * 2.0 ** -24)
