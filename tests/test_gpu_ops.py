"""The recurrent-state operators on the GPU against the same formulas in 64
bits.

Tolerances.  Outputs are rounded once to their type: eps / 2 of the value.
Before that, linear attention is 32-bit arithmetic on sums whose terms add up
to M (the formula on absolute values): a token's decay, update and rounding,
and truncating 32-bit adders, cost at most six steps of 2^-24 of M each, the
products over dk and the exponentials another dk + 32; operands that pass the
tensor cores as two 16-bit pieces (outputs of 16-bit types) add 2^-15 of M,
as three (32-bit ones, and every state) 2^-22.
"""
import math

import numpy as np
import pytest
import torch

from ssla_rt_b200 import ops

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def rand(seed, *shape, dtype=torch.float32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def reference(q, k, v, decay, seqs, state, scale, absolute=False):
    """The recurrence in 64 bits; seqs: (rows, slot).  absolute: of all terms' sizes."""
    q, k, v, state = (None if t is None else t.double().abs() if absolute else t.double() for t in (q, k, v, state))
    n, h, dv = v.shape
    q, k = (t.repeat_interleave(h // t.shape[1], 1) for t in (q, k))
    a = decay.double().expand(n, h).exp()
    out = torch.zeros_like(v)
    new = None if state is None else state.clone()
    for rows, slot in seqs:
        S = torch.zeros(h, q.shape[2], dv, dtype=torch.float64, device=v.device) if slot < 0 else new[slot].clone()
        for r in rows:
            S = a[r][:, None, None] * S + k[r][:, :, None] * v[r][:, None, :]
            out[r] = scale * torch.einsum("hk,hkv->hv", q[r], S)
        if slot >= 0:
            new[slot] = S
    return out, new


def close(got, want, size, dtype, steps, dk, what):
    split = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -15
    tol = (torch.finfo(dtype).eps / 2 * want.abs() + size * (split + (6 * steps + dk + 32) * 2.0 ** -24) +
           torch.finfo(dtype).smallest_normal)
    off = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), what
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


def check_attention(q, k, v, decay, seqs, state0, scale, out, state, rows=None):
    want, new = reference(q, k, v, decay, seqs, state0, scale)
    size, big = reference(q, k, v, decay, seqs, state0, abs(scale), absolute=True)
    steps = max([len(r) for r, _ in seqs] + [1])
    rows = sorted(r for rr, _ in seqs for r in rr) if rows is None else rows
    close(out[rows], want[rows], size[rows], v.dtype, steps, q.shape[2], "out")
    if state is not None:
        close(state, new, big, torch.float32, steps, q.shape[2], "state")


def inputs(seed, n, h, hq, hk, dk, dv, dtype, gated, slots=0):
    q, k = rand(seed, n, hq, dk, dtype=dtype, std=dk ** -0.25), rand(seed + 1, n, hk, dk, dtype=dtype, std=dk ** -0.25)
    v = rand(seed + 2, n, h, dv, dtype=dtype)
    d = -rand(seed + 3, n, h).abs() * 0.3 if gated else -rand(seed + 3, h).abs() * 0.1
    return q, k, v, d, (rand(seed + 4, slots, h, dk, dv) if slots else None)


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 1, 8, 8), (4, 4, 4, 24, 24), (2, 1, 2, 33, 17), (3, 3, 1, 64, 96), (2, 2, 2, 128, 128),
          (1, 1, 1, 128, 256), (2, 2, 2, 12, 12), (2, 2, 2, 96, 40), (2, 1, 1, 100, 130), (2, 2, 2, 64, 64), (1, 1, 1, 16, 200)]
LENGTHS = [[1], [0, 1, 63, 64, 65, 0, 130], [257, 3]]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_linear_attention(dtype, shape, lengths):
    h, hq, hk, dk, dv = shape
    n, gated = sum(lengths), (dk + dv) % 3 != 0
    q, k, v, d, state = inputs(7, n, h, hq, hk, dk, dv, DT[dtype], gated, slots=len(lengths) + 1)
    off = np.concatenate([[0], np.cumsum(lengths)])
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, offsets=off, scale=dk ** -0.5)
    seqs = [(list(range(off[i], off[i + 1])), i) for i in range(len(lengths))]
    check_attention(q, k, v, d, seqs, before, dk ** -0.5, out, state)
    assert torch.equal(state[-1], before[-1])
    for i, n in enumerate(lengths):
        if n == 0:
            assert torch.equal(state[i], before[i])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", [(24, 24), (64, 64), (128, 128), (40, 72)], ids=str)
def test_linear_attention_long(dtype, dims):
    """Long enough that one sequence is divided among CTAs."""
    n = 5003
    q, k, v, d, state = inputs(17, n, 2, 2, 2, *dims, DT[dtype], True, slots=1)
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.5)
    # decays of e^-0.24 on average: what is over 2000 tokens back is below 2^-500
    close_steps = 200
    want, new = reference(q, k, v, d, [(range(n), 0)], before, 0.5)
    size, big = reference(q, k, v, d, [(range(n), 0)], before, 0.5, absolute=True)
    close(out, want, size, v.dtype, close_steps, dims[0], "out")
    close(state, new, big, torch.float32, close_steps, dims[0], "state")
    # the same call again gives the same bits
    again = before.clone()
    assert torch.equal(ops.linear_attention(q, k, v, d, state=again, scale=0.5), out)
    assert torch.equal(again, state)


@pytest.mark.parametrize("dtype", DT)
def test_linear_attention_without_state(dtype):
    q, k, v, d, _ = inputs(27, 90, 2, 2, 2, 24, 40, DT[dtype], True)
    out = ops.linear_attention(q, k, v, d)
    check_attention(q, k, v, d, [(list(range(90)), -1)], None, 1.0, out, None)
    state = rand(1, 3, 2, 24, 40)
    before = state.clone()
    out2 = ops.linear_attention(q, k, v, d, state=state, offsets=[0, 50, 90], slots=[-1, 2])
    check_attention(q, k, v, d, [(list(range(50)), -1), (list(range(50, 90)), 2)], before, 1.0, out2, state)


@pytest.mark.parametrize("dtype", DT)
def test_linear_attention_strides_and_padding(dtype):
    """A padded batch out of one interleaved buffer, into a strided out: what
    lies outside the sequences is neither read nor written."""
    b, t, h, dk, dv = 3, 70, 2, 20, 36
    buf = rand(3, b * t, h, 2 * dk + dv + 3, dtype=DT[dtype])
    q, k, v = buf[:, :, :dk], buf[:, :, dk:2 * dk], buf[:, :, 2 * dk:2 * dk + dv]
    d = (-rand(4, h, b * t).abs()).t()
    lengths, offsets = [70, 0, 33], [0, 70, 140]
    for i, n in enumerate(lengths):
        buf[offsets[i] + n:offsets[i] + 70] = math.nan
        d[offsets[i] + n:offsets[i] + 70] = math.nan
    state = rand(5, 4, h, dk, dv)
    before = state.clone()
    whole = torch.full((b * t + 2, dv + 5, h), 7.0, dtype=DT[dtype], device="cuda")
    out = whole.transpose(1, 2)[1:-1, :, :dv]
    with pytest.raises(ValueError):
        ops.linear_attention(q, k, v, d, state=state, offsets=offsets, lengths=lengths, out=out)
    whole = torch.full((b * t + 2, h, dv + 5), 7.0, dtype=DT[dtype], device="cuda")
    out = whole[1:-1, :, 2:2 + dv]
    assert ops.linear_attention(q, k, v, d, state=state, offsets=offsets, lengths=lengths, slots=[3, 1, 0], out=out) is out
    rows = [r for i, n in enumerate(lengths) for r in range(offsets[i], offsets[i] + n)]
    seqs = [(list(range(offsets[i], offsets[i] + n)), s) for i, (n, s) in enumerate(zip(lengths, [3, 1, 0]))]
    ok = torch.zeros(b * t, dtype=torch.bool, device="cuda")
    ok[rows] = True
    clean = [torch.where(ok[:, None, None], x, 0) for x in (q, k, v)]
    check_attention(*clean, torch.where(ok[:, None], d, 0), seqs, before, 1.0, out, state, rows)
    mask = torch.ones_like(whole, dtype=torch.bool)
    mask[1:-1, :, 2:2 + dv] = ~ok[:, None, None]
    assert (whole[mask] == 7.0).all()
    assert torch.equal(state[1:3], before[1:3])
    new = ops.linear_attention(q, k, v, d, offsets=offsets, lengths=lengths)
    assert (new[~ok] == 0).all() and torch.isfinite(new).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dk,dv", [(100, 130), (50, 35), (71, 127), (33, 250)])
def test_linear_attention_odd_widths_in_aligned_rows(dtype, dk, dv):
    n, h = 150, 2
    wide = lambda seed, w, std: rand(seed, n, h, -(-w // 8) * 8, dtype=DT[dtype], std=std)[:, :, :w]  # noqa: E731
    q, k, v = wide(1, dk, dk ** -0.25), wide(2, dk, dk ** -0.25), wide(3, dv, 1.0)
    d, state = -rand(4, n, h).abs() * 0.3, rand(5, 2, h, dk, dv)
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, offsets=[0, 67, 150], scale=0.2)
    check_attention(q, k, v, d, [(range(67), 0), (range(67, 150), 1)], before, 0.2, out, state)


@pytest.mark.parametrize("dtype", DT)
def test_linear_attention_heads_outermost(dtype):
    """(heads, rows, width) memory, expanded queries, and a decay for each head given with a stride of 0."""
    h, n, dk, dv = 3, 100, 24, 24
    q = rand(1, 1, n, dk, dtype=DT[dtype]).expand(h, n, dk).transpose(0, 1)
    k, v = rand(2, h, n, dk, dtype=DT[dtype]).transpose(0, 1), rand(3, h, n, dv, dtype=DT[dtype]).transpose(0, 1)
    d = -rand(4, h).abs()
    out = torch.empty(h, n, dv, dtype=DT[dtype], device="cuda").transpose(0, 1)
    ops.linear_attention(q, k, v, d.expand(n, h), out=out)
    check_attention(q, k, v, d, [(list(range(n)), -1)], None, 1.0, out, None)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", [(24, 24), (128, 64)], ids=str)
def test_decay_extremes(dtype, dims):
    """No decay at all; -inf clears the state; the type's lowest value and -1e4 do the same in effect."""
    n, h = 150, 2
    q, k, v, d, state = inputs(31, n, h, h, h, *dims, DT[dtype], True, slots=1)
    d[:40] = 0.0
    d[40, 0] = -math.inf
    d[77, 1] = torch.finfo(torch.float32).min
    d[100] = -1e4
    d[64:66, 0] = -math.inf
    d[128, 1] = -math.inf
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.25)
    check_attention(q, k, v, d, [(list(range(n)), 0)], before, 0.25, out, state)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("which", ["q", "k", "v", "decay", "state"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_non_finite_reaches_no_earlier_token(dtype, which, value):
    if which == "decay" and value != math.nan and not math.isnan(value):
        pytest.skip("an infinite decay has a meaning of its own")
    n, h, dk, dv, bad = 140, 2, 40, 24, 90
    q, k, v, d, state = inputs(41, n + 30, h, h, h, dk, dv, DT[dtype], True, slots=2)
    t = {"q": q, "k": k, "v": v, "decay": d}
    before = state.clone()
    if which == "state":
        before[0, 1, 3, 5] = value
    else:
        t[which][(bad, 1) if which == "decay" else (bad, 1, 7)] = value
    state = before.clone()
    out = ops.linear_attention(q, k, v, d, state=state, offsets=[0, n, n + 30])
    # the other head, the other sequence and the tokens before are as without it
    def checked(rows_sel, heads, seqs, st=None, stout=None):
        c = [torch.nan_to_num(x[:, heads].float(), nan=0, posinf=0, neginf=0).to(x.dtype) for x in (q, k, v)]
        dd = torch.nan_to_num(d[:, heads])
        check_attention(*c, dd, seqs, None if st is None else st[:, heads], 1.0, out[:, heads], None, rows_sel)
    checked(list(range(n)), [0], [(range(n), 0)], before)
    checked(list(range(n, n + 30)), [0, 1], [(range(n, n + 30), 1)], torch.nan_to_num(before))
    finite = torch.isfinite(out[:n, 1].float())
    if which == "state":
        assert not finite[0, 5] and finite[:, [c for c in range(dv) if c != 5]].all()
        assert not torch.isfinite(state[0, 1, :, 5]).all()
        return
    checked(list(range(bad)), [1], [(range(bad), 0)], before)
    if which == "q":
        assert not finite[bad].any() and finite[bad + 1:].all() and torch.isfinite(state[0]).all()
    elif which == "v":
        assert not finite[bad:, 7].any() and finite[:, [c for c in range(dv) if c != 7]].all()
        assert not torch.isfinite(state[0, 1, :, 7]).any()
        assert torch.isfinite(state[0, 1, :, [c for c in range(dv) if c != 7]]).all()
    else:
        assert not finite[bad:].any()
        assert not torch.isfinite(state[0, 1]).all()
    assert torch.isfinite(state[0, 0]).all() and torch.isfinite(state[1]).all()


@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (64, 96), (96, 200)], ids=str)
@pytest.mark.parametrize("bad", [0, 5, 63, 64, 100, 199])
@pytest.mark.parametrize("which", ["q", "k", "v"])
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_non_finite_with_wide_heads(dims, bad, which, value):
    """The same on the tensor memory path: in whole chunks and in the last, partial one."""
    n, h, (dk, dv) = 201, 2, dims
    q, k, v, d, state = inputs(141, n, h, h, h, dk, dv, torch.bfloat16, True, slots=1)
    t = {"q": q, "k": k, "v": v}
    before = state.clone()
    out_clean = ops.linear_attention(q, k, v, d, state=state.clone(), scale=0.5)
    col = 7 if which != "v" else dv - 3
    t[which][bad, 1, col] = value
    out = ops.linear_attention(q, k, v, d, state=state, scale=0.5)
    seqs = [(range(n), 0)]
    clean = [torch.nan_to_num(x, nan=0, posinf=0, neginf=0) for x in (q, k, v)]
    check_attention(*[x[:, :1] for x in clean], d[:, :1], seqs, before[:, :1], 0.5, out[:, :1], None)
    if bad:
        check_attention(*[x[:, 1:] for x in clean], d[:, 1:], [(range(bad), 0)], before[:, 1:], 0.5, out[:, 1:], None, list(range(bad)))
    finite = torch.isfinite(out[:, 1].float())
    rest = [c for c in range(dv) if c != col]
    if which == "q":
        assert not finite[bad].any() and finite[bad + 1:].all() and torch.isfinite(state).all()
        check_attention(*[x[:, 1:] for x in clean], d[:, 1:], seqs, before[:, 1:], 0.5, out[:, 1:], None,
                        [r for r in range(n) if r != bad])
    elif which == "v":
        assert not finite[bad:, col].any() and finite[:, rest].all()
        assert not torch.isfinite(state[0, 1, :, col]).any() and torch.isfinite(state[0, 1][:, rest]).all()
        assert torch.equal(out[:, 1][:, rest], out_clean[:, 1][:, rest])
    else:
        assert not finite[bad:].any() and not torch.isfinite(state[0, 1]).all()
    assert torch.isfinite(state[0, 0]).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dims", [(64, 64), (128, 128)], ids=str)
def test_linear_attention_broadcast_inputs_and_unaligned_outputs(dtype, dims):
    """Queries shared by all heads, keys by all rows, values by both (strides of 0); outputs off 16-byte places."""
    h, n, (dk, dv) = 3, 200, dims
    q = rand(1, n, 1, dk, dtype=DT[dtype], std=dk ** -0.25).expand(n, h, dk)
    k = rand(2, 1, h, dk, dtype=DT[dtype], std=dk ** -0.25).expand(n, h, dk)
    v = rand(3, 1, 1, dv, dtype=DT[dtype]).expand(n, h, dv)
    d = -rand(4, n, h).abs() * 0.3
    whole = torch.full((n, h, dv + 3), 7.0, dtype=DT[dtype], device="cuda")
    out = whole[:, :, 1:1 + dv]
    ops.linear_attention(q, k, v, d, offsets=[0, 130, n], out=out)
    check_attention(q, k, v, d, [(range(130), -1), (range(130, n), -1)], None, 1.0, out, None)
    assert (whole[:, :, 0] == 7).all() and (whole[:, :, 1 + dv:] == 7).all()


def test_wide_heads_on_two_streams_and_threads():
    """Two calls at once, each from a thread and on a stream of its own, against the same calls alone."""
    import threading
    sets = [inputs(151 + i, 3000, 8, 8, 8, 128, 128, torch.bfloat16, True, slots=1) for i in range(2)]
    alone = []
    for q, k, v, d, state in sets:
        st = state.clone()
        alone.append((ops.linear_attention(q, k, v, d, state=st), st))
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        q, k, v, d, state = sets[i]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                st = state.clone()
                got[i] = (ops.linear_attention(q, k, v, d, state=st), st)
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    for (o, s), (wo, ws) in zip(got, alone):
        assert torch.equal(o, wo) and torch.equal(s, ws)


def test_linear_attention_empty():
    q, k, v, d, state = inputs(1, 0, 2, 2, 2, 8, 8, torch.bfloat16, True, slots=2)
    before = state.clone()
    assert ops.linear_attention(q, k, v, d, state=state).shape == (0, 2, 8)
    assert ops.linear_attention(q, k, v, d, state=state, offsets=[0]).shape == (0, 2, 8)
    assert ops.linear_attention_step(q, k, v, d, state, slots=torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 2, 8)
    q, k, v, d, _ = inputs(1, 5, 2, 2, 2, 8, 8, torch.bfloat16, True)
    assert (ops.linear_attention(q, k, v, d, state=state, offsets=[2, 2, 2]) == 0).all()
    assert torch.equal(state, before)


def test_many_sequences():
    """More sequences than one launch's table holds."""
    lengths = [(i * 7) % 4 for i in range(1100)]
    off = np.concatenate([[0], np.cumsum(lengths)])
    n = int(off[-1])
    q, k, v, d, state = inputs(51, n, 1, 1, 1, 8, 8, torch.float32, True, slots=1100)
    slots = np.arange(1100)[::-1].copy()
    before = state.clone()
    out = ops.linear_attention(q, k, v, d, state=state, offsets=off, slots=slots)
    cpu = [t.cpu() for t in (q, k, v, d, before)]
    seqs = [(range(off[i], off[i + 1]), int(slots[i])) for i in range(1100)]
    check_attention(*cpu[:4], seqs, cpu[4], 1.0, out.cpu(), state.cpu())


# ---- one token per row ------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("rows", [1, 5, 130])
def test_step(dtype, shape, rows):
    h, hq, hk, dk, dv = shape
    q, k, v, d, state = inputs(61, rows, h, hq, hk, dk, dv, DT[dtype], (dk + dv) % 3 != 0, slots=rows + 3)
    slots = torch.randperm(rows + 3, generator=torch.Generator().manual_seed(rows))[:rows].to(torch.int32)
    before = state.clone()
    out = ops.linear_attention_step(q, k, v, d, state, slots=slots.cuda(), scale=0.3)
    check_attention(q, k, v, d, [([r], int(s)) for r, s in enumerate(slots)], before, 0.3, out, state)
    state = before.clone()
    out = ops.linear_attention_step(q, k, v, d, state, scale=0.3)
    check_attention(q, k, v, d, [([r], r) for r in range(rows)], before, 0.3, out, state)


@pytest.mark.parametrize("dtype", DT)
def test_step_padding_and_repeated_slots(dtype):
    slots = [4, -1, 2, 4, 9, 4, 2, -7, 1000000]
    q, k, v, d, state = inputs(71, len(slots), 2, 2, 1, 24, 40, DT[dtype], True, slots=6)
    before = state.clone()
    out = ops.linear_attention_step(q, k, v, d, state, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    pads = [r for r, s in enumerate(slots) if not 0 <= s < 6]
    seqs = [([r for r, x in enumerate(slots) if x == s], s) for s in (4, 2)]
    check_attention(q, k, v, d, seqs, before, 1.0, out, state)
    assert (out[pads] == 0).all()
    assert torch.equal(state[[0, 1, 3, 5]], before[[0, 1, 3, 5]])


def test_step_padding_rows_are_not_read():
    q, k, v, d, state = inputs(73, 4, 2, 2, 2, 24, 40, torch.bfloat16, True, slots=3)
    for t in (q, k, v, d):
        t[2] = math.nan
    out = ops.linear_attention_step(q, k, v, d, state, slots=torch.tensor([0, 1, -1, 2], dtype=torch.int32, device="cuda"))
    assert torch.isfinite(out.float()).all() and torch.isfinite(state).all() and (out[2] == 0).all()


@pytest.mark.parametrize("dtype", DT)
def test_step_strides(dtype):
    rows, h, dk, dv = 9, 3, 20, 33
    buf = rand(3, rows, h, 2 * dk + dv + 1, dtype=DT[dtype])
    q, k, v = buf[:, :, 1:1 + dk], buf[:, :, dk:2 * dk], buf[:, :, 2 * dk + 1:]
    d = (-rand(4, h, rows).abs()).t()
    state = rand(5, rows, h, dk, dv)
    before = state.clone()
    whole = torch.full((rows, h, dv + 2), 7.0, dtype=DT[dtype], device="cuda")
    out = whole[:, :, 1:-1]
    ops.linear_attention_step(q, k, v, d, state, out=out)
    check_attention(q, k, v, d, [([r], r) for r in range(rows)], before, 1.0, out, state)
    assert (whole[:, :, 0] == 7).all() and (whole[:, :, -1] == 7).all()


def test_state_pool_past_32_bits():
    """Slots whose states lie more than 2^31 values into the pool."""
    h, d = 16, 128
    n_slots = 2 ** 31 // (h * d * d) + 3
    state = torch.empty(n_slots, h, d, d, device="cuda")
    q, k, v, dec, _ = inputs(81, 3, h, h, h, d, d, torch.bfloat16, True)
    slots = [n_slots - 1, 0, n_slots - 2]
    for s in slots:
        state[s] = rand(s, h, d, d)
    keep = {s: state[s].clone() for s in slots}
    out = ops.linear_attention_step(q, k, v, dec, state, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    small = torch.stack([keep[s] for s in slots])
    check_attention(q, k, v, dec, [([r], r) for r in range(3)], small, 1.0, out, torch.stack([state[s] for s in slots]))
    for s in slots:
        state[s] = keep[s]
    out = ops.linear_attention(q, k, v, dec, state=state, offsets=[0, 1, 2, 3], slots=slots)
    check_attention(q, k, v, dec, [([r], r) for r in range(3)], small, 1.0, out, torch.stack([state[s] for s in slots]))


def test_rows_past_32_bits():
    """Rows whose first element lies more than 2^31 values into the tensor."""
    h, d, row = 2, 64, 1 << 30
    buf = torch.empty(3 * row, dtype=torch.bfloat16, device="cuda")
    v = buf.as_strided((3, h, d), (row, d, 1))
    v.copy_(rand(1, 3, h, d, dtype=torch.bfloat16))
    q, k, _, dec, state = inputs(83, 3, h, h, h, d, d, torch.bfloat16, True, slots=3)
    before = state.clone()
    out = ops.linear_attention(q, k, v, dec, state=state)
    check_attention(q, k, v, dec, [(range(3), 0)], before, 1.0, out, state)


# ---- the 8-bit cache --------------------------------------------------------------------


def quantised(x, block, fmt):
    """(codes as values, scales) by the definition, in numpy, one block at a time."""
    x = x.float().cpu().numpy()
    codes, scales = np.zeros(x.shape), np.zeros(x.shape[:2] + (-(-x.shape[2] // block),), np.float32)
    most = 127 if fmt == torch.int8 else 448
    for b, lo in enumerate(range(0, x.shape[2], block)):
        part = x[:, :, lo:lo + block]
        with np.errstate(all="ignore"):
            s = (np.abs(part).max(2).astype(np.float64) / most).astype(np.float32)
            s = np.where(np.isinf(s * np.float32(most)), np.nextafter(s, np.float32(0)), s)
            s[~np.isfinite(part).all(2)] = np.nan
            qt = np.where(s[:, :, None] > 0, (part.astype(np.float64) / s[:, :, None].astype(np.float64)).astype(np.float32), 0)
        if fmt == torch.int8:
            c = np.clip(np.rint(qt), -127, 127)
        else:
            size = np.abs(qt.astype(np.float64))
            step = 2.0 ** (np.floor(np.log2(np.maximum(size, 2.0 ** -6))) - 3)
            c = np.clip(np.rint(qt / step) * step, -448, 448)
        codes[:, :, lo:lo + block], scales[:, :, b] = c, s
    return codes, scales


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,cols,block", [(1, 1, 1), (3, 12, 12), (5, 24, 64), (7, 99, 32), (40, 128, 64), (9, 200, 128),
                                             (6, 130, 64), (4, 256, 256), (3, 250, 256), (11, 96, 8), (2, 17, 5)])
def test_state_cache(fmt, dtype, rows, cols, block):
    """Codes, scales and the values read back are the definition's, bit for bit."""
    n, slots = 5, torch.tensor([6, 0, 3, 7, 2], dtype=torch.int32, device="cuda")
    x = rand(cols, n, rows, cols, dtype=DT[dtype])
    x *= torch.exp2(torch.randint(-6, 6, (n, rows, 1), device="cuda")).to(x.dtype)
    x[0, 0] = 0.0
    codes, scales = ops.state_cache(8, rows, cols, block=block, dtype=fmt)
    codes.view(torch.int8).fill_(33)
    scales.fill_(2.0)
    ops.state_store(x, codes, scales, block=block, slots=slots)
    want_c, want_s = quantised(x, block, fmt)
    assert np.array_equal(codes.float()[slots.long()].cpu().numpy(), want_c)
    assert np.array_equal(scales[slots.long()].cpu().numpy(), want_s)
    rest = [1, 4, 5]
    assert (codes.view(torch.int8)[rest] == 33).all() and (scales[rest] == 2.0).all()
    for back in DT.values():
        y = ops.state_load(codes, scales, block=block, slots=slots, dtype=back)
        spread = np.repeat(want_s, block, 2)[:, :, :cols]
        want = torch.from_numpy(want_c.astype(np.float32) * spread).to(back)
        assert torch.equal(y.cpu(), want)
    whole = ops.state_load(codes, scales, block=block)
    assert torch.equal(whole[slots.long()], ops.state_load(codes, scales, block=block, slots=slots))


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn], ids=str)
def test_state_cache_edges(fmt):
    """Ties, quotients next to a border, tiny and huge blocks, non-finite values."""
    most = 127.0 if fmt == torch.int8 else 448.0
    rows, cols, block = 64, 64, 32
    x = rand(5, 2, rows, cols) * 3
    for r in range(16):       # multiples of half a step, and their neighbours, for scales that are not powers of two
        s = torch.tensor(0.37 + 0.11 * r)
        steps = torch.arange(0, 32) * (most / 64) + 0.5
        line = (steps * s).cuda()
        x[0, r, :32] = torch.nextafter(line, torch.tensor(9e9 if r % 3 == 0 else -9e9 if r % 3 == 1 else 0.0).cuda())
        x[0, r, 31] = most * s
    x[0, 20] *= 1e-30
    x[0, 21] *= 1e-38
    x[0, 22] *= 1e-44
    x[0, 23] *= 1e37
    x[0, 24] = torch.finfo(torch.float32).max
    x[0, 25] = torch.finfo(torch.float32).tiny
    x[1, 3, 5] = math.nan
    x[1, 4, 40] = math.inf
    x[1, 5, 0] = -math.inf
    codes, scales = ops.state_cache(2, rows, cols, block=block, dtype=fmt)
    ops.state_store(x, codes, scales, block=block)
    want_c, want_s = quantised(x, block, fmt)
    want_c[1, 3, :32] = want_c[1, 4, 32:] = want_c[1, 5, :32] = 0
    assert np.array_equal(scales.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(codes.float().cpu().numpy(), want_c)
    back = ops.state_load(codes, scales, block=block)
    assert torch.isnan(back[1, 3, :32]).all() and torch.isnan(back[1, 4, 32:]).all() and torch.isnan(back[1, 5, :32]).all()
    assert torch.isfinite(back[0]).all() and torch.isfinite(back[1, 3, 32:]).all() and torch.isfinite(back[1, 4, :32]).all()


def test_state_cache_slots():
    """A slot named twice keeps the last state; slots outside are skipped, and read as zeros."""
    x = rand(7, 5, 6, 40)
    codes, scales = ops.state_cache(3, 6, 40, block=16)
    s = torch.tensor([1, -1, 1, 5, 0], dtype=torch.int32, device="cuda")
    ops.state_store(x, codes, scales, block=16, slots=s)
    c1, s1 = ops.state_cache(3, 6, 40, block=16)
    ops.state_store(x[[4, 2]].contiguous(), c1, s1, block=16)
    assert torch.equal(codes, c1) and torch.equal(scales, s1)
    y = ops.state_load(codes, scales, block=16, slots=s, out=torch.full((5, 6, 40), 9.0, device="cuda"))
    assert (y[[1, 3]] == 0).all() and torch.equal(y[0], y[2]) and (y[0] != 0).any()


def test_state_cache_strides():
    big = rand(8, 4, 9, 50, dtype=torch.bfloat16)
    x = big[::2, 1:8, 3:43]
    codes, scales = ops.state_cache(2, 7, 40, block=16)
    c1, s1 = ops.state_cache(2, 7, 40, block=16)
    ops.state_store(x, codes, scales, block=16)
    ops.state_store(x.contiguous(), c1, s1, block=16)
    assert torch.equal(codes, c1) and torch.equal(scales, s1)
    dst = torch.full_like(big, 7.0)
    ops.state_load(codes, scales, block=16, out=dst[::2, 1:8, 3:43])
    assert torch.equal(dst[::2, 1:8, 3:43], ops.state_load(codes, scales, block=16, dtype=torch.bfloat16))
    dst[::2, 1:8, 3:43] = 7.0
    assert (dst == 7.0).all()


def test_state_cache_past_32_bits():
    rows, cols = 1 << 16, 128
    n = 2 ** 31 // (rows * cols) + 2
    codes = torch.empty(n, rows, cols, dtype=torch.int8, device="cuda")
    scales = torch.empty(n, rows, 2, device="cuda")
    x = rand(9, 2, rows, cols)
    s = torch.tensor([n - 1, 0], dtype=torch.int32, device="cuda")
    ops.state_store(x, codes, scales, slots=s)
    c1, s1 = ops.state_cache(2, rows, cols)
    ops.state_store(x, c1, s1)
    assert torch.equal(codes[n - 1], c1[0]) and torch.equal(codes[0], c1[1]) and torch.equal(scales[n - 1], s1[0])
    assert torch.equal(ops.state_load(codes, scales, slots=s), ops.state_load(c1, s1))


# ---- group norm -------------------------------------------------------------------------


def norm_reference(x, groups, w, b, eps, act):
    x = x.double()
    n, p, c = x.shape
    g = x.reshape(n, p, groups, c // groups)
    m = g.mean((1, 3), keepdim=True)
    var = (g - m).square().mean((1, 3), keepdim=True)
    hat = ((g - m) / (var + eps).sqrt()).reshape(n, p, c)
    y = hat * (1 if w is None else w.double()) + (0 if b is None else b.double())
    scale = (m.abs() / (var + eps).sqrt()).expand_as(g).reshape(n, p, c)
    return (y * torch.sigmoid(y) if act == "silu" else y), hat.abs(), scale


def check_norm(x, groups, w, b, act, got, eps=1e-5):
    """Per-thread 32-bit sums of up to 128 terms (2^-17 of the spread for the mean and the deviation alike), the
    mean rounded to 32 bits, the output rounded once; the activation's slope is below 1.1 and its fast exponential
    and quotient (16-bit outputs only) add 2^-18 of the value."""
    want, hat, mean = norm_reference(x, groups, w, b, eps, act)
    wa = 1.0 if w is None else w.double().abs()
    tol = (torch.finfo(x.dtype).eps / 2 * want.abs() + 1.1 * wa * (2.0 ** -16 * (hat + 1) + 2.0 ** -22 * mean) +
           2.0 ** -18 * want.abs() + torch.finfo(x.dtype).smallest_normal)
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max()


NORMS = [(1, 1, 1, 1), (5, 1, 2048, 16), (700, 1, 96, 4), (3, 47, 120, 2), (2, 300, 96, 8), (4, 5120, 24, 3), (1, 20000, 12, 1),
         (2, 9, 33, 11), (2, 1, 4098, 2), (3, 1000, 7, 7), (1, 33, 5000, 1), (65, 64, 99, 9), (2, 2500, 130, 1), (1, 70, 10240, 5)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,p,c,g", NORMS)
@pytest.mark.parametrize("act", ["silu", "none"])
def test_group_norm(dtype, n, p, c, g, act):
    x = (rand(n + c, n, p, c) * 1.5 + 0.3).to(DT[dtype])
    w, b = 1 + 0.2 * rand(2, c), 0.1 * rand(3, c)
    check_norm(x, g, w, b, act, ops.group_norm(x, g, w, b, activation=act))
    check_norm(x, g, None, None, act, ops.group_norm(x, g, activation=act))


@pytest.mark.parametrize("p,c,g", [(1, 3, 1), (1, 8196, 1), (4100, 2, 1)])
def test_group_norm_more_samples_than_a_grid_is_deep(p, c, g):
    n = 65535 + 70
    x = rand(p, n, p, c)
    y = ops.group_norm(x, g, activation="none")
    for part in (slice(0, 40), slice(65500, None)):
        check_norm(x[part], g, None, None, "none", y[part])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,p,c,g", [(3, 1, 96, 4), (2, 300, 96, 8), (2, 5120, 24, 3)])
def test_group_norm_large_mean(dtype, n, p, c, g):
    x = (rand(1, n, p, c) + 500.0).to(DT[dtype])
    check_norm(x, g, None, None, "none", ops.group_norm(x, g, activation="none"))
    flat = torch.full_like(x, 3.0)
    assert (ops.group_norm(flat, g, activation="none") == 0).all()


@pytest.mark.parametrize("n,p,c,g", [(3, 1, 96, 4), (3, 2000, 96, 8)])
def test_group_norm_in_place_and_strided(n, p, c, g):
    x = rand(1, n, p, c, dtype=torch.bfloat16)
    want = ops.group_norm(x, g)
    y = x.clone()
    assert ops.group_norm(y, g, out=y) is y and torch.equal(y, want)
    wide = torch.full((n, p, c + 6), 7.0, dtype=x.dtype, device="cuda")
    wide[:, :, 3:-3] = x
    out = torch.full((p, n, c + 2), 7.0, dtype=x.dtype, device="cuda")
    ops.group_norm(wide[:, :, 3:-3], g, out=out.transpose(0, 1)[:, :, 1:-1])
    assert torch.allclose(out.transpose(0, 1)[:, :, 1:-1].float(), want.float(), rtol=2.0 ** -7, atol=1e-3)
    assert (out[:, :, 0] == 7).all() and (out[:, :, -1] == 7).all()


@pytest.mark.parametrize("n,p,c,g", [(3, 1, 96, 4), (3, 2000, 96, 8)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_group_norm_non_finite_stays_in_its_slab(n, p, c, g, value):
    x = rand(1, n, p, c)
    clean = ops.group_norm(x, g, activation="none")
    x[1, p - 1, 13] = value
    y = ops.group_norm(x, g, activation="none")
    w = c // g
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[1, :, 13 // w * w:(13 // w + 1) * w] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


def test_group_norm_empty_and_rows():
    assert ops.group_norm(torch.empty(0, 5, 8, device="cuda"), 2).shape == (0, 5, 8)
    assert ops.group_norm(torch.empty(3, 0, 8, device="cuda"), 2).shape == (3, 0, 8)
    x = rand(1, 37, 64)
    assert torch.equal(ops.group_norm(x, 4), ops.group_norm(x[:, None], 4)[:, 0])
    out = torch.empty_like(x)
    assert ops.group_norm(x, 4, out=out) is out


# ---- together, and how they are called --------------------------------------------------


@pytest.mark.parametrize("dtype", DT)
def test_streams_prompted_parked_resumed_and_stepped(dtype):
    """Prompts, the states parked in 8 bits and resumed, single tokens, and the
    output norm: each operator on what the one before it gave."""
    h, dk, dv, lengths = 3, 24, 40, [70, 5, 130]
    n = sum(lengths)
    off = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v, d, _ = inputs(91, n, h, h, h, dk, dv, DT[dtype], True)
    state = torch.zeros(4, h, dk, dv, device="cuda")
    ops.linear_attention(q, k, v, d, state=state, offsets=off, slots=[2, 0, 3])
    want = reference(q, k, v, d, [(range(off[i], off[i + 1]), s) for i, s in enumerate([2, 0, 3])],
                     torch.zeros_like(state), 1.0)[1]
    codes, scales = ops.state_cache(6, h * dk, dv, block=20, dtype=torch.float8_e4m3fn)
    parked = torch.tensor([5, 1], dtype=torch.int32, device="cuda")
    ops.state_store(state[[2, 3]].reshape(2, h * dk, dv), codes, scales, block=20, slots=parked)
    got = ops.state_load(codes, scales, block=20, slots=parked).reshape(2, h, dk, dv)
    # e4m3: half a step, 2^-4 of a value, or 2^-10 of the smallest normal code's scale
    amax = want[[2, 3]].abs().amax(-1, keepdim=True)
    assert ((got - want[[2, 3]]).abs() <= 2.0 ** -4 * want[[2, 3]].abs() * 1.001 + amax / 448 * 2.0 ** -9 + 1e-5).all()
    state[[2, 3]] = got
    before = state.clone()
    q1, k1, v1, d1, _ = inputs(95, 3, h, h, h, dk, dv, DT[dtype], True)
    slots = torch.tensor([3, 0, 2], dtype=torch.int32, device="cuda")
    o = ops.linear_attention_step(q1, k1, v1, d1, state, slots=slots)
    check_attention(q1, k1, v1, d1, [([r], int(s)) for r, s in enumerate(slots)], before, 1.0, o, state)
    y = ops.group_norm(o.reshape(3, h * dv), h)
    check_norm(o.reshape(3, 1, h * dv), h, None, None, "silu", y[:, None])


@pytest.mark.parametrize("dtype", DT)
def test_steps_follow_the_chunked_form(dtype):
    """A prompt in pieces: chunked, then token by token, then chunked again, against the recurrence."""
    h, dk, dv, n = 2, 48, 32, 150
    q, k, v, d, state = inputs(97, n, h, h, h, dk, dv, DT[dtype], True, slots=1)
    before = state.clone()
    out = torch.empty_like(v)
    ops.linear_attention(q[:70], k[:70], v[:70], d[:70], state=state, out=out[:70])
    for r in range(70, 80):
        ops.linear_attention_step(q[r:r + 1], k[r:r + 1], v[r:r + 1], d[r:r + 1], state, out=out[r:r + 1])
    ops.linear_attention(q[80:], k[80:], v[80:], d[80:], state=state, out=out[80:])
    check_attention(q, k, v, d, [(range(n), 0)], before, 1.0, out, state)


def everything(s, stream=None):
    o = ops.linear_attention(s["q"], s["k"], s["v"], s["d"], state=s["state"], offsets=[0, 900, 1000], stream=stream)
    o1 = ops.linear_attention_step(s["q"][:3], s["k"][:3], s["v"][:3], s["d"][:3], s["state"], slots=s["slots"], stream=stream)
    y = ops.group_norm(o.reshape(1, 1000, -1), 2, stream=stream)
    y1 = ops.group_norm(o1.reshape(3, -1), 2, stream=stream)
    x = s["state"].reshape(3, -1, s["state"].shape[-1])
    ops.state_store(x, s["codes"], s["scales"], block=32, slots=s["slots"], stream=stream)
    z = ops.state_load(s["codes"], s["scales"], block=32, slots=s["slots"], stream=stream)
    return [o, o1, y, y1, z]


def make(seed):
    q, k, v, d, state = inputs(seed, 1000, 2, 2, 2, 24, 40, torch.bfloat16, True, slots=3)
    codes, scales = ops.state_cache(4, 48, 40, block=32)
    return {"q": q, "k": k, "v": v, "d": d, "state": state, "codes": codes, "scales": scales,
            "slots": torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")}


def test_captured_and_replayed():
    """Two graphs of the whole set, replayed in turn on new inputs and slots."""
    graphs = []
    for seed in (1, 2):
        s = make(seed)
        everything(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = everything(s)
        graphs.append((g, s, r))
    for seed in (11, 12, 13):
        for i, (g, s, r) in enumerate(graphs):
            new = make(seed + 10 * i)
            new["slots"] = torch.tensor([[0, 1, 2], [1, 2, 0], [2, 0, -1]][seed - 11], dtype=torch.int32, device="cuda")
            for name, t in new.items():
                s[name].copy_(t)
            g.replay()
            want = everything(new)
            torch.cuda.synchronize()
            for a, b in zip(r, want):
                assert torch.equal(a, b)
            assert torch.equal(s["state"], new["state"]) and torch.equal(s["codes"], new["codes"])


def test_on_other_streams():
    """The current stream, an explicit one, and two at once."""
    want = everything(make(5))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    s1, s2 = make(5), make(5)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        r1 = everything(s1)
    r2 = everything(s2, stream=b)
    r3 = everything(make(5), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for r in (r1, r2, r3):
        for x, y in zip(r, want):
            assert torch.equal(x, y)


def test_a_stream_given_as_zero_is_the_legacy_default():
    x = rand(1, 4, 64)
    assert torch.equal(ops.group_norm(x, 4, stream=0), ops.group_norm(x, 4))


def test_no_wait_ran_out():
    assert ops.linear_attention_status() == 0


# ---- the repeated call --------------------------------------------------------------------


def test_repeated_calls_answer_like_the_first():
    """The same shapes again (the extension module's path): new values, new
    places, given outputs; and the same refusals as the first call."""
    assert ops._fast is not None, "build with `python ssla_rt_b200/build.py`"
    for rep in range(3):
        q, k, v, d, state = inputs(101 + 7 * rep, 5, 2, 2, 2, 24, 40, torch.bfloat16, True, slots=6)
        slots = torch.tensor([[0, 1, 2, 3, 4], [5, 4, 3, 3, -1], [2, 2, 2, 9, 0]][rep], dtype=torch.int32, device="cuda")
        before = state.clone()
        out = ops.linear_attention_step(q, k, v, d, state, slots=slots, scale=0.5)
        named = [s for s in dict.fromkeys(slots.tolist()) if 0 <= s < 6]
        seqs = [([r for r, x in enumerate(slots.tolist()) if x == s], s) for s in named]
        check_attention(q, k, v, d, seqs, before, 0.5, out, state)
        given = torch.empty_like(v)
        assert ops.linear_attention_step(q, k, v, d, before, slots=slots, scale=0.5, out=given) is given
        assert torch.equal(given, out) and torch.equal(before, state)

        x = rand(rep, 3, 7, 40)
        codes, scales = ops.state_cache(4, 7, 40, block=16)
        s3 = torch.tensor([3, 0, 2], dtype=torch.int32, device="cuda")
        ops.state_store(x, codes, scales, block=16, slots=s3)
        want_c, want_s = quantised(x, 16, torch.int8)
        assert np.array_equal(codes[s3.long()].float().cpu().numpy(), want_c)
        for back in DT.values():
            y = ops.state_load(codes, scales, block=16, slots=s3, dtype=back)
            assert torch.equal(y.cpu(), torch.from_numpy(want_c.astype(np.float32) * np.repeat(want_s, 16, 2)[:, :, :40]).to(back))

        for n, p, c, g in ((3, 1, 96, 4), (2, 300, 96, 8), (1, 20000, 12, 1)):
            x = rand(rep + 9, n, p, c)
            w = 1 + 0.1 * rand(rep, c)
            check_norm(x, g, w, None, "silu", ops.group_norm(x, g, w))
            y = torch.empty_like(x)
            assert ops.group_norm(x, g, w, out=y) is y and torch.equal(y, ops.group_norm(x, g, w))
    from ssla_rt_b200.engine import SslaError
    with pytest.raises(SslaError):
        ops.linear_attention_step(q, k, v, d, state, slots=slots, scale=0.5, out=v)
    with pytest.raises(ValueError, match="gradient"):
        ops.linear_attention_step(q.clone().requires_grad_(), k, v, d, state, slots=slots, scale=0.5)
    with pytest.raises(ValueError, match="slots"):
        ops.linear_attention_step(q, k, v, d, state, slots=slots.long(), scale=0.5)
    with pytest.raises(SslaError):
        ops.group_norm(x, g, x.reshape(-1)[:c], out=x)


def test_repeated_sequence_calls_answer_like_the_first():
    """linear_attention again on the same shapes: other sequences, host arrays of every kind, gaps, given outputs, refusals."""
    from ssla_rt_b200.engine import SslaError
    n = 90
    for rep, kw in enumerate([dict(offsets=[0, 30, 90]), dict(offsets=np.array([0, 30, 90], np.int32)),
                              dict(offsets=np.array([0, 30, 80], np.int32)), dict(offsets=torch.tensor([0, 1, 90])),
                              dict(offsets=np.array([5, 50], np.int32), lengths=np.array([20, 40], np.int32)),
                              dict(offsets=np.array([5, 50], np.int64), lengths=[20, 0]),
                              dict(offsets=np.array([0, 30, 90], np.int32), slots=np.array([2, -1], np.int32)),
                              dict(), dict(offsets=np.array([10], np.int32)),
                              dict(offsets=np.array([0, 30, 90, 7], np.int32)[:3])]):
        q, k, v, d, state = inputs(201 + rep, n, 2, 2, 2, 24, 40, torch.bfloat16, True, slots=3)
        before = state.clone()
        off = [int(x) for x in kw.get("offsets", [0, n])]
        lens = [int(x) for x in kw["lengths"]] if "lengths" in kw else [b - a for a, b in zip(off, off[1:])]
        slots = [int(x) for x in kw.get("slots", range(len(lens)))]
        seqs = [(range(off[i], off[i] + m), s) for i, (m, s) in enumerate(zip(lens, slots))]
        out = ops.linear_attention(q, k, v, d, state=state, scale=0.5, **kw)
        inside = sorted(r for rr, _ in seqs for r in rr)
        if inside:
            check_attention(q, k, v, d, seqs, before, 0.5, out, state, inside)
        assert (out[[r for r in range(n) if r not in set(inside)]] == 0).all()
        given = torch.full_like(v, 7.0)
        again = before.clone()
        assert ops.linear_attention(q, k, v, d, state=again, scale=0.5, out=given, **kw) is given
        assert torch.equal(given[inside], out[inside]) and torch.equal(again, state)
        assert (given[[r for r in range(n) if r not in set(inside)]] == 7).all()
    for bad in (dict(offsets=np.array([0, 91], np.int32)), dict(offsets=np.array([50, 30], np.int32)),
                dict(offsets=np.array([0, 30, 90], np.int32), slots=np.array([1, 1], np.int32)),
                dict(offsets=np.array([0, 30, 90], np.int32), slots=np.array([3, 0], np.int32))):
        with pytest.raises(SslaError):
            ops.linear_attention(q, k, v, d, state=state, scale=0.5, **bad)
    for bad in (dict(offsets=np.array([0, 30, 90], np.int32), slots=np.array([1], np.int32)), dict(lengths=[3]),
                dict(offsets=np.array([], np.int32)), dict(offsets=np.zeros((2, 2), np.int32)),
                dict(offsets=torch.tensor([0, 90], device="cuda", dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.linear_attention(q, k, v, d, state=state, scale=0.5, **bad)
