"""More sequences than states: those of slot -1 start from zero and leave
nothing, whatever their number."""
import ctypes as C

import numpy as np
import pytest
import torch

from ssla_rt_b200 import abi, ops
from ssla_rt_b200.engine import load_library

A = 1 << 20     # addresses that are never read


@pytest.mark.parametrize("lengths", [None, [1, 1, 0, 2, 1, 0]])
def test_workspace_does_not_depend_on_slots(lengths):
    a = abi.SslaLinAttn(q=A, k=2 * A, v=3 * A, out=4 * A, decay=5 * A, state=6 * A, q_row=32, q_head=8, k_row=32,
                        k_head=8, v_row=32, v_head=8, out_row=32, out_head=8, decay_head=1, n_rows=6, heads=4,
                        q_heads=4, k_heads=4, dk=8, dv=8, dtype=abi.DT_F32, n_slots=2, scale=1.0)
    off = [0, 1, 2, 2, 4, 5, 5][:6 if lengths else 7]
    arr = lambda x: (C.c_int * len(x))(*x) if x else None  # noqa: E731
    need, lib = C.c_size_t(77), load_library()
    rc = lib.ssla_linattn_chunk_workspace(C.byref(a), arr(off), arr(lengths), 6, C.byref(need))
    assert rc == abi.SSLA_OK and need.value == 0, lib.ssla_last_error()
    # the call itself still refuses slots that are not there
    for slots in (None, [0, -1, 2, -1, -1, 1], [0, -1, 0, -1, -1, -1]):
        assert lib.ssla_linattn_chunk(C.byref(a), arr(off), arr(lengths), arr(slots), 6, None, 0, None) == abi.SSLA_ERR_ARG
        assert "slot" in lib.ssla_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dims", [(24, 40), (64, 64)], ids=str)
@pytest.mark.parametrize("fast", [True, False])
def test_more_sequences_than_slots(dtype, dims, fast):
    from test_gpu_ops import DT, check_attention, inputs
    off, slots = np.array([0, 70, 70, 90, 150, 151, 200], np.int32), np.array([1, -1, -1, 0, -1, -1], np.int32)
    q, k, v, d, state = inputs(501, 200, 2, 2, 1, *dims, DT[dtype], True, slots=2)
    before = state.clone()
    stream = None if fast else torch.cuda.current_stream()
    for _ in range(2):                                    # the second by the kept plan
        state.copy_(before)
        out = ops.linear_attention(q, k, v, d, state=state, offsets=off, slots=slots, scale=0.5, stream=stream)
        seqs = [(range(off[i], off[i + 1]), int(slots[i])) for i in range(6)]
        check_attention(q, k, v, d, seqs, before, 0.5, out, state)
    state.copy_(before)
    lengths = np.diff(off).astype(np.int32)
    assert torch.equal(ops.linear_attention(q, k, v, d, state=state, offsets=off[:-1], lengths=lengths, slots=slots, scale=0.5,
                                            stream=stream), out)
