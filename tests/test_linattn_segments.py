"""Divided sequences stay within a grid's depth of 65535 segments, however
many and long they are (from the workspace's size: no GPU needed)."""
import ctypes as C

import pytest

from ssla_rt_b200 import abi
from ssla_rt_b200.engine import load_library

A = 1 << 45     # addresses that are never read


def segments(n_seq, tokens, heads=1, dk=24, dv=24, dtype=abi.DT_F32):
    n = n_seq * tokens
    size = 4 if dtype == abi.DT_F32 else 2
    row = heads * max(dk, dv)
    a = abi.SslaLinAttn(q=A, k=2 * A, v=3 * A, out=4 * A, decay=5 * A, state=6 * A, q_row=row, q_head=dk, k_row=row, k_head=dk,
                        v_row=row, v_head=dv, out_row=row, out_head=dv, decay_head=1, n_rows=n, heads=heads, q_heads=heads,
                        k_heads=heads, dk=dk, dv=dv, dtype=dtype, n_slots=n_seq, scale=1.0)
    assert n * row * size < A
    off = (C.c_int * (n_seq + 1))(*range(0, n + 1, tokens))
    need, lib = C.c_size_t(), load_library()
    assert lib.ssla_linattn_chunk_workspace(C.byref(a), off, None, n_seq, C.byref(need)) == abi.SSLA_OK, lib.ssla_last_error()
    per = heads * (8 + 4 * dk * dv)
    assert need.value % per == 0
    return need.value // per


@pytest.mark.parametrize("n_seq,tokens", [(256, 131072), (200, 131072), (256, 65536), (256, 1 << 22), (150, 1 << 23), (1, 1 << 30)])
@pytest.mark.parametrize("dtype", [abi.DT_F32, abi.DT_BF16])
def test_segments_of_a_launch(n_seq, tokens, dtype):
    assert segments(n_seq, tokens, dtype=dtype) <= 65535
    assert segments(n_seq, tokens, dk=64, dv=64, dtype=dtype) <= 65535


def test_ordinary_calls_are_divided_as_before():
    assert segments(8, 25000, heads=4) == 144
    assert segments(1, 65537, heads=4, dk=64, dv=64, dtype=abi.DT_BF16) == 36
    assert segments(8, 2048, heads=16, dk=128, dv=128, dtype=abi.DT_BF16) == 0


def test_segments_pay_for_their_setup():
    """Enough CTAs without a division, if not evenly loaded: none in the tcgen05 form."""
    assert segments(8, 4096, heads=16, dk=128, dv=128, dtype=abi.DT_BF16) == 0
    assert segments(4, 4096, heads=16, dk=128, dv=128, dtype=abi.DT_BF16) == 0
    assert segments(2, 8192, heads=16, dk=128, dv=128, dtype=abi.DT_BF16) == 8
    assert segments(8, 8192, heads=4, dk=64, dv=64, dtype=abi.DT_BF16) == 32
