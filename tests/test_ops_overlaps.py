"""Workspaces and slots that lie in a tensor of the call are refused; so is a
workspace that is missing, too small or unaligned (no GPU needed: every check
comes before the first CUDA call)."""
import ctypes as C

import pytest

from ssla_rt_b200 import abi
from ssla_rt_b200.engine import load_library

A = 1 << 34     # addresses that are never read, far apart


def attention(n, heads=2, d=24):
    row = heads * d
    return abi.SslaLinAttn(q=A, k=2 * A, v=3 * A, out=4 * A, decay=5 * A, state=6 * A, q_row=row, q_head=d, k_row=row, k_head=d,
                           v_row=row, v_head=d, out_row=row, out_head=d, decay_row=heads, decay_head=1, n_rows=n, heads=heads,
                           q_heads=heads, k_heads=heads, dk=d, dv=d, dtype=abi.DT_F32, n_slots=1, scale=1.0)


def refused(rc, text):
    return rc == abi.SSLA_ERR_ARG and text in load_library().ssla_last_error().decode()


@pytest.mark.parametrize("which", range(1, 7))
@pytest.mark.parametrize("inside", [True, False])
def test_sequence_workspace_in_a_tensor(which, inside):
    lib, a, n = load_library(), attention(100000), 100000
    off, need = (C.c_int * 2)(0, n), C.c_size_t()
    assert lib.ssla_linattn_chunk_workspace(C.byref(a), off, None, 1, C.byref(need)) == abi.SSLA_OK and need.value > 0
    at = which * A + 64 if inside else which * A - need.value + 16
    assert refused(lib.ssla_linattn_chunk(C.byref(a), off, None, None, 1, at, need.value, None), "workspace overlaps")


@pytest.mark.parametrize("at,less", [(None, 0), (7 * A, 1), (7 * A + 8, 0)])
def test_sequence_workspace_is_needed(at, less):
    lib, a, n = load_library(), attention(100000), 100000
    off, need = (C.c_int * 2)(0, n), C.c_size_t()
    lib.ssla_linattn_chunk_workspace(C.byref(a), off, None, 1, C.byref(need))
    assert refused(lib.ssla_linattn_chunk(C.byref(a), off, None, None, 1, at, need.value - less, None), "workspace of")


@pytest.mark.parametrize("at", [4 * A, 4 * A + 100, 4 * A - 8, 6 * A, 6 * A + 64])
def test_step_slots_in_what_is_written(at):
    a = attention(5)
    a.n_slots = 9
    assert refused(load_library().ssla_linattn_step(C.byref(a), at, None), "overlaps slots")


def norm():
    """One sample larger than any cluster's shared memory: the form with a workspace."""
    c, p = 96, 200000
    a = abi.SslaGroupNorm(x=A, y=2 * A, weight=3 * A, bias=4 * A, x_sample=p * c, x_pos=c, y_sample=p * c, y_pos=c, n=1,
                          positions=p, channels=c, groups=8, eps=1e-5)
    need = C.c_size_t()
    assert load_library().ssla_group_norm_workspace(C.byref(a), C.byref(need)) == abi.SSLA_OK and need.value > 0
    return a, need.value


@pytest.mark.parametrize("at,less", [(None, 0), (7 * A, 1), (7 * A + 8, 0)])
def test_norm_workspace_is_needed(at, less):
    a, need = norm()
    assert refused(load_library().ssla_group_norm(C.byref(a), at, need - less, None), "workspace of")


@pytest.mark.parametrize("which", range(1, 5))
@pytest.mark.parametrize("inside", [True, False])
def test_norm_workspace_in_a_tensor(which, inside):
    a, need = norm()
    at = which * A + 16 if inside else which * A - need // 16 * 16 + 16
    assert refused(load_library().ssla_group_norm(C.byref(a), at, need, None), "workspace overlaps")
