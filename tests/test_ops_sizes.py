"""Sizes next to what 32-bit counts hold are refused, never wrapped (no GPU
needed: every check comes before the first CUDA call)."""
import ctypes as C

import pytest
import torch

from ssla_rt_b200 import abi, ops
from ssla_rt_b200.engine import load_library

A = 1 << 20     # addresses that are never read: the checks refuse first
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("kw", [dict(positions=MOST), dict(positions=MOST - 65536 + 1), dict(n=MOST), dict(n=MOST - 65536 + 1),
                                dict(n=(MOST - 65536) // 2 + 1, channels=2, groups=2)])
def test_group_norm_counts(kw):
    """Positions and samples that a kernel's or the host's steps would carry past 2^31."""
    a = abi.SslaGroupNorm(x=A, y=1 << 45, x_sample=1, x_pos=1, y_sample=2, y_pos=2, n=1, positions=1, channels=1, groups=1,
                          dtype=abi.DT_BF16, eps=1e-5)
    for name, x in kw.items():
        setattr(a, name, x)
    lib, need = load_library(), C.c_size_t()
    for rc in (lib.ssla_group_norm_workspace(C.byref(a), C.byref(need)), lib.ssla_group_norm(C.byref(a), None, 0, None)):
        assert rc == abi.SSLA_ERR_ARG and "too large" in lib.ssla_last_error().decode()


def test_group_norm_largest_counts_are_planned():
    a = abi.SslaGroupNorm(x=A, y=1 << 45, x_sample=1, x_pos=1, y_sample=1, y_pos=1, n=1, positions=MOST - 65536, channels=1,
                          groups=1, dtype=abi.DT_BF16, eps=1e-5)
    lib, need = load_library(), C.c_size_t()
    assert lib.ssla_group_norm_workspace(C.byref(a), C.byref(need)) == abi.SSLA_OK and need.value > 0
    assert lib.ssla_group_norm(C.byref(a), None, 0, None) == abi.SSLA_ERR_ARG
    assert "workspace" in lib.ssla_last_error().decode()


WRAPS = 2 ** 32 + 6     # 6 in 32 bits


def broad(*shape, dtype=torch.float32):
    return torch.zeros((), dtype=dtype).expand(*shape)


@pytest.mark.parametrize("call", [
    lambda: ops.linear_attention(broad(WRAPS, 4, 8), broad(WRAPS, 4, 8), broad(WRAPS, 4, 8), torch.zeros(4)),
    lambda: ops.linear_attention(broad(6, WRAPS, 8), broad(6, 2, 8), broad(6, 2, 8), torch.zeros(2)),
    lambda: ops.linear_attention_step(*[torch.zeros(6, 4, 8)] * 3, torch.zeros(4), broad(WRAPS, 4, 8, 8)),
    lambda: ops.group_norm(broad(WRAPS, 3, 8), 2), lambda: ops.group_norm(broad(WRAPS, 8), 2),
    lambda: ops.group_norm(broad(2, WRAPS, 8), 2),
    lambda: ops.state_store(broad(WRAPS, 3, 8), *ops.state_cache(4, 3, 8, block=4, device="cpu"), block=4),
    lambda: ops.state_load(torch.zeros(WRAPS, 0, 1, dtype=torch.int8), torch.zeros(WRAPS, 0, 1), block=4),
])
def test_sizes_past_32_bits(call):
    with pytest.raises(ValueError, match="below 2\\^31"):
        call()
