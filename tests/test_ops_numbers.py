"""Numbers that are not plain Python ones -- numpy's -- mean what they hold,
in first and repeated calls."""
import numpy as np
import pytest
import torch

from ssla_rt_b200 import ops


@pytest.mark.parametrize("kind", [int, np.int64, np.int32, np.uint8])
def test_keys_of_whole_numbers_differ(kind):
    """The extension module's key holds the number itself, or there is none."""
    assert ops._fast is not None, "build with `python ssla_rt_b200/build.py`"
    x = torch.zeros(2, 3, 8)
    norm = [ops._fast.norm(x, kind(g), None, None, 1e-5, 0, None, True) for g in (2, 4)]
    codes, scales = ops.state_cache(2, 3, 8, block=4, device="cpu")
    store = [ops._fast.store(x, codes, scales, kind(b), None, True) for b in (5, 6)]
    load = [ops._fast.load(codes, scales, kind(b), None, 0, None, True) for b in (5, 6)]
    for a, b in (norm, store, load):
        assert a is None or a != b
    assert kind is not int or norm[0] is not None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [np.int64, np.int32])
def test_repeated_norms_and_caches(kind):
    x = torch.randn(3, 7, 24, device="cuda")
    for g in (2, 4, 8, 3, 2):
        for _ in range(2):
            assert torch.equal(ops.group_norm(x, kind(g)), ops.group_norm(x, g))
    for b in (13, 20, 12, 13):                            # two blocks a row, each time
        c0, s0 = ops.state_cache(3, 7, 24, block=b)
        c1, s1 = ops.state_cache(3, 7, 24, block=b)
        for _ in range(2):
            ops.state_store(x, c0, s0, block=b)
            ops.state_store(x, c1, s1, block=kind(b))
            assert torch.equal(c0, c1) and torch.equal(s0, s1)
            assert torch.equal(ops.state_load(c0, s0, block=b), ops.state_load(c0, s0, block=kind(b)))
