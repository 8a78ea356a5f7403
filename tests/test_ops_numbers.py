"""Numbers that are not plain Python ones -- numpy's, zero-dimensional tensors
-- mean what they hold at the time of the call, in first and repeated calls."""
import types

import numpy as np
import pytest
import torch

from ssla_rt_b200 import ops


def qkv():
    return (torch.zeros(6, 4, 8), torch.zeros(6, 4, 8), torch.zeros(6, 4, 8), torch.zeros(4))


@pytest.mark.parametrize("kind", [int, np.int64, np.int32, np.uint8, lambda x: torch.tensor(x)])
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


def on_cpu(monkeypatch):
    """The argument blocks of CPU tensors, as if they were on device 0."""
    monkeypatch.setattr(ops, "_device", lambda first, **others: 0)
    monkeypatch.setattr(ops, "_PLANS", {})


def test_a_scale_in_a_tensor_is_read_each_time(monkeypatch):
    on_cpu(monkeypatch)
    s = torch.tensor(0.5)
    assert ops._linattn(*qkv(), None, s, None).scale == 0.5
    s.fill_(0.25)
    assert ops._linattn(*qkv(), None, s, None).scale == 0.25
    assert ops._linattn(*qkv(), None, np.float64(0.125), None).scale == 0.125
    assert ops._linattn(*qkv(), None, np.array(2.0), None).scale == 2.0


def test_a_block_in_a_tensor_is_read_each_time(monkeypatch):
    on_cpu(monkeypatch)
    codes, scales = ops.state_cache(2, 3, 8, block=5, device="cpu")
    b = torch.tensor(5)
    assert ops._cache(codes, scales, b, None, 2, "x", None, torch.float32).block == 5
    b.fill_(6)
    assert ops._cache(codes, scales, b, None, 2, "x", None, torch.float32).block == 6


@pytest.mark.parametrize("bad", [2.5, "2", None, types.SimpleNamespace()])
def test_what_is_no_whole_number_is_refused(bad):
    x = torch.zeros(2, 3, 8)
    codes, scales = ops.state_cache(2, 3, 8, block=4, device="cpu")
    with pytest.raises(ValueError, match="groups"):
        ops.group_norm(x, bad)
    with pytest.raises(ValueError, match="block"):
        ops.state_store(x, codes, scales, block=bad)
    with pytest.raises(ValueError, match="block"):
        ops.state_load(codes, scales, block=bad)


@pytest.mark.parametrize("bad", ["x", None, torch.zeros(2), 1j])
def test_what_is_no_number_is_refused(bad):
    with pytest.raises(ValueError, match="scale"):
        ops.linear_attention(*qkv(), scale=bad)
    with pytest.raises(ValueError, match="scale"):
        ops.linear_attention_step(*qkv(), torch.zeros(6, 4, 8, 8), scale=bad)
    with pytest.raises(ValueError, match="eps"):
        ops.group_norm(torch.zeros(2, 3, 8), 2, eps=bad)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [np.int64, np.int32, lambda x: torch.tensor(x)])
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


@pytest.mark.gpu
def test_repeated_scales_and_eps():
    q, k, v = (torch.randn(9, 2, 24, device="cuda") for _ in range(3))
    d, state = -torch.rand(2, device="cuda"), torch.randn(9, 2, 24, 24, device="cuda")
    s = torch.tensor(0.5)
    for x in (0.5, 0.25, 2.0, 0.25):
        s.fill_(x)
        a = ops.linear_attention(q, k, v, d, scale=s)
        b = ops.linear_attention_step(q, k, v, d, state.clone(), scale=s)
        assert torch.equal(a, ops.linear_attention(q, k, v, d, scale=x))
        assert torch.equal(b, ops.linear_attention_step(q, k, v, d, state.clone(), scale=x))
        assert torch.equal(ops.group_norm(q, 2, eps=s), ops.group_norm(q, 2, eps=x))
