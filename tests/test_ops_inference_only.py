"""Inference only: what autograd would have to follow is refused, in either
mode, for inputs and for given outputs (no GPU needed; the repeated calls'
route refuses the same on one)."""
import pytest
import torch
from torch.autograd import forward_ad

from ssla_rt_b200 import ops


def calls(dev="cpu"):
    """name -> (tensors by name, call of them)"""
    z = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    codes, scales = ops.state_cache(2, 3, 8, block=4, device=dev)
    return {
        "chunk": (dict(q=z(6, 4, 8), k=z(6, 4, 8), v=z(6, 4, 8), decay=z(4), state=z(1, 4, 8, 8), out=z(6, 4, 8)),
                  lambda t: ops.linear_attention(t["q"], t["k"], t["v"], t["decay"], state=t["state"], out=t["out"])),
        "step": (dict(q=z(6, 4, 8), k=z(6, 4, 8), v=z(6, 4, 8), decay=z(4), state=z(6, 4, 8, 8), out=z(6, 4, 8)),
                 lambda t: ops.linear_attention_step(t["q"], t["k"], t["v"], t["decay"], t["state"], out=t["out"])),
        "store": (dict(x=z(2, 3, 8), scales=scales), lambda t: ops.state_store(t["x"], codes, t["scales"], block=4)),
        "load": (dict(scales=scales, out=z(2, 3, 8)), lambda t: ops.state_load(codes, t["scales"], block=4, out=t["out"])),
        "norm": (dict(x=z(2, 3, 8), weight=z(8), bias=z(8), out=z(2, 3, 8)),
                 lambda t: ops.group_norm(t["x"], 2, t["weight"], t["bias"], out=t["out"])),
    }


CASES = [(op, name) for op, (tensors, _) in calls().items() for name in tensors]


@pytest.mark.parametrize("op,name", CASES)
def test_gradient_refused(op, name):
    t, call = calls()[op]
    t[name].requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        call(t)


@pytest.mark.parametrize("op,name", CASES)
@pytest.mark.parametrize("mode", [torch.no_grad, torch.enable_grad])
def test_tangent_refused(op, name, mode):
    t, call = calls()[op]
    with forward_ad.dual_level(), mode():
        t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(ValueError, match="tangent"):
            call(t)


@pytest.mark.gpu
@pytest.mark.parametrize("op,name", CASES)
def test_refused_in_repeated_calls_too(op, name):
    t, call = calls("cuda")[op]
    call(t)
    call(t)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            call({**t, name: forward_ad.make_dual(t[name], torch.ones_like(t[name]))})
    with pytest.raises(ValueError, match="gradient"):
        call({**t, name: t[name].detach().requires_grad_()})
    call(t)
    with torch.no_grad():
        call({**t, name: t[name].detach().requires_grad_()})
