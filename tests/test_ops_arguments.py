"""Arguments of the wrong kind are refused with ValueError, whatever else is
given (no GPU needed)."""
import numpy as np
import pytest
import torch

from ssla_rt_b200 import ops


@pytest.mark.parametrize("slots", [[0, 1], (1,), 0])
@pytest.mark.parametrize("out", [False, True])
def test_load_refuses_slots_that_are_no_tensor(slots, out):
    codes, scales = ops.state_cache(4, 3, 8, block=4, device="cpu")
    with pytest.raises(ValueError, match="slots"):
        ops.state_load(codes, scales, block=4, slots=slots, out=torch.zeros(2, 3, 8) if out else None)


def calls():
    z = torch.zeros
    codes, scales = ops.state_cache(2, 3, 8, block=4, device="cpu")
    att = dict(q=z(6, 4, 8), k=z(6, 4, 8), v=z(6, 4, 8), decay=z(4))
    return {
        "chunk": (dict(att, state=z(1, 4, 8, 8), out=z(6, 4, 8)), lambda **t: ops.linear_attention(**t)),
        "step": (dict(att, state=z(6, 4, 8, 8), out=z(6, 4, 8)), lambda **t: ops.linear_attention_step(**t)),
        "store": (dict(x=z(2, 3, 8), codes=codes, scales=scales), lambda **t: ops.state_store(block=4, **t)),
        "load": (dict(codes=codes, scales=scales, out=z(2, 3, 8)), lambda **t: ops.state_load(block=4, **t)),
        "norm": (dict(x=z(2, 3, 8), weight=z(8), bias=z(8), out=z(2, 3, 8)), lambda **t: ops.group_norm(groups=2, **t)),
    }


@pytest.mark.parametrize("op,name", [(op, name) for op, (tensors, _) in calls().items() for name in tensors])
@pytest.mark.parametrize("bad", [np.zeros((6, 4, 8), np.float32), [1.0], 3, "x", torch.tensor(1.0)], ids=lambda b: type(b).__name__)
def test_what_is_no_tensor_is_refused(op, name, bad):
    tensors, call = calls()[op]
    with pytest.raises(ValueError):
        call(**{**tensors, name: bad})


@pytest.mark.parametrize("op,name", [("chunk", "q"), ("chunk", "v"), ("step", "state"), ("step", "decay"), ("store", "x"),
                                     ("load", "codes"), ("norm", "x")])
def test_what_is_needed_is_not_none(op, name):
    tensors, call = calls()[op]
    with pytest.raises(ValueError, match="tensor|needed"):
        call(**{**tensors, name: None})


def test_rows_out_shape():
    with pytest.raises(ValueError, match="out is"):
        ops.group_norm(torch.zeros(3, 8), 2, out=torch.zeros(8))
