"""What the operators write in place advances its version, so that autograd
refuses to use a value that it saved before (torch's own rule)."""
import pytest
import torch

from ssla_rt_b200 import ops

pytestmark = pytest.mark.gpu


def rand(*s):
    return torch.randn(*s, device="cuda")


@pytest.mark.parametrize("fast", [True, False])
def test_versions_advance(fast):
    kw = {} if fast else {"stream": torch.cuda.current_stream()}
    q, k, v, d, state = rand(6, 2, 8), rand(6, 2, 8), rand(6, 2, 8), -rand(2).abs(), rand(6, 2, 8, 8)
    out, x, y = torch.empty_like(v), rand(2, 3, 8), rand(2, 3, 8)
    codes, scales = ops.state_cache(2, 3, 8, block=4)
    for written, call in (((state, out), lambda: ops.linear_attention(q, k, v, d, state=state, out=out, **kw)),
                          ((state, out), lambda: ops.linear_attention_step(q, k, v, d, state, out=out, **kw)),
                          ((codes, scales), lambda: ops.state_store(x, codes, scales, block=4, **kw)),
                          ((y,), lambda: ops.state_load(codes, scales, block=4, out=y, **kw)),
                          ((y,), lambda: ops.group_norm(x, 2, out=y, **kw))):
        for _ in range(3):
            before, kept = [t._version for t in written], [t._version for t in (q, k, v, d, x)]
            call()
            assert all(t._version > b for t, b in zip(written, before))
            assert [t._version for t in (q, k, v, d, x)] == kept


@pytest.mark.parametrize("fast", [True, False])
def test_a_saved_state_is_not_used_after_a_step(fast):
    kw = {} if fast else {"stream": torch.cuda.current_stream()}
    q, k, v, d, state = rand(6, 2, 8), rand(6, 2, 8), rand(6, 2, 8), -rand(2).abs(), rand(6, 2, 8, 8)
    ops.linear_attention_step(q, k, v, d, state, **kw)
    w = torch.ones(8, device="cuda", requires_grad=True)
    loss = (state * w).sum()
    ops.linear_attention_step(q, k, v, d, state, **kw)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_inference_tensors_are_written_too():
    with torch.inference_mode():
        q, k, v, d, state = rand(6, 2, 8), rand(6, 2, 8), rand(6, 2, 8), -rand(2).abs(), rand(6, 2, 8, 8)
        for kw in ({}, {}, {"stream": torch.cuda.current_stream()}):
            ops.linear_attention_step(q, k, v, d, state, out=torch.empty_like(v), **kw)
            ops.group_norm(v, 2, out=v, **kw)
    ops.linear_attention_step(q, k, v, d, state)
