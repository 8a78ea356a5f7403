"""The recurrent-state operators' refusals and ABI (no GPU needed): every
argument check comes before the first CUDA call, so a wrong call is refused
the same way on any host."""
import ctypes as C
import os
import re

import pytest
import torch

from ssla_rt_b200 import abi, ops
from ssla_rt_b200.engine import SslaError, load_library
from conftest import REPO


def test_exports_match_header():
    hdr = open(os.path.join(REPO, "include", "ssla_ops.h")).read()
    declared = set(re.findall(r"^int\s+(ssla_[a-z0-9_]+)\s*\(", hdr, re.M))
    assert declared == set(abi.OPS_EXPORTED)
    lib = load_library()
    for name in declared:
        assert hasattr(lib, name), name


def test_struct_layouts():
    # pointers, then 64-bit strides, then 32-bit fields, no holes
    assert C.sizeof(abi.SslaLinAttn) == 6 * 8 + 10 * 8 + 10 * 4
    assert C.sizeof(abi.SslaStateCache) == 3 * 8 + 2 * 8 + 8 * 4
    assert C.sizeof(abi.SslaGroupNorm) == 4 * 8 + 4 * 8 + 8 * 4


def qkv(n=6, h=4, hq=4, hk=4, dk=8, dv=8, dtype=torch.bfloat16):
    return (torch.zeros(n, hq, dk, dtype=dtype), torch.zeros(n, hk, dk, dtype=dtype),
            torch.zeros(n, h, dv, dtype=dtype), torch.zeros(h))


REFUSED_ATTENTION = {
    "two dimensions": lambda q, k, v, d: ((q[0], k, v, d), {}, "rows, heads, width"),
    "mixed types": lambda q, k, v, d: ((q.float(), k, v, d), {}, "not torch.bfloat16"),
    "64-bit": lambda q, k, v, d: ((q.double(), k.double(), v.double(), d), {}, "not supported"),
    "strided last dimension": lambda q, k, v, d: ((q, k, v.transpose(1, 2).contiguous().transpose(1, 2), d), {},
                                                  "last dimension"),
    "rows": lambda q, k, v, d: ((q[:5], k, v, d), {}, "fit together"),
    "widths": lambda q, k, v, d: ((q, k[:, :, :7], v, d), {}, "fit together"),
    "decay type": lambda q, k, v, d: ((q, k, v, d.double()), {}, "decay"),
    "decay shape": lambda q, k, v, d: ((q, k, v, d[:3]), {}, "decay"),
    "state type": lambda q, k, v, d: ((q, k, v, d), {"state": torch.zeros(1, 4, 8, 8, dtype=torch.bfloat16)}, "state"),
    "state shape": lambda q, k, v, d: ((q, k, v, d), {"state": torch.zeros(1, 4, 8, 9)}, "state"),
    "state strides": lambda q, k, v, d: ((q, k, v, d), {"state": torch.zeros(1, 4, 8, 8).transpose(2, 3)}, "contiguous"),
    "out shape": lambda q, k, v, d: ((q, k, v, d), {"out": v[:, :2]}, "out"),
    "out type": lambda q, k, v, d: ((q, k, v, d), {"out": v.float()}, "out"),
    "gradient": lambda q, k, v, d: ((q.clone().requires_grad_(), k, v, d), {}, "gradient"),
    "cpu": lambda q, k, v, d: ((q, k, v, d), {}, "CUDA"),
    "lengths alone": lambda q, k, v, d: ((q, k, v, d), {"lengths": [6]}, "offsets"),
    "empty offsets": lambda q, k, v, d: ((q, k, v, d), {"offsets": []}, "empty"),
    "float offsets": lambda q, k, v, d: ((q, k, v, d), {"offsets": [0.0, 6.0]}, "integers"),
    "wide offsets": lambda q, k, v, d: ((q, k, v, d), {"offsets": [0, 2**31]}, "32 bits"),
    "lengths count": lambda q, k, v, d: ((q, k, v, d), {"offsets": [0, 3], "lengths": [3]}, "lengths"),
    "slots count": lambda q, k, v, d: ((q, k, v, d), {"offsets": [0, 6], "slots": [0, 1]}, "slots"),
}


@pytest.mark.parametrize("case", REFUSED_ATTENTION)
def test_linear_attention_refuses(case):
    args, kw, msg = REFUSED_ATTENTION[case](*qkv())
    with pytest.raises(ValueError, match=msg):
        ops.linear_attention(*args, **kw)


@pytest.mark.parametrize("slots,msg", [(torch.zeros(6, dtype=torch.int64), "int32"), (torch.zeros(5, dtype=torch.int32), "entries"),
                                       (torch.zeros(12, dtype=torch.int32)[::2], "entries"), ([0] * 6, "int32")])
def test_step_refuses_slots(slots, msg):
    with pytest.raises(ValueError, match=msg):
        ops.linear_attention_step(*qkv(), torch.zeros(6, 4, 8, 8), slots=slots)


def test_step_needs_a_state():
    with pytest.raises(ValueError, match="state"):
        ops.linear_attention_step(*qkv(), None)


A = 1 << 20     # addresses that are never read: the checks refuse first


def block(**kw):
    a = abi.SslaLinAttn(q=A, k=2 * A, v=3 * A, out=4 * A, decay=5 * A, state=6 * A, q_row=32, q_head=8, k_row=32,
                        k_head=8, v_row=32, v_head=8, out_row=32, out_head=8, decay_head=1, n_rows=6, heads=4,
                        q_heads=4, k_heads=4, dk=8, dv=8, dtype=abi.DT_F32, n_slots=3, scale=1.0)
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def chunk(a, offsets=(0, 6), lengths=None, slots=None, n_seq=None):
    lib = load_library()
    arr = lambda x: (C.c_int * len(x))(*x) if x is not None else None  # noqa: E731
    n = n_seq if n_seq is not None else len(offsets) - (lengths is None)
    rc = lib.ssla_linattn_chunk(C.byref(a), arr(offsets), arr(lengths), arr(slots), n, None, 0, None)
    return rc, lib.ssla_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"), (dict(heads=0), "heads"), (dict(q_heads=3), "q_heads"), (dict(k_heads=8), "k_heads"),
    (dict(dk=0), "dk"), (dict(dk=129), "dk"), (dict(dv=257), "dv"), (dict(scale=float("nan")), "scale"),
    (dict(q=None), "null"), (dict(decay=None), "null"), (dict(out=None), "null"), (dict(n_rows=-1), "negative"),
    (dict(q=A + 2), "aligned"), (dict(state=6 * A + 1), "aligned"), (dict(v_row=-32), "stride"),
    (dict(out_row=16), "overlaps itself"), (dict(out_head=0), "overlaps itself"),
    (dict(out=3 * A + 4), "overlaps an input"), (dict(state=A), "overlaps an input"), (dict(state=4 * A), "overlaps state"),
])
def test_linattn_block_refused(kw, msg):
    rc, text = chunk(block(**kw))
    assert rc == abi.SSLA_ERR_ARG and msg in text, text
    rc = load_library().ssla_linattn_step(C.byref(block(**kw, **({} if "n_rows" in kw else {"n_rows": 3}))), None, None)
    assert rc == abi.SSLA_ERR_ARG


@pytest.mark.parametrize("kw,msg", [
    (dict(offsets=(0, 7)), "rows"), (dict(offsets=(-1, 6)), "rows"), (dict(offsets=(0, 4, 3)), "rows"),
    (dict(offsets=(0, 4), lengths=(2, -1)), "rows"), (dict(offsets=(0, 4), lengths=(2, 3)), "rows"),
    (dict(offsets=(0, 2), lengths=(3, 3)), "overlap"), (dict(slots=(3,)), "slot"), (dict(slots=(-2,)), "slot"),
    (dict(offsets=(0, 1, 2, 3), slots=(1, 0, 1)), "twice"), (dict(offsets=(0, 1, 2, 3, 4)), "slot"),
])
def test_linattn_sequences_refused(kw, msg):
    rc, text = chunk(block(), **kw)
    assert rc == abi.SSLA_ERR_ARG and msg in text, text


def test_linattn_null_arguments():
    lib = load_library()
    assert lib.ssla_linattn_chunk(None, None, None, None, 0, None, 0, None) == abi.SSLA_ERR_ARG
    assert lib.ssla_linattn_step(None, None, None) == abi.SSLA_ERR_ARG
    assert lib.ssla_linattn_status(0, None) == abi.SSLA_ERR_ARG
    assert lib.ssla_linattn_chunk(C.byref(block()), None, None, None, 1, None, 0, None) == abi.SSLA_ERR_ARG
    assert lib.ssla_linattn_chunk_workspace(C.byref(block()), None, None, 0, None) == abi.SSLA_ERR_ARG
    # a state-less call that names slots
    rc, text = chunk(block(state=None), slots=(0,))
    assert rc == abi.SSLA_ERR_ARG and "slot" in text
    # more rows than slots, in the step
    assert lib.ssla_linattn_step(C.byref(block()), None, None) == abi.SSLA_ERR_ARG


def cache_args():
    x = torch.zeros(2, 3, 8)
    codes, scales = ops.state_cache(4, 3, 8, block=4, device="cpu")
    return x, codes, scales


@pytest.mark.parametrize("change,kw,msg", [
    (lambda x, c, s: (x, c.float(), s), {}, "int8"), (lambda x, c, s: (x, c[:, :, :7], s), {}, "codes"),
    (lambda x, c, s: (x, c, s[:, :, :1]), {}, "scales"), (lambda x, c, s: (x, c, s.double()), {}, "scales"),
    (lambda x, c, s: (x[:, :, :7], c, s), {}, "x is"), (lambda x, c, s: (x.double(), c, s), {}, "x is"),
    (lambda x, c, s: (x.transpose(1, 2).contiguous().transpose(1, 2), c, s), {}, "last dimension"),
    (lambda x, c, s: (x, c, s), {"block": 0}, "block"), (lambda x, c, s: (x, c, s), {"block": 300}, "block"),
    (lambda x, c, s: (x, c, s), {"slots": torch.zeros(2)}, "int32"),
    (lambda x, c, s: (x, c, s), {"slots": torch.zeros(3, dtype=torch.int32)}, "entries"),
    (lambda x, c, s: (x, c, s), {}, "CUDA"),
])
def test_state_store_refuses(change, kw, msg):
    with pytest.raises(ValueError, match=msg):
        ops.state_store(*change(*cache_args()), **{"block": 4, **kw})


def test_state_load_refuses():
    _, codes, scales = cache_args()
    with pytest.raises(ValueError, match="not supported"):
        ops.state_load(codes, scales, block=4, dtype=torch.float64)
    with pytest.raises(ValueError, match="out is"):
        ops.state_load(codes, scales, block=4, out=torch.zeros(4, 3, 9))
    with pytest.raises(ValueError, match="CUDA"):
        ops.state_load(codes, scales, block=4)
    with pytest.raises(ValueError, match="not supported"):
        ops.state_cache(4, 3, 8, dtype=torch.uint8, device="cpu")


def cache_block(**kw):
    c = abi.SslaStateCache(codes=2 * A, scales=3 * A, x_state=24, x_row=8, n=2, n_slots=4, rows=3, cols=8, block=4)
    for n, x in kw.items():
        setattr(c, n, x)
    return c


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=5), "dtype"), (dict(format=2), "format"), (dict(n=70000), "n "), (dict(block=257), "block"),
    (dict(n=5), "slots"), (dict(n_slots=0), "slots"), (dict(codes=None), "null"), (dict(x_row=7), "overlap"),
    (dict(x_state=20), "overlap"), (dict(codes=A + 8), "overlap"), (dict(scales=2 * A + 8), "overlap"),
    (dict(scales=3 * A + 1), "aligned"), (dict(rows=1 << 30, cols=16, x_row=16, x_state=1 << 40), "blocks"),
])
def test_cache_block_refused(kw, msg):
    lib = load_library()
    for f in (lib.ssla_state_store, lib.ssla_state_load):
        assert f(C.byref(cache_block(**kw)), A, None) == abi.SSLA_ERR_ARG
        assert msg in lib.ssla_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(groups=3), "groups"), (dict(groups=0), "groups"), (dict(activation="gelu"), "activation"),
    (dict(weight=torch.zeros(7)), "weight"), (dict(bias=torch.zeros(8, dtype=torch.float64)), "bias"),
    (dict(x=torch.zeros(2, 3, 8, dtype=torch.float64)), "x is"), (dict(x=torch.zeros(2, 8, 3).transpose(1, 2)), "channels"),
    (dict(out=torch.zeros(2, 3, 9)), "out"), (dict(), "CUDA"),
])
def test_group_norm_refuses(kw, msg):
    kw = {"x": torch.zeros(2, 3, 8), "groups": 2, **kw}
    with pytest.raises(ValueError, match=msg):
        ops.group_norm(kw.pop("x"), kw.pop("groups"), **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=9), "dtype"), (dict(activation=7), "activation"), (dict(eps=-1.0), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(n=-1), "negative"), (dict(x=None), "null"), (dict(x=A + 1), "aligned"), (dict(y_pos=4), "overlaps itself"),
    (dict(y=A + 4), "overlaps x"), (dict(weight=2 * A), "overlaps weight"), (dict(x_pos=-8), "stride"),
])
def test_group_norm_block_refused(kw, msg):
    a = abi.SslaGroupNorm(x=A, y=2 * A, x_sample=24, x_pos=8, y_sample=24, y_pos=8, n=2, positions=3, channels=8,
                          groups=2, eps=1e-5)
    for n, x in kw.items():
        setattr(a, n, x)
    lib = load_library()
    assert lib.ssla_group_norm(C.byref(a), None, 0, None) == abi.SSLA_ERR_ARG
    assert msg in lib.ssla_last_error().decode()


def test_group_norm_needs_its_workspace():
    a = abi.SslaGroupNorm(x=A, y=1 << 40, x_sample=80 * 64 * 96, x_pos=96, y_sample=80 * 64 * 96, y_pos=96, n=8,
                          positions=80 * 64, channels=96, groups=8, eps=1e-5)
    lib = load_library()
    need = C.c_size_t()
    assert lib.ssla_group_norm_workspace(C.byref(a), C.byref(need)) == abi.SSLA_OK
    if need.value:
        assert lib.ssla_group_norm(C.byref(a), None, 0, None) == abi.SSLA_ERR_ARG
        assert "workspace" in lib.ssla_last_error().decode()
    a.n = 0
    assert lib.ssla_group_norm_workspace(C.byref(a), C.byref(need)) == abi.SSLA_OK and need.value == 0


def test_errors_name_the_code():
    with pytest.raises(SslaError):
        from ssla_rt_b200.engine import _check
        _check(load_library().ssla_linattn_step(None, None, None))


def test_park_refuses_null_arguments():
    lib = load_library()
    assert lib.ssla_engine_park_bytes(None, None) == abi.SSLA_ERR_ARG
    assert lib.ssla_engine_park(None, 0, 0, None, 0, None) == abi.SSLA_ERR_ARG
    assert lib.ssla_engine_resume(None, 0, 0, None, 0, None) == abi.SSLA_ERR_ARG
    from ssla_rt_b200.engine import SslaEngine
    for buf in (None, torch.zeros(8), [0]):
        with pytest.raises(ValueError, match="CUDA tensor"):
            SslaEngine._buffer_bytes(buf)
