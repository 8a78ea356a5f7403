"""Parking a partition's state in 8 bits and resuming it (ssla_engine_park,
ssla_engine_resume): the gates' counters, timestamps, predictions and versions
come back bit for bit, every hidden value within half a step of its cell's
scale, and a resumed stream's gates decide as if it had never been parked."""
import numpy as np
import pytest

from ssla_rt_b200 import abi
from ssla_rt_b200 import events as E
from ssla_rt_b200.engine import SslaEngine, SslaError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def engine(stub_dir, layout, parts=3):
    return SslaEngine(stub_dir(), n_partitions=parts, max_events=6000, layout=layout, max_events_per_partition=4000)


def drain(eng, ev, p):
    counts = [0] * eng.n_partitions
    counts[p] = len(ev)
    eng.drain(torch.from_numpy(np.ascontiguousarray(ev)).cuda(), eng.offsets(counts))
    torch.cuda.synchronize()
    return eng.flags(len(ev)).copy()


def same_but_hidden(a, p, b, q, layout):
    for g in range(4 if layout == abi.LAYOUT_HYBRID else 3):
        np.testing.assert_array_equal(a.counters(g, p), b.counters(g, q))
    np.testing.assert_array_equal(a.last_t(p), b.last_t(q))
    np.testing.assert_array_equal(a.preds_dec(p), b.preds_dec(q))
    np.testing.assert_array_equal(a.preds_raw(p), b.preds_raw(q))
    np.testing.assert_array_equal(a.version(p), b.version(q))


@pytest.mark.parametrize("layout", [abi.LAYOUT_HYBRID, abi.LAYOUT_DECOMP])
@pytest.mark.parametrize("fmt", [abi.FMT_INT8, abi.FMT_E4M3])
def test_park_and_resume(stub_dir, layout, fmt):
    eng = engine(stub_dir, layout)
    ev = E.config_events(0, n=8000)
    drain(eng, ev[:4000], 1)
    buf = torch.full((eng.park_bytes(),), 0x5A, dtype=torch.uint8, device="cuda")
    full = sum(eng.hidden(l, 1).nbytes for l in range(8))
    assert eng.park_bytes() < full / 2
    eng.park(buf, 1, fmt)
    eng.resume(buf, 2, fmt)
    torch.cuda.synchronize()
    same_but_hidden(eng, 1, eng, 2, layout)
    for l in range(8):
        c = eng.CHANS[l // 2]
        h, r = eng.hidden(l, 1).reshape(-1, c), eng.hidden(l, 2).reshape(-1, c)
        amax = np.abs(h).max(1, keepdims=True).astype(np.float64)
        # half a step: of the scale (int8), of the value's own binade or the subnormal step (e4m3);
        # the scale, the quotient and the product are each rounded to 32 bits once
        step = amax / 127 / 2 if fmt == abi.FMT_INT8 else np.maximum(2.0 ** -4 * np.abs(h), amax / 448 * 2.0 ** -10)
        assert (np.abs(r.astype(np.float64) - h) <= step * (1 + 2.0 ** -12) + amax * 2.0 ** -22).all()
        assert (np.abs(h).max(1) == 0).any() or l > 1
        assert (r[np.abs(h).max(1) == 0] == 0).all()
    # the same events from there on: the gates' decisions do not depend on hidden state
    a, b = drain(eng, ev[4000:6000], 1), drain(eng, ev[4000:6000], 2)
    np.testing.assert_array_equal(a, b)
    assert (a & abi.F_R1).any()
    # parked in one engine, resumed in another
    other = engine(stub_dir, layout, parts=1)
    other.resume(buf, 0, fmt)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(drain(other, ev[4000:6000], 0), a)
    for l in range(8):
        np.testing.assert_array_equal(other.hidden(l, 0), eng.hidden(l, 2))
    same_but_hidden(other, 0, eng, 2, layout)
    other.close()
    eng.close()


def test_park_on_a_stream_of_its_own(stub_dir):
    eng = engine(stub_dir, abi.LAYOUT_HYBRID)
    ev = E.config_events(0, n=3000)
    t = torch.from_numpy(np.ascontiguousarray(ev)).cuda()
    buf = torch.zeros(eng.park_bytes(), dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    eng.drain(t, eng.offsets([len(ev), 0, 0]), stream=st)
    eng.park(buf, 0, stream=st)
    eng.resume(buf, 1, stream=st)
    torch.cuda.synchronize()
    same_but_hidden(eng, 0, eng, 1, abi.LAYOUT_HYBRID)
    eng.close()


def test_park_refuses(stub_dir):
    eng = engine(stub_dir, abi.LAYOUT_HYBRID)
    buf = torch.zeros(eng.park_bytes() + 16, dtype=torch.uint8, device="cuda")
    for bad in (lambda: eng.park(buf[:eng.park_bytes() - 1], 0), lambda: eng.park(buf, 3), lambda: eng.park(buf, -1),
                lambda: eng.park(buf, 0, 7), lambda: eng.resume(buf[1:], 0), lambda: eng.resume(buf[:100], 0)):
        with pytest.raises(SslaError) as ei:
            bad()
        assert ei.value.code == abi.SSLA_ERR_ARG
    with pytest.raises(ValueError):
        eng.park(buf[::2], 0)
    eng.close()
