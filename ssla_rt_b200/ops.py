"""Operators on recurrent per-stream state, next to the engine's own layers
(include/ssla_ops.h): linear attention with a decay per head -- chunked over
sequences, and one token per stream --, the 8-bit cache that parks states,
and the channels-last group norm with an activation.

Arguments are torch CUDA tensors.  A call runs on ``stream`` (default: torch's
current stream of the tensors' device), is asynchronous, takes its workspace
from torch's allocator, keeps nothing between calls, and can be captured into
a CUDA graph.  With an explicit ``stream``, ordering against work on other
streams is the caller's, as it is for the engine's drains.  Inference only:
inputs and given outputs that require a gradient are refused while gradients
are enabled, those with a forward-mode tangent always.
Wrong arguments raise ValueError (SslaError where the C entry finds them); there
is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad

from . import abi
from .engine import _check, load_library

_DTYPES = {torch.float32: abi.DT_F32, torch.bfloat16: abi.DT_BF16, torch.float16: abi.DT_F16}
_FORMATS = {torch.int8: abi.FMT_INT8, torch.float8_e4m3fn: abi.FMT_E4M3}
_ACTIVATIONS = {"none": abi.ACT_NONE, None: abi.ACT_NONE, "silu": abi.ACT_SILU}


# What a call's shapes, strides, types and device decide -- its checks and the
# filled argument block -- is kept by exactly those, so that a repeated call
# only sets its pointers (the C entry checks those every time).
_PLANS: dict = {}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _fast_module():
    """The extension module that answers repeated calls (build.py), set up; None where it is not built."""
    try:
        from . import _ops_torch as m
    except ImportError:
        return None
    lib = load_library()
    m.init(_PLANS, *[C.cast(getattr(lib, n), C.c_void_p).value for n in (
        "ssla_linattn_step", "ssla_state_store", "ssla_state_load", "ssla_group_norm", "ssla_group_norm_workspace",
        "ssla_linattn_chunk", "ssla_linattn_chunk_workspace")])
    return m


_fast = _fast_module()


def _keep_plan(key: Optional[bytes], block) -> None:
    """Leaves a checked argument block for the extension module."""
    if key is not None:
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        _PLANS[key] = bytes(block)


def _fast_result(r):
    """What the extension module returned: a negative code is an error of the C entry."""
    if type(r) is int:
        _check(-r)
    return r


def _real(name: str, x) -> float:
    """x's value now: a tensor would be kept, and compared, by what it is rather than by what it holds."""
    try:
        return float(x)
    except (TypeError, ValueError, RuntimeError):
        raise ValueError(f"{name} is {x!r}: a number is needed") from None


def _whole(name: str, x) -> int:
    try:
        return operator.index(x)
    except (TypeError, RuntimeError):
        raise ValueError(f"{name} is {x!r}: a whole number is needed") from None


def _sig(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _plan(key, make):
    p = _PLANS.get(key)
    if p is None:
        p = make()
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        _PLANS[key] = p
    return p


def _tensors(needed: dict, **optional) -> None:
    for given, may_lack in ((needed, False), (optional, True)):
        for name, t in given.items():
            if not isinstance(t, torch.Tensor) and not (may_lack and t is None):
                raise ValueError(f"{name} is {type(t).__name__}: a tensor is needed")


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("inference only: an input or a given output requires a gradient")
    level = forward_ad._current_level
    if level >= 0:
        for t in tensors:
            if t is not None and torch._VF._unpack_dual(t, level=level)[1] is not None:
                raise ValueError("inference only: an input or a given output has a forward-mode tangent")


def _written(*tensors) -> None:
    """Tells autograd that these were changed in place, as torch's own operators do."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _device(first: torch.Tensor, **others) -> int:
    """The CUDA device index that every given tensor is on."""
    dev = first.device
    for name, t in others.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, not {dev}")
    if dev.type != "cuda":
        raise ValueError(f"CUDA tensors are needed, got {dev}")
    return dev.index


def _stream_of(stream, device: int):
    """(handle to launch on, torch stream to allocate and synchronise with, or None for the current one)."""
    if stream is None:
        if _raw_stream is not None:
            return _raw_stream(device), None
        return torch.cuda.current_stream(device).cuda_stream, None
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(getattr(stream, "cuda_stream", stream)), device=device)
    return stream.cuda_stream, stream


def _keep(ts, *tensors) -> None:
    """On an explicit stream other than the current one: the tensors' memory
    is not handed out again before the work enqueued there is done."""
    if ts is not None and ts != torch.cuda.current_stream(ts.device):
        for t in tensors:
            if t is not None:
                t.record_stream(ts)


def _like(x: torch.Tensor, stream, zero: bool = False) -> torch.Tensor:
    """A new contiguous tensor of x's shape that belongs to the launch's stream."""
    make = torch.zeros_like if zero else torch.empty_like
    if stream is None:
        return make(x, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return make(x, memory_format=torch.contiguous_format)


def _new(x: torch.Tensor, shape, dtype, stream) -> torch.Tensor:
    if stream is None:
        return x.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return x.new_empty(shape, dtype=dtype)


def _counts(name: str, t: Optional[torch.Tensor]) -> None:
    """An argument block counts in 32 bits, and ctypes would wrap what does not fit."""
    if t is not None and t.dim() and max(t.shape) > 2**31 - 1:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: sizes are below 2^31")


def _rows_heads(name: str, t: torch.Tensor, dtype=None) -> None:
    if t.dim() != 3:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: (rows, heads, width) is needed")
    _counts(name, t)
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}, not {dtype}")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}'s last dimension is not contiguous")


def _host_ints(name: str, x) -> np.ndarray:
    """A host array of int32 (as a drain's part_offsets)."""
    if isinstance(x, torch.Tensor):
        if x.device.type != "cpu":
            raise ValueError(f"{name} is a host array")
        x = x.numpy()
    if type(x) is np.ndarray and x.dtype == np.int32 and x.ndim == 1 and x.flags.c_contiguous:
        return x
    a = np.asarray(x)
    if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
        raise ValueError(f"{name} is a one-dimensional array of integers")
    if a.dtype != np.int32:
        if a.size and (a.max() > 2**31 - 1 or a.min() < -2**31):
            raise ValueError(f"{name} does not fit 32 bits")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


def _device_slots(slots: Optional[torch.Tensor], n: int) -> None:
    if slots is None:
        return
    if not isinstance(slots, torch.Tensor) or slots.dtype != torch.int32 or slots.dim() != 1:
        raise ValueError("slots is a one-dimensional int32 tensor")
    if slots.shape[0] != n or (n > 1 and slots.stride(0) != 1):
        raise ValueError(f"slots has shape {tuple(slots.shape)}: {n} contiguous entries are needed")


def _linattn_block(q, k, v, decay, state, scale, out, step_slots=None):
    """Checks what both forms share; the argument block without its pointers."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _rows_heads(name, t, v.dtype)
    if v.dtype not in _DTYPES:
        raise ValueError(f"{v.dtype} is not supported: float32, bfloat16 or float16")
    n, heads, dv = v.shape
    dk = q.shape[2]
    if q.shape[0] != n or k.shape[0] != n or k.shape[2] != dk:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    if decay.dtype != torch.float32 or tuple(decay.shape) not in ((heads,), (n, heads)):
        raise ValueError(f"decay is {decay.dtype} {tuple(decay.shape)}: float32 ({heads},) or ({n}, {heads}) is needed")
    a = abi.SslaLinAttn()
    _counts("state", state)
    if state is not None:
        if state.dtype != torch.float32 or state.dim() != 4 or tuple(state.shape[1:]) != (heads, dk, dv):
            raise ValueError(f"state is {state.dtype} {tuple(state.shape)}: float32 (slots, {heads}, {dk}, {dv}) is needed")
        if not state.is_contiguous():
            raise ValueError("state is not contiguous")
        a.n_slots = state.shape[0]
    if out is not None:
        _rows_heads("out", out, v.dtype)
        if out.shape != v.shape:
            raise ValueError(f"out has shape {tuple(out.shape)}, not {tuple(v.shape)}")
        a.out_row, a.out_head, _ = out.stride()
    else:
        a.out_row, a.out_head = heads * dv, dv
    _device_slots(step_slots, n)
    a.device = _device(q, k=k, v=v, decay=decay, state=state, out=out, slots=step_slots)
    a.q_row, a.q_head, _ = q.stride()
    a.k_row, a.k_head, _ = k.stride()
    a.v_row, a.v_head, _ = v.stride()
    if decay.dim() == 2:
        a.decay_row, a.decay_head = decay.stride()
    else:
        a.decay_head = decay.stride(0)
    a.n_rows, a.heads, a.q_heads, a.k_heads, a.dk, a.dv = n, heads, q.shape[1], k.shape[1], dk, dv
    a.dtype = _DTYPES[v.dtype]
    a.scale = scale
    return a


def _linattn(q, k, v, decay, state, scale, out, slots=None):
    """The checked argument block of a call with every pointer but out's."""
    _no_grad(q, k, v, decay, state, out)
    scale = _real("scale", scale)
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(),
           v.shape, v.stride(), v.dtype, v.get_device(), decay.shape, decay.stride(), decay.dtype, decay.get_device(),
           scale, _sig(state), _sig(out), _sig(slots))
    a = abi.SslaLinAttn.from_buffer_copy(
        _plan(key, lambda: _linattn_block(q, k, v, decay, state, scale, out, slots)))
    a.q, a.k, a.v, a.decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr()
    if state is not None:
        a.state = state.data_ptr()
    return a


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, *,
                     state: Optional[torch.Tensor] = None, offsets: Optional[Sequence[int]] = None,
                     lengths: Optional[Sequence[int]] = None, slots: Optional[Sequence[int]] = None,
                     scale: float = 1.0, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Linear attention with a decay per head over whole sequences.

    Per head, token by token: ``S = exp(decay) * S + outer(k, v)`` and
    ``out = scale * (q @ S)``.

    q, k: (rows, heads or a divisor of them, dk); v: (rows, heads, dv); any row
    and head strides, last dimension contiguous; float32, bfloat16 or float16.
    decay: float32 logarithms, at most 0, (heads,) or (rows, heads); -inf
    clears the state, whatever it holds.
    Sequence i is rows offsets[i] : offsets[i + 1], or lengths[i] rows from
    offsets[i] (a padded batch); one sequence of all rows without offsets.
    state: (slots, heads, dk, dv) float32, contiguous: sequence i starts from
    and updates state[slots[i]] (state[i] without slots, no state for -1);
    without state, from zero.  offsets, lengths and slots are host arrays.
    Returns out, (rows, heads, dv); rows outside every sequence are zero in a
    new tensor and left as they were in a given one.
    """
    if _fast is not None and stream is None:
        r = _fast.chunk(q, k, v, decay, state, scale, out, offsets, lengths, slots, False)
        if r is not None:
            return _fast_result(r)
    given = out
    _tensors({"q": q, "k": k, "v": v, "decay": decay}, state=state, out=out)
    if v.dim() != 3:
        raise ValueError(f"v has shape {tuple(v.shape)}: (rows, heads, width) is needed")
    _counts("v", v)
    if offsets is None:
        if lengths is not None:
            raise ValueError("lengths without offsets")
        off = np.array([0, v.shape[0]], dtype=np.int32)
        n_seq, gaps = 1, False
    else:
        off = _host_ints("offsets", offsets)
        if lengths is None:
            if off.size < 1:
                raise ValueError("offsets is empty")
            n_seq = off.size - 1
            gaps = bool(n_seq == 0 or off[0] != 0 or off[-1] != v.shape[0])
        else:
            lengths = _host_ints("lengths", lengths)
            n_seq = off.size
            if lengths.size != n_seq:
                raise ValueError(f"{lengths.size} lengths for {n_seq} offsets")
            gaps = int(lengths.sum(dtype=np.int64)) != v.shape[0]
    if slots is not None:
        slots = _host_ints("slots", slots)
        if slots.size != n_seq:
            raise ValueError(f"{slots.size} slots for {n_seq} sequences")
    a = _linattn(q, k, v, decay, state, scale, out)
    if _fast is not None:
        _keep_plan(_fast.chunk(q, k, v, decay, state, scale, given, None, None, None, True), a)
    handle, ts = _stream_of(stream, a.device)
    if out is None:
        out = _like(v, ts, zero=gaps)
    a.out = out.data_ptr()
    lib = load_library()
    po, pl = off.ctypes.data, lengths.ctypes.data if lengths is not None else None
    need = C.c_size_t()
    _check(lib.ssla_linattn_chunk_workspace(C.byref(a), po, pl, n_seq, C.byref(need)))
    ws = _new(v, (need.value,), torch.uint8, ts) if need.value else None
    _check(lib.ssla_linattn_chunk(C.byref(a), po, pl, slots.ctypes.data if slots is not None else None, n_seq,
                                  ws.data_ptr() if ws is not None else None, need.value, handle))
    _written(state, given)
    if ts is not None:
        _keep(ts, q, k, v, decay, state, out)
    return out


def linear_attention_status(device: int = 0) -> int:
    """Status bits of linear_attention's kernels on a device since the last
    call (0: fine; 1: a bounded wait ran out and results since are not valid).
    Synchronises the device."""
    st = C.c_uint(0)
    _check(load_library().ssla_linattn_status(device, C.byref(st)))
    return st.value


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor,
                          state: torch.Tensor, *, slots: Optional[torch.Tensor] = None, scale: float = 1.0,
                          out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """One token for each row (``linear_attention`` for sequences of one token,
    with the slots on the device, so that a captured graph can be replayed for
    other streams).

    Row r updates state[slots[r]] (slots: int32 CUDA tensor; state[r] without).
    Rows that name the same slot are applied in row order; a slot outside the
    state marks a padding row: zero output, no state touched.
    """
    if _fast is not None and stream is None:
        r = _fast.step(q, k, v, decay, state, slots, scale, out, False)
        if r is not None:
            return _fast_result(r)
    given = out
    if state is None:
        raise ValueError("state is needed")
    _tensors({"q": q, "k": k, "v": v, "decay": decay, "state": state}, out=out)
    if slots is not None and not isinstance(slots, torch.Tensor):
        raise ValueError("slots is a one-dimensional int32 tensor")
    a = _linattn(q, k, v, decay, state, scale, out, slots)
    if _fast is not None:
        _keep_plan(_fast.step(q, k, v, decay, state, slots, scale, given, True), a)
    handle, ts = _stream_of(stream, a.device)
    if out is None:
        out = _like(v, ts)
    a.out = out.data_ptr()
    _check(load_library().ssla_linattn_step(C.byref(a), slots.data_ptr() if slots is not None else None, handle))
    _written(state, given)
    if ts is not None:
        _keep(ts, q, k, v, decay, state, slots, out)
    return out


def state_cache(n_slots: int, rows: int, cols: int, *, block: int = 64, dtype: torch.dtype = torch.int8,
                device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of an empty cache: every slot reads back as zeros."""
    if dtype not in _FORMATS:
        raise ValueError(f"{dtype} is not supported: int8 or float8_e4m3fn")
    if block < 1:
        raise ValueError(f"block {block}")
    codes = torch.zeros((n_slots, rows, cols), dtype=torch.int8, device=device).view(dtype)
    return codes, torch.zeros((n_slots, rows, -(-cols // block)), dtype=torch.float32, device=device)


def _cache_block(codes, scales, block, slots, n, name, x, dtype):
    """Checks a store or load; the argument block without its pointers."""
    if codes.dtype not in _FORMATS or codes.dim() != 3 or not codes.is_contiguous():
        raise ValueError("codes is a contiguous (slots, rows, cols) tensor of int8 or float8_e4m3fn")
    _counts("codes", codes)
    _counts(name, x)
    if not 1 <= block <= 256:
        raise ValueError(f"block {block} must be 1..256")
    n_slots, rows, cols = codes.shape
    if (scales.dtype != torch.float32 or tuple(scales.shape) != (n_slots, rows, -(-cols // block)) or
            not scales.is_contiguous()):
        raise ValueError(f"scales is {scales.dtype} {tuple(scales.shape)}: contiguous float32 "
                         f"({n_slots}, {rows}, {-(-cols // block)}) is needed")
    _device_slots(slots, n)
    c = abi.SslaStateCache()
    c.n, c.n_slots, c.rows, c.cols, c.block = n, n_slots, rows, cols, block
    c.format = _FORMATS[codes.dtype]
    if x is not None:
        if x.dtype not in _DTYPES or x.dim() != 3 or tuple(x.shape[1:]) != (rows, cols):
            raise ValueError(f"{name} is {x.dtype} {tuple(x.shape)}: (states, {rows}, {cols}) of float32, bfloat16 "
                             f"or float16 is needed")
        if cols > 1 and x.stride(2) != 1:
            raise ValueError(f"{name}'s last dimension is not contiguous")
        c.x_state, c.x_row, _ = x.stride()
    else:
        c.x_state, c.x_row = rows * cols, cols
    if dtype not in _DTYPES:
        raise ValueError(f"{dtype} is not supported: float32, bfloat16 or float16")
    c.dtype = _DTYPES[dtype]
    c.device = _device(codes, scales=scales, slots=slots, **{name: x})
    return c


def _cache(codes, scales, block, slots, n, name, x, dtype):
    if slots is not None and not isinstance(slots, torch.Tensor):
        raise ValueError("slots is a one-dimensional int32 tensor")
    _no_grad(x, scales)
    block = _whole("block", block)
    key = ("cache", _sig(codes), _sig(scales), block, _sig(slots), n, name, _sig(x), dtype)
    c = abi.SslaStateCache.from_buffer_copy(
        _plan(key, lambda: _cache_block(codes, scales, block, slots, n, name, x, dtype)))
    c.codes, c.scales = codes.data_ptr(), scales.data_ptr()
    if slots is not None:
        c.slots = slots.data_ptr()
    return c


def state_store(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, *, block: int = 64,
                slots: Optional[torch.Tensor] = None, stream=None) -> None:
    """Quantises states into the 8-bit cache as they are written.

    x: (states, rows, cols), no two of them in one place; codes: (slots, rows, cols) int8 or float8_e4m3fn;
    scales: (slots, rows, ceil(cols / block)) float32.  State i goes to slot
    slots[i] (int32 CUDA tensor; slot i without).  Each ``block`` values of a
    row share scale = max|x| / 127 (int8) or / 448 (e4m3); a code is x / scale,
    nearest, ties to even.  Slots outside the cache are skipped; where a slot
    is named twice the last state is kept; other slots stay as they were.  A
    block with a non-finite value reads back as NaN.
    """
    if _fast is not None and stream is None:
        r = _fast.store(x, codes, scales, block, slots, False)
        if r is not None:
            return _check(-r)
    _tensors({"x": x, "codes": codes, "scales": scales})
    if x.dim() == 0:
        raise ValueError("x has no dimensions: (states, rows, cols) is needed")
    c = _cache(codes, scales, block, slots, x.shape[0], "x", x, x.dtype)
    if _fast is not None:
        _keep_plan(_fast.store(x, codes, scales, block, slots, True), c)
    handle, ts = _stream_of(stream, c.device)
    _check(load_library().ssla_state_store(C.byref(c), x.data_ptr(), handle))
    _written(codes, scales)
    if ts is not None:
        _keep(ts, x, codes, scales, slots)


def state_load(codes: torch.Tensor, scales: torch.Tensor, *, block: int = 64, slots: Optional[torch.Tensor] = None,
               dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Reads states back from the 8-bit cache: (states, rows, cols), state i
    from slot slots[i] (every slot in order without); a slot outside the cache
    gives zeros."""
    code = _DTYPES.get(dtype if out is None else getattr(out, "dtype", None), -1)
    if _fast is not None and stream is None:
        r = _fast.load(codes, scales, block, slots, code, out, False)
        if r is not None:
            return _fast_result(r)
    given = out
    _tensors({"codes": codes, "scales": scales}, out=out)
    if slots is not None and not isinstance(slots, torch.Tensor):
        raise ValueError("slots is a one-dimensional int32 tensor")
    if not all(t.dim() for t in (codes, slots, out) if t is not None):
        raise ValueError("codes, slots and out have at least one dimension")
    if out is not None:
        n, dtype = out.shape[0], out.dtype
    else:
        n = slots.shape[0] if slots is not None else codes.shape[0]
    c = _cache(codes, scales, block, slots, n, "out", out, dtype)
    if _fast is not None:
        _keep_plan(_fast.load(codes, scales, block, slots, code, out, True), c)
    handle, ts = _stream_of(stream, c.device)
    if out is None:
        out = _new(codes, (n, c.rows, c.cols), dtype, ts)
    _check(load_library().ssla_state_load(C.byref(c), out.data_ptr(), handle))
    _written(given)
    if ts is not None:
        _keep(ts, codes, scales, slots, out)
    return out


def _norm_block(x, groups, weight, bias, eps, activation, out):
    if x.dtype not in _DTYPES or x.dim() != 3:
        raise ValueError(f"x is {x.dtype} {tuple(x.shape)}: (samples, positions, channels) or (rows, channels) of "
                         f"float32, bfloat16 or float16 is needed")
    _counts("x", x)
    n, positions, channels = x.shape
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: silu or none")
    if groups < 1 or channels % groups:
        raise ValueError(f"{channels} channels in {groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (channels,) or not t.is_contiguous()):
            raise ValueError(f"{name} is {t.dtype} {tuple(t.shape)}: contiguous float32 ({channels},) is needed")
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype):
        raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, x {x.dtype} {tuple(x.shape)}")
    for name, t in (("x", x), ("out", out)):
        if t is not None and channels > 1 and t.stride(2) != 1:
            raise ValueError(f"{name}'s channels are not contiguous")
    a = abi.SslaGroupNorm()
    a.device = _device(x, weight=weight, bias=bias, out=out)
    a.x_sample, a.x_pos, _ = x.stride()
    if out is not None:
        a.y_sample, a.y_pos, _ = out.stride()
    else:
        a.y_sample, a.y_pos = positions * channels, channels
    a.n, a.positions, a.channels, a.groups = n, positions, channels, groups
    a.dtype, a.activation, a.eps = _DTYPES[x.dtype], _ACTIVATIONS[activation], eps
    return a


def group_norm(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5, activation: Optional[str] = "silu",
               out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Group norm with an activation, channels last.

    x: (samples, positions, channels), channels contiguous, any other strides;
    (rows, channels) is rows of one position each, so that with one group per
    head it normalises linear_attention's output rows.  Statistics over a
    sample's positions and the channels of a group; weight, bias: (channels,)
    float32.  activation: "silu" or "none".  ``out`` may be x.
    """
    act = _ACTIVATIONS.get(activation, -1)
    if _fast is not None and stream is None:
        r = _fast.norm(x, groups, weight, bias, eps, act, out, False)
        if r is not None:
            return _fast_result(r)
    _tensors({"x": x}, weight=weight, bias=bias, out=out)
    if x.dim() == 2:
        if out is not None and out.shape != x.shape:
            raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, x {x.dtype} {tuple(x.shape)}")
        y = group_norm(x[:, None], groups, weight, bias, eps=eps, activation=activation,
                       out=None if out is None else out[:, None], stream=stream)
        return y[:, 0] if out is None else out
    _no_grad(x, weight, bias, out)
    groups, eps = _whole("groups", groups), _real("eps", eps)
    given = out
    key = ("norm", _sig(x), groups, _sig(weight), _sig(bias), eps, activation, _sig(out))
    a = abi.SslaGroupNorm.from_buffer_copy(
        _plan(key, lambda: _norm_block(x, groups, weight, bias, eps, activation, out)))
    if _fast is not None:
        _keep_plan(_fast.norm(x, groups, weight, bias, eps, act, given, True), a)
    handle, ts = _stream_of(stream, a.device)
    if out is None:
        out = _like(x, ts)
    a.x, a.y = x.data_ptr(), out.data_ptr()
    if weight is not None:
        a.weight = weight.data_ptr()
    if bias is not None:
        a.bias = bias.data_ptr()
    lib = load_library()
    need = C.c_size_t()
    _check(lib.ssla_group_norm_workspace(C.byref(a), C.byref(need)))
    ws = _new(x, (need.value,), torch.uint8, ts) if need.value else None
    _check(lib.ssla_group_norm(C.byref(a), ws.data_ptr() if ws is not None else None, need.value, handle))
    _written(given)
    if ts is not None:
        _keep(ts, x, weight, bias, out)
    return out
