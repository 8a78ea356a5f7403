"""Measured cases of the recurrent-state operators: linear attention with a
decay per head (chunked over prompts, and one token at a time), the 8-bit
cache that parks per-stream states, and the channels-last group norm with an
activation that follows the attention.

``run`` computes a case in elementary torch operations, or, with ``own`` set,
through ssla_rt_b200.ops on the same inputs.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


def listed():
    return [
        # -- chunked linear attention -------------------------------------------------
        # eight event streams drained together (25,000 events each, 96 channels as 4
        # heads of 24), continuing from each stream's state
        {"name": "streams fp32 4x24", "op": "attention", "dtype": "fp32", "n_seq": 8, "lo": 25000, "hi": 25000,
         "heads": 4, "qk_heads": 4, "dk": 24, "dv": 24, "gated": True},
        # a batch of prompts of uneven length, heads of 128, a fixed decay for each head
        {"name": "prompts bf16 16x128", "op": "attention", "dtype": "bf16", "n_seq": 8, "lo": 511, "hi": 4096,
         "heads": 16, "qk_heads": 16, "dk": 128, "dv": 128, "gated": False},
        # one long recording, few heads: the parallel work has to come from its length
        {"name": "long bf16 4x64", "op": "attention", "dtype": "bf16", "n_seq": 1, "lo": 65537, "hi": 65537,
         "heads": 4, "qk_heads": 4, "dk": 64, "dv": 64, "gated": True},
        # a handful of short prompts, queries and keys shared by pairs of heads: latency
        {"name": "short fp16 8x64x96", "op": "attention", "dtype": "fp16", "n_seq": 5, "lo": 1, "hi": 77,
         "heads": 8, "qk_heads": 4, "dk": 64, "dv": 96, "gated": True},
        # -- one token per stream -------------------------------------------------------
        # 64 live streams, the small heads of the event network
        {"name": "step fp32 64 rows 4x24", "op": "step", "dtype": "fp32", "rows": 64, "slots": 80,
         "heads": 4, "qk_heads": 4, "dk": 24, "dv": 24, "gated": True},
        # a large serving batch: the states' traffic is everything
        {"name": "step bf16 256 rows 16x128", "op": "step", "dtype": "bf16", "rows": 256, "slots": 300,
         "heads": 16, "qk_heads": 16, "dk": 128, "dv": 128, "gated": True},
        # a single stream: the smallest call
        {"name": "step bf16 1 row 8x64", "op": "step", "dtype": "bf16", "rows": 1, "slots": 4,
         "heads": 8, "qk_heads": 8, "dk": 64, "dv": 64, "gated": False},
        # -- states parked in 8 bits ------------------------------------------------------
        # matrix states of 192 streams (16 heads of 128 x 128) written as e4m3
        {"name": "park e4m3 192x2048x128", "op": "park", "dtype": "fp32", "format": "e4m3", "n": 192, "slots": 200,
         "rows": 2048, "cols": 128, "block": 64},
        # one layer's hidden state of 64 streams (80 x 64 cells of 12 channels), parked and resumed
        {"name": "park+resume int8 64x5120x12", "op": "both", "dtype": "fp32", "format": "int8", "n": 64, "slots": 64,
         "rows": 5120, "cols": 12, "block": 12},
        # parked matrix states read back, with rows of an odd length
        {"name": "resume int8 37x1000x99", "op": "resume", "dtype": "bf16", "format": "int8", "n": 37, "slots": 50,
         "rows": 1000, "cols": 99, "block": 32},
        # -- group norm + SiLU -------------------------------------------------------------
        # the attention's output rows, one group per head
        {"name": "head norm bf16 16384x2048", "op": "norm", "dtype": "bf16", "n": 16384, "positions": 1,
         "channels": 2048, "groups": 16, "activation": "silu"},
        # feature maps of eight sensors (80 x 64 cells of 96 channels)
        {"name": "map norm fp32 8x5120x96", "op": "norm", "dtype": "fp32", "n": 8, "positions": 5120,
         "channels": 96, "groups": 8, "activation": "silu"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "step", "park", "resume", "both", "norm"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("attention", "step"):
        qk = rng.choice([1, 2, 3, 4, 6, 8])
        heads = qk * rng.choice([1, 1, 2])
        dk, dv = _log_int(rng, 8, 128), _log_int(rng, 8, 192)
        c = {"op": op, "dtype": dtype, "heads": heads, "qk_heads": qk, "dk": dk, "dv": dv, "gated": rng.random() < 0.6}
        if op == "step":
            rows = _log_int(rng, 1, 300)
            return {**c, "rows": rows, "slots": rows + rng.randint(0, 40)}
        # bounded so that tokens x heads x (dk + dv) stays within the listed cases
        total = _log_int(rng, 1, max(64, min(60000, 30_000_000 // (heads * (dk + dv)))))
        n_seq = min(_log_int(rng, 1, 40), total)
        hi = max(1, total // n_seq)
        return {**c, "n_seq": n_seq, "lo": max(1, _log_int(rng, 1, hi)), "hi": hi}
    if op == "norm":
        groups = rng.choice([1, 2, 3, 4, 8, 16])
        channels = groups * _log_int(rng, 1, 128)
        positions = rng.choice([1, _log_int(rng, 2, 20000)])
        n = _log_int(rng, 1, max(2, 20_000_000 // (positions * channels)))
        return {"op": "norm", "dtype": dtype, "n": min(n, 16384), "positions": positions, "channels": channels,
                "groups": groups, "activation": rng.choice(["silu", "none"])}
    rows, cols = _log_int(rng, 1, 4000), _log_int(rng, 4, 200)
    n = max(1, min(_log_int(rng, 1, 200), 20_000_000 // (rows * cols)))
    return {"op": op, "dtype": dtype, "format": rng.choice(["e4m3", "int8"]), "n": n, "slots": n + rng.randint(0, 9),
            "rows": rows, "cols": cols, "block": rng.choice([8, 12, 16, 32, 64, 128])}


def _lengths(case):
    """Sequence lengths between lo and hi, the first the longest (fixed by the case, so that a pass's work is too)."""
    n, lo, hi = case["n_seq"], case["lo"], case["hi"]
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, std=1.0):
        return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)

    s = {"case": dict(case)}
    if case["op"] in ("attention", "step"):
        h, hq, dk, dv = case["heads"], case["qk_heads"], case["dk"], case["dv"]
        if case["op"] == "attention":
            length = np.array(_lengths(case), dtype=np.int32)
            offsets = np.concatenate([[0], np.cumsum(length)]).astype(np.int32)
            n, slots = int(offsets[-1]), len(length)
            s |= {"offsets": offsets, "starts": torch.tensor(offsets[:-1], device=DEV, dtype=torch.int64),
                  "length": torch.tensor(length, device=DEV, dtype=torch.int64), "longest": int(length.max())}
        else:
            n, slots = case["rows"], case["slots"]
            s["slots"] = torch.randperm(slots, generator=gen, device=DEV)[:n].to(torch.int32)
        # queries and keys of about unit length, values of unit variance
        s |= {"q": normal(n, hq, dk, std=dk ** -0.25), "k": normal(n, hq, dk, std=dk ** -0.25), "v": normal(n, h, dv)}
        if case["gated"]:   # a gate for each token and head, as sigmoid gates give it
            s["decay"] = torch.nn.functional.logsigmoid(2.5 + 1.5 * torch.randn((n, h), generator=gen, device=DEV))
        else:               # a fixed decay for each head, from short memories to long ones
            s["decay"] = torch.log1p(-torch.exp2(-3.0 - 5.0 * torch.rand((h,), generator=gen, device=DEV)))
        s["state"] = normal(slots, h, dk, dv, dtype=torch.float32)
        s["scale"] = dk ** -0.5
        return s
    if case["op"] == "norm":
        c = case["channels"]
        s["x"] = (torch.randn((case["n"], case["positions"], c), generator=gen, device=DEV) * 1.5 + 0.25).to(dt)
        s["weight"] = 1.0 + 0.2 * normal(c, dtype=torch.float32)
        s["bias"] = 0.1 * normal(c, dtype=torch.float32)
        return s
    rows, cols, block, slots = case["rows"], case["cols"], case["block"], case["slots"]
    code_t = torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn
    s["slots"] = torch.randperm(slots, generator=gen, device=DEV)[:case["n"]].to(torch.int32)
    s["x"] = normal(case["n"], rows, cols)
    blocks = -(-cols // block)
    if case["op"] == "resume":
        s["codes"] = (torch.randint(-127, 128, (slots, rows, cols), generator=gen, device=DEV, dtype=torch.int8)
                      if code_t == torch.int8 else
                      (80 * torch.randn((slots, rows, cols), generator=gen, device=DEV)).clamp(-448, 448).to(code_t))
        s["scales"] = torch.rand((slots, rows, blocks), generator=gen, device=DEV) * 0.05 + 0.001
    else:
        s["codes"] = torch.zeros((slots, rows, cols), device=DEV, dtype=torch.int8).view(code_t)
        s["scales"] = torch.zeros((slots, rows, blocks), device=DEV)
    return s


# ---- plain forms -----------------------------------------------------------------------


def _heads(x, h):
    return x.float().repeat_interleave(h // x.shape[-2], dim=-2)


def _plain_attention(s, chunk=64):
    q, k, v, state = s["q"], s["k"], s["v"], s["state"]
    n, h, dv = v.shape
    dk, p = q.shape[-1], s["starts"].numel()
    m = -(-s["longest"] // chunk)                                   # chunks of the longest sequence
    at = torch.arange(m * chunk, device=q.device)
    live = at < s["length"][:, None]                                # (p, m * chunk)
    index = (s["starts"][:, None] + at).clamp(max=n - 1)
    decay = s["decay"].double().expand(n, h)

    def laid(x, width):                                              # (p, m, h, chunk, width)
        x = torch.where(live[..., None, None], x[index], 0)
        return x.reshape(p, m, chunk, h, width).transpose(2, 3)

    qc, kc, vc = laid(_heads(q, h), dk), laid(_heads(k, h), dk), laid(v.float(), dv)
    g = laid(decay[..., None], 1)[..., 0].cumsum(-1)                 # (p, m, h, chunk)
    causal = torch.ones(chunk, chunk, device=q.device, dtype=torch.bool).tril()
    d = torch.where(causal, g[..., :, None] - g[..., None, :], -math.inf).exp().float()
    inner = ((qc @ kc.transpose(-1, -2)) * d) @ vc
    end = g[..., -1:]
    local = (kc * (end - g).exp().float()[..., None]).transpose(-1, -2) @ vc   # (p, m, h, dk, dv)
    # every chunk's first state: the initial one and the earlier chunks' own, decayed to there
    e = torch.cat([torch.zeros_like(end[:, :1, :, 0]), end[..., 0].cumsum(1)], 1)      # (p, m + 1, h)
    e = e.transpose(1, 2)                                            # (p, h, m + 1)
    before = torch.ones(m + 1, m + 1, device=q.device, dtype=torch.bool).tril()
    w = torch.where(before, e[..., :, None] - e[..., None, :], -math.inf).exp().float()
    parts = torch.cat([state[:, None], local], 1).transpose(1, 2).reshape(p, h, m + 1, dk * dv)
    first = (w @ parts).reshape(p, h, m + 1, dk, dv)
    outer = g.exp().float()[..., None] * (qc @ first[:, :, :m].transpose(1, 2))
    o = ((inner + outer) * s["scale"]).transpose(2, 3).reshape(p, m * chunk, h, dv)
    state.copy_(first[:, :, m])
    out = torch.empty_like(v)
    out[index[live]] = o[live].to(v.dtype)
    return {"out": out, "state": state}


def _plain_step(s):
    q, k, v, state, slots = s["q"], s["k"], s["v"], s["state"], s["slots"].long()
    h = v.shape[1]
    a = s["decay"].exp().expand(v.shape[0], h)[..., None, None]
    new = a * state[slots] + _heads(k, h)[..., None] * v.float()[..., None, :]
    o = (_heads(q, h)[..., None] * new).sum(-2) * s["scale"]
    state[slots] = new
    return {"out": o.to(v.dtype), "state": state}


def _blocks(x, block):
    pad = -x.shape[-1] % block
    x = torch.nn.functional.pad(x, (0, pad))
    return x.reshape(*x.shape[:-1], -1, block)


def _plain_park(s):
    x, codes, scales, slots = s["x"], s["codes"], s["scales"], s["slots"].long()
    block, cols = s["case"]["block"], x.shape[-1]
    most = 127.0 if codes.dtype == torch.int8 else 448.0
    xb = _blocks(x.float(), block)
    scale = (xb.abs().amax(-1).double() / most).float()
    quotient = torch.where(scale[..., None] > 0, xb / scale[..., None], 0.0)
    quotient = quotient.clamp(-most, most).flatten(-2)[..., :cols]
    new = quotient.round().to(torch.int8) if codes.dtype == torch.int8 else quotient.to(codes.dtype)
    codes.view(torch.int8)[slots] = new.view(torch.int8)
    scales[slots] = scale
    return {"codes": codes, "scales": scales}


def _plain_resume(s):
    codes, scales, slots = s["codes"].view(torch.int8), s["scales"], s["slots"].long()
    block, cols = s["case"]["block"], codes.shape[-1]
    values = codes[slots].view(s["codes"].dtype).float()
    spread = scales[slots].repeat_interleave(block, -1)[..., :cols]
    return (values * spread).to(s["x"].dtype)


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    n, p, ch = x.shape
    xg = x.reshape(n, p, c["groups"], ch // c["groups"])
    mean = xg.double().mean((1, 3), keepdim=True).float()
    xg = xg - mean
    var = xg.square().mean((1, 3), keepdim=True)
    y = (xg / (var + 1e-5).sqrt()).reshape(n, p, ch) * s["weight"] + s["bias"]
    if c["activation"] == "silu":
        y = y / (1 + (-y).exp())
    return y.to(s["x"].dtype)


def run(s):
    op = s["case"]["op"]
    if own:
        from ssla_rt_b200 import ops
        if op == "attention":
            out = ops.linear_attention(s["q"], s["k"], s["v"], s["decay"], state=s["state"], offsets=s["offsets"],
                                       scale=s["scale"])
            return {"out": out, "state": s["state"]}
        if op == "step":
            out = ops.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], slots=s["slots"],
                                            scale=s["scale"])
            return {"out": out, "state": s["state"]}
        if op == "norm":
            c = s["case"]
            return ops.group_norm(s["x"], c["groups"], s["weight"], s["bias"], eps=1e-5, activation=c["activation"])
        block = s["case"]["block"]
        if op in ("park", "both"):
            ops.state_store(s["x"], s["codes"], s["scales"], block=block, slots=s["slots"])
        if op in ("resume", "both"):
            values = ops.state_load(s["codes"], s["scales"], block=block, slots=s["slots"], dtype=s["x"].dtype)
            return values if op == "resume" else {"values": values, "scales": s["scales"]}
        return {"codes": s["codes"], "scales": s["scales"]}
    if op == "attention":
        return _plain_attention(s)
    if op == "step":
        return _plain_step(s)
    if op == "norm":
        return _plain_norm(s)
    if op == "resume":
        return _plain_resume(s)
    parked = _plain_park(s)
    return parked if op == "park" else {"values": _plain_resume(s), "scales": s["scales"]}


# ---- the definitions in 64 bits ---------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("attention", "step"):
        return _exact_attention(s)
    if case["op"] == "norm":
        x = s["x"].double()
        y = torch.empty_like(x)
        width = case["channels"] // case["groups"]
        for g in range(case["groups"]):
            part = x[:, :, g * width:(g + 1) * width]
            centred = part - part.mean(dim=(1, 2), keepdim=True)
            y[:, :, g * width:(g + 1) * width] = centred * (centred.pow(2).mean(dim=(1, 2), keepdim=True) + 1e-5).rsqrt()
        y = y * s["weight"].double() + s["bias"].double()
        return y * torch.sigmoid(y) if case["activation"] == "silu" else y
    return _exact_cache(s)


def _exact_attention(s):
    """The recurrence itself, one token of every sequence at a time."""
    q, k, v, decay, state = (s[n].double() for n in ("q", "k", "v", "decay", "state"))
    rows, h, _ = v.shape
    share = h // q.shape[1]
    decay = decay.expand(rows, h)
    out = torch.zeros_like(v)
    if s["case"]["op"] == "attention":
        offsets = [int(x) for x in s["offsets"]]
        order = [(offsets[i + 1] - offsets[i], i) for i in range(len(offsets) - 1)]
        where = torch.arange(len(order), device=v.device)
    else:
        offsets, order, where = list(range(rows + 1)), [(1, i) for i in range(rows)], s["slots"].long()
    length = torch.tensor([n for n, _ in order], device=v.device)
    start = torch.tensor(offsets[:-1], device=v.device)
    # drop the finished sequences each time a length is passed
    cuts = sorted({n for n, _ in order})
    t = 0
    for cut in cuts:
        alive = (length >= cut).nonzero()[:, 0]
        slot, at, S = where[alive], start[alive], state[where[alive]]
        while t < cut:
            r = at + t
            kt, qt = (x[r][:, :, None, :].expand(-1, -1, share, -1).flatten(1, 2) for x in (k, q))
            S.mul_(torch.exp(decay[r])[..., None, None]).add_(kt[..., :, None] * v[r][..., None, :])
            out[r] = torch.einsum("phk,phkv->phv", qt, S) * s["scale"]
            t += 1
        state[slot] = S
    return {"out": out, "state": state}


def _exact_cache(s):
    """Each column block of a row by itself; a code is the quotient, rounded to 32 bits, at the format's nearest value."""
    case = s["case"]
    op, block, cols, eight = case["op"], case["block"], case["cols"], case["format"] == "int8"
    codes, scales, slots = s["codes"].float().double(), s["scales"].double(), s["slots"].long()
    if op != "resume":
        x = s["x"].double()
        for b, lo in enumerate(range(0, cols, block)):
            part = x[:, :, lo:lo + block]
            scale = (part.abs().max(dim=2).values / (127 if eight else 448)).float().double()
            quotient = (part / scale.masked_fill(scale == 0, 1.0)[:, :, None]).float().double()
            if eight:
                code = torch.round(quotient).clamp(-127, 127)
            else:
                size = quotient.abs().clamp(min=2.0 ** -6)
                step = torch.exp2(torch.floor(torch.log2(size)) - 3)
                code = (torch.round(quotient / step) * step).clamp(-448, 448)
            codes[slots, :, lo:lo + block] = code
            scales[slots, :, b] = scale
        if op == "park":
            return {"codes": codes, "scales": scales}
    values = torch.empty((len(slots), case["rows"], cols), dtype=torch.float64, device=codes.device)
    for b, lo in enumerate(range(0, cols, block)):
        values[:, :, lo:lo + block] = codes[slots, :, lo:lo + block] * scales[slots, :, b][:, :, None]
    return values if op == "resume" else {"values": values, "scales": scales}


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] in ("attention", "step"):
        h, hq, dk, dv = case["heads"], case["qk_heads"], case["dk"], case["dv"]
        n = sum(_lengths(case)) if case["op"] == "attention" else case["rows"]
        states = case["n_seq"] if case["op"] == "attention" else n
        # queries, keys, values, outputs and gates once; each state read and written
        bytes_ = size * n * (2 * hq * dk + 2 * h * dv) + 4 * (n * h if case["gated"] else h) + 8 * states * h * dk * dv
        # the recurrence: decay and update of the state, and the output's product
        return {"bytes": bytes_, "flops": 5 * n * h * dk * dv}
    if case["op"] == "norm":
        n = case["n"] * case["positions"] * case["channels"]
        return {"bytes": 2 * size * n + 8 * case["channels"], "flops": 8 * n}
    n = case["n"] * case["rows"] * case["cols"]
    scales = 4 * case["n"] * case["rows"] * -(-case["cols"] // case["block"])
    one = size * n + n + scales
    return {"bytes": 2 * one if case["op"] == "both" else one, "flops": 4 * n}
