"""Timed cases of the operators that a layer of a linear-attention model,
served in 8 bits, is made of.

A case is a dict of plain values; its `kind` names the operator:

* norm       h = x + r, RMS norm of h's rows, the output in 8-bit integers with
             a scale for each row; h is returned too (the next residual).
* product    out = sa[m]·sb[n]·Σ_k a[m, k]·b[n, k] of 8-bit integers.
* attention  linear attention with a decay e^g for each head:
             S_t = e^g·S_{t-1} + k_tᵀv_t, o_t = scale·q_t·S_t, from a state that
             comes in to the state that goes out.

`run` computes them with elementary torch operations, or, where `own` is set,
through the package's entry points on the device's own stream, from plans that
a program prepares once for its buffers.
"""
from __future__ import annotations

import math

import torch

own = False  # set by the program that times: the package's kernels, or the plain form

EPSILON = 1e-5
CHUNK = 64  # tokens that the plain form of the attention takes together

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token of a decoder: a launch and a few KiB.
        {"name": "norm_1x4096", "kind": "norm", "dtype": "bf16", "rows": 1, "cols": 4096, "residual": True, "pad": 0},
        # Rows of odd width in f32 with no residual, off 16-byte boundaries.
        {"name": "norm_1000x5001_f32", "kind": "norm", "dtype": "f32", "rows": 1000, "cols": 5001, "residual": False,
         "pad": 0},
        # A long prompt of a wide model: memory bandwidth alone.
        {"name": "norm_16384x8192", "kind": "norm", "dtype": "bf16", "rows": 16384, "cols": 8192, "residual": True,
         "pad": 0},
        # One token through a square projection: the weights are read once.
        {"name": "product_1x4096x4096", "kind": "product", "dtype": "bf16", "m": 1, "n": 4096, "k": 4096, "pad": 0},
        # A decode step of 64 sequences through a wide projection.
        {"name": "product_64x8192x8192", "kind": "product", "dtype": "bf16", "m": 64, "n": 8192, "k": 8192, "pad": 0},
        # Odd sizes all round, f32 out: rows of the operands lie off any vector's boundary.
        {"name": "product_1000x1027x4099_f32", "kind": "product", "dtype": "f32", "m": 1000, "n": 1027, "k": 4099,
         "pad": 0},
        # A long prompt through a wide projection: matrix instructions alone.
        {"name": "product_8192x8192x8192", "kind": "product", "dtype": "bf16", "m": 8192, "n": 8192, "k": 8192,
         "pad": 0},
        # One token of one sequence: the state is read and written once.
        {"name": "attention_step_1x16", "kind": "attention", "dtype": "bf16", "batch": 1, "tokens": 1, "heads": 16,
         "kv_heads": 16, "dk": 128, "dv": 128, "lengths": False, "order": "tokens"},
        # A decode step of 128 sequences: 512 MiB of state in and out.
        {"name": "attention_step_128x32", "kind": "attention", "dtype": "bf16", "batch": 128, "tokens": 1, "heads": 32,
         "kv_heads": 32, "dk": 128, "dv": 128, "lengths": False, "order": "tokens"},
        # One long prompt with few heads, q, k and v side by side as a fused
        # projection leaves them: the tokens have to be split over the card.
        {"name": "attention_1x16x16384", "kind": "attention", "dtype": "bf16", "batch": 1, "tokens": 16384,
         "heads": 16, "kv_heads": 16, "dk": 128, "dv": 128, "lengths": False, "order": "packed"},
        # A batch of prompts: heads enough to fill the card.
        {"name": "attention_8x32x4096", "kind": "attention", "dtype": "bf16", "batch": 8, "tokens": 4096, "heads": 32,
         "kv_heads": 32, "dk": 128, "dv": 128, "lengths": False, "order": "tokens"},
        # Prompts of their own lengths in f32, shared key and value heads, heads of unequal widths.
        {"name": "attention_5x12x1000_f32", "kind": "attention", "dtype": "f32", "batch": 5, "tokens": 1000,
         "heads": 12, "kv_heads": 4, "dk": 80, "dv": 96, "lengths": True, "order": "heads"},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 64 or 16, at times any number."""
    n, unit = _log_int(rng, lo, hi), rng.choice((64, 64, 16, 1))
    return min(hi, max(lo, n // unit * unit))


def draw(rng):
    kind = rng.choice(("norm", "product", "product", "attention", "attention"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind == "norm":
        rows, cols = _log_int(rng, 1, 16384), _width(rng, 64, 16384)
        rows = min(rows, (1 << 26) // cols)
        return {"kind": kind, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.7,
                "pad": rng.choice((0, 0, 0, 8, 3))}
    if kind == "product":
        m, n, k = _log_int(rng, 1, 8192), _width(rng, 64, 16384), _width(rng, 64, 16384)
        m = max(1, min(m, (1 << 38) // (n * k)))
        return {"kind": kind, "dtype": dtype, "m": m, "n": n, "k": k, "pad": rng.choice((0, 0, 0, 16, 5))}
    kv_heads = rng.choice((1, 2, 4, 8, 8, 16, 32))
    heads = kv_heads * rng.choice((1, 1, 1, 2, 4))
    dk, dv = rng.choice(((64, 64), (128, 128), (128, 128), (32, 64), (64, 128), (96, 80), (256, 128), (37, 53)))
    batch = _log_int(rng, 1, 64)
    if rng.random() < 0.4:  # a decode step
        batch = max(1, min(batch, (1 << 26) // (heads * dk * dv)))
        tokens = 1
    else:
        tokens = _log_int(rng, 2, 16384)
        batch = max(1, min(batch, (1 << 27) // (tokens * heads * (dk + dv))))
        tokens = min(tokens, (1 << 27) // (batch * heads * (dk + dv)))
    return {"kind": kind, "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dk": dk, "dv": dv, "lengths": tokens > 1 and rng.random() < 0.3,
            "order": rng.choice(("tokens", "heads", "packed"))}


# ----------------------------------------------------------------- inputs
def _rows(values, pad):
    """The same rows, `pad` elements further apart."""
    if not pad:
        return values
    wide = torch.empty((values.shape[0], values.shape[1] + pad), dtype=values.dtype, device=values.device)
    wide[:, :values.shape[1]] = values
    return wide[:, :values.shape[1]]


def _inputs(case, seed):
    """The operands of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=g)

    def bytes_(rows, cols):
        return torch.randint(-127, 128, (rows, cols), device="cuda", dtype=torch.int8, generator=g)

    dtype = TYPES[case["dtype"]]
    if case["kind"] == "norm":
        rows, cols, pad = case["rows"], case["cols"], case["pad"]
        x = {"x": _rows(normal(rows, cols, dtype=dtype), pad), "w": uniform(0.5, 1.5, cols).to(dtype), "r": None}
        if case["residual"]:
            x["r"] = _rows(normal(rows, cols, std=3.0, dtype=dtype), pad)
        return x
    if case["kind"] == "product":
        m, n, k, pad = case["m"], case["n"], case["k"], case["pad"]
        return {"a": _rows(bytes_(m, k), pad), "b": _rows(bytes_(n, k), pad), "sa": uniform(0.005, 0.05, m),
                "sb": uniform(1e-4, 1e-3, n)}
    b, t, h, hk, dk, dv = (case[key] for key in ("batch", "tokens", "heads", "kv_heads", "dk", "dv"))
    if case["order"] == "packed":  # one row of q | k | v for a token
        rows = normal(b, t, h * dk + hk * (dk + dv), dtype=dtype)
        q, k, v = (part.unflatten(-1, (-1, d)) for part, d in zip(
            rows.split((h * dk, hk * dk, hk * dv), dim=-1), (dk, dk, dv)))
    elif case["order"] == "tokens":
        q, k, v = (normal(b, t, n, d, dtype=dtype) for n, d in ((h, dk), (hk, dk), (hk, dv)))
    else:  # heads outside tokens
        q, k, v = (normal(b, n, t, d, dtype=dtype).transpose(1, 2) for n, d in ((h, dk), (hk, dk), (hk, dv)))
    # Decays from 1 - 2^-10 to 1 - 2^-2 a token: a head remembers 4 to 1000 tokens.
    decay = torch.log1p(-torch.exp2(uniform(-10.0, -2.0, h)))
    lengths = None
    if case["lengths"]:
        lengths = torch.randint(0, t + 1, (b,), device="cuda", dtype=torch.int32, generator=g)
    return {"q": q, "k": k, "v": v, "decay": decay, "state": normal(b, h, dk, dv, std=2.0), "lengths": lengths}


# ---------------------------------------------------------------- prepare
def prepare(case, seed):
    """The operands, and the buffers that a program's outputs go to."""
    state = {"case": case, **_inputs(case, seed)}
    dtype = TYPES[case["dtype"]]
    if case["kind"] == "norm":
        shape = case["rows"], case["cols"]
        state["out"] = {"h": torch.empty(shape, dtype=dtype, device="cuda") if case["residual"] else None,
                        "q": torch.empty(shape, dtype=torch.int8, device="cuda"),
                        "scales": torch.empty(shape[0], device="cuda"),
                        "values": torch.empty(shape, dtype=torch.bfloat16, device="cuda")}
    elif case["kind"] == "product":
        state["out"] = torch.empty((case["m"], case["n"]), dtype=dtype, device="cuda")
    else:
        q, v = state["q"], state["v"]
        if case["order"] == "heads":
            o = torch.empty((q.shape[0], q.shape[2], q.shape[1], v.shape[3]), dtype=dtype, device="cuda").transpose(1, 2)
        else:
            o = torch.empty((*q.shape[:3], v.shape[3]), dtype=dtype, device="cuda")
        state["out"] = {"o": o, "state": torch.empty_like(state["state"])}
    torch.cuda.synchronize()  # the device's own stream does not wait for torch's
    return state


_device = None


def _dev(hx):
    global _device
    if _device is None:
        _device = hx.RocmDevice.try_default()
    return _device


def _view(hx, dev, t):
    """A tensor's memory as a strided view of the package."""
    if t is None:
        return None
    dtype = {torch.float32: "float32", torch.int8: "int8", torch.int32: "uint32"}.get(t.dtype) or hx.bfloat16
    size = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0
    return hx.StridedView(dev.borrow(t.data_ptr(), dtype, size, owner=t), hx.Layout.try_new(t.shape, t.stride()))


def _plan(state):
    """The case's plan: its operands and outputs bound once."""
    import hephaestus_amd as hx

    case, dev, out = state["case"], _dev(hx), state["out"]

    def view(t):
        return _view(hx, dev, t)

    def buffer(t):
        return None if t is None else view(t).buffer

    if case["kind"] == "norm":
        # Returned values are read back on the stream that wrote them.
        state["stream"] = torch.cuda.ExternalStream(dev.stream)
        return hx.RocmNormOps().prepare_rms_norm_quantize(
            dev, view(state["x"]), buffer(state["w"]), EPSILON, view(out["q"]), buffer(out["scales"]),
            residual=view(state["r"]), residual_out=view(out["h"]))
    if case["kind"] == "product":
        return hx.RocmMatrixOps().prepare_matmul_i8(dev, view(state["a"]), buffer(state["sa"]), view(state["b"]),
                                                    buffer(state["sb"]), view(out))
    return hx.RocmLinearAttentionOps().prepare_linear_attention(
        dev, view(state["q"]), view(state["k"]), view(state["v"]), buffer(state["decay"]), view(out["o"]),
        scale=_scale(case), state_in=view(state["state"]), state_out=view(out["state"]),
        lengths=buffer(state["lengths"]))


def _scale(case):
    return 1.0 / math.sqrt(case["dk"])


# -------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if own:
        if "plan" not in state:
            state["plan"] = _plan(state)
        state["plan"].dispatch()
        out = state["out"]
        if case["kind"] != "norm":
            return out
        with torch.cuda.stream(state["stream"]):  # 8-bit integers as the values they stand for
            torch.mul(out["q"], out["scales"][:, None], out=out["values"])
        return {"h": out["h"], "values": out["values"], "scales": out["scales"]}
    if case["kind"] == "norm":
        return _plain_norm(state["x"], state["r"], state["w"])
    if case["kind"] == "product":
        total = state["a"].float() @ state["b"].float().t()
        return (total * state["sa"][:, None] * state["sb"]).to(TYPES[case["dtype"]])
    if case["tokens"] == 1 and state["lengths"] is None:
        return _plain_step(state["q"], state["k"], state["v"], state["decay"], state["state"], _scale(case))
    return _plain_attention(state["q"], state["k"], state["v"], state["decay"], state["state"], state["lengths"],
                            _scale(case))


def _plain_norm(x, r, w):
    h = x.float() if r is None else x.float() + r.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPSILON) * w.float()
    top = y.abs().amax(-1, keepdim=True)
    scales = top / 127
    q = torch.round(y * (127 / top)).clamp(-127, 127)
    return {"h": None if r is None else h.to(x.dtype), "values": (q * scales).to(torch.bfloat16),
            "scales": scales[:, 0]}


def _plain_step(q, k, v, decay, state, scale):
    """The recurrence, for one token of each sequence."""
    group = q.shape[2] // k.shape[2]
    k_, v_ = (x[:, 0].float().repeat_interleave(group, 1) for x in (k, v))
    last = torch.exp(decay)[:, None, None] * state + k_[..., None] * v_[..., None, :]
    o = (q.transpose(1, 2).float() @ last).transpose(1, 2) * scale
    return {"o": o.to(q.dtype), "state": last}


def _plain_attention(q, k, v, decay, state, lengths, scale):
    """Products within chunks of tokens, and the chunks' states joined by
    one product with the powers of the decay between them."""
    batch, tokens, heads, dk = q.shape
    dv, c = v.shape[3], min(CHUNK, tokens)
    chunks = -(-tokens // c)
    alive = torch.arange(tokens, device=q.device)[None] < (
        torch.full((batch,), tokens, device=q.device) if lengths is None else lengths)[:, None]

    def split(x):  # [batch, heads, chunks, c, width], f32
        x = x.float() * alive[:, :, None, None]
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, chunks * c - tokens)).transpose(1, 2)
        x = x.unflatten(2, (chunks, c))
        return x if x.shape[1] == heads else x.repeat_interleave(heads // x.shape[1], 1)

    q_, k_, v_ = split(q), split(k), split(v)
    at = torch.arange(c, device=q.device)
    g = decay[:, None, None]
    far = at[:, None] - at
    within = torch.where(far >= 0, torch.exp(g * far.clamp(min=0)), 0.0)  # [heads, c, c]
    o = ((q_ @ k_.transpose(-1, -2)) * within[:, None]) @ v_
    added = (k_ * torch.exp(g * (c - 1 - at)[:, None])[:, None]).transpose(-1, -2) @ v_
    n = torch.arange(chunks, device=q.device)
    far = n[:, None] - n - 1
    between = torch.where(far >= 0, torch.exp(g * (far * c).clamp(min=0)), 0.0)  # [heads, chunks, chunks]
    before = (between @ added.flatten(3)).unflatten(3, (dk, dv))
    before = before + torch.exp(g * (n * c))[:, 0, :, None, None] * state[:, :, None]
    o = o + (q_ @ before) * torch.exp(g * (at + 1)[:, None])[:, None]
    o = (o * scale).flatten(2, 3)[:, :, :tokens].transpose(1, 2)
    # The state after the last token of each sequence.
    count = alive.sum(1)
    left = (count[:, None] - 1 - torch.arange(chunks * c, device=q.device)).clamp(min=0)  # [batch, tokens]
    weight = torch.exp(decay[None, :, None] * left[:, None])  # v is 0 past the last token
    last = (k_.flatten(2, 3) * weight[..., None]).transpose(-1, -2) @ v_.flatten(2, 3)
    last = last + torch.exp(decay[None, :] * count[:, None])[..., None, None] * state
    return {"o": (o * alive[:, :, None, None]).to(q.dtype), "state": last}


# ------------------------------------------------------------------- work
def work(case):
    """Each operand read once, each result written once; the attention's
    arithmetic is that of the recurrence."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + size * case["cols"] + 4 * case["rows"],
                "flops": 6 * n}
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + 4) + size * m * n, "flops": 2 * m * n * k}
    b, t, h, hk, dk, dv = (case[key] for key in ("batch", "tokens", "heads", "kv_heads", "dk", "dv"))
    return {"bytes": size * b * t * (h + hk) * (dk + dv) + 8 * b * h * dk * dv, "flops": 4 * b * t * h * dk * dv}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "norm":
        h = x["x"].double()
        if x["r"] is not None:
            h = h + x["r"].double()
        y = h / ((h * h).sum(1, keepdim=True) / h.shape[1] + EPSILON).sqrt() * x["w"].double()
        step = y.abs().max(1, keepdim=True).values / 127
        return {"h": None if x["r"] is None else h, "values": torch.round(y / step) * step, "scales": step[:, 0]}
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        total = torch.empty((m, n), dtype=torch.float64, device="cuda")
        b = x["b"].double().t().contiguous()
        for at in range(0, m, 2048):  # sums of integers below 2^53: exact in any order
            total[at:at + 2048] = x["a"][at:at + 2048].double() @ b
        return x["sa"].double()[:, None] * total * x["sb"].double()
    b, t, h, hk, dk, dv = (case[key] for key in ("batch", "tokens", "heads", "kv_heads", "dk", "dv"))
    o = torch.zeros((b, t, h, dv), dtype=torch.float64, device="cuda")
    last = torch.empty((b, h, dk, dv), dtype=torch.float64, device="cuda")
    counts = [t] * b if x["lengths"] is None else x["lengths"].tolist()
    for i, count in enumerate(counts):
        at = torch.arange(count, device="cuda", dtype=torch.float64)
        for j in range(h):
            g, first = x["decay"][j].double(), x["state"][i, j].double()
            q = x["q"][i, :count, j].double()
            k, v = (x[name][i, :count, j * hk // h].double() for name in "kv")
            for lo in range(0, count, 2048):  # rows of tokens against all before them
                hi = min(count, lo + 2048)
                far = at[lo:hi, None] - at[None, :hi]
                score = (q[lo:hi] @ k[:hi].t().contiguous()) * torch.exp(g * far).where(far >= 0, torch.zeros_like(far))
                o[i, lo:hi, j] = score @ v[:hi] + torch.exp(g * (at[lo:hi, None] + 1)) * (q[lo:hi] @ first)
            last[i, j] = (k * torch.exp(g * (count - 1 - at[:, None]))).t().contiguous() @ v + torch.exp(g * count) * first
    return {"o": o * _scale(case), "state": last}
