"""Timed cases of the operators that train a language model whose layers mix
tokens by a gated recurrence.

A case is a dict of plain values; its `kind` names the operator:

* norm             h = x + r, y = (h - mean)·rstd·w + b for each row; y, h, mean and
                   rstd are returned.
* norm_grad        its backward pass: the gradients of h, w and b from that of y, and
                   the gradient that reaches h past the norm added to the first.
* recurrence       h_t = f_t·h_{t-1} + (1 - f_t)·x_t with f = 1 / (1 + e^-z), for each
                   channel, from a state that comes in to the state that goes out.
* recurrence_grad  its backward pass: the gradients of z, x and the state that came in.
* loss             softmax cross entropy of the logits x·wᵀ over a vocabulary: the loss
                   and the logarithm of the softmax's denominator of each row.  Rows
                   with a target beyond the vocabulary are left out.
* loss_grad        its backward pass: the gradients of x and w.

`run` computes them with elementary torch operations, or, where `own` is set,
through the package's entry points on the device's own stream, from plans that
a program prepares once for its buffers.
"""
from __future__ import annotations

import math

import torch

own = False  # set by the program that times: the package's kernels, or the plain form

EPSILON = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token of a decoder: a launch and a few KiB.
        {"name": "norm_1x4096", "kind": "norm", "dtype": "bf16", "rows": 1, "cols": 4096, "residual": True, "pad": 0},
        # A step's tokens through a wide layer: memory bandwidth alone.
        {"name": "norm_16384x8192", "kind": "norm", "dtype": "bf16", "rows": 16384, "cols": 8192, "residual": True,
         "pad": 0},
        # Rows of odd width in f32, off 16-byte boundaries, of a layer with no residual.
        {"name": "norm_grad_1000x5001_f32", "kind": "norm_grad", "dtype": "f32", "rows": 1000, "cols": 5001,
         "residual": False, "pad": 0},
        # The backward pass of a step: the weight's gradient is a sum over all rows.
        {"name": "norm_grad_16384x8192", "kind": "norm_grad", "dtype": "bf16", "rows": 16384, "cols": 8192,
         "residual": True, "pad": 0},
        # One token of 64 sequences that are decoded together.
        {"name": "recurrence_64x1x4096", "kind": "recurrence", "dtype": "bf16", "batch": 64, "tokens": 1,
         "channels": 4096, "lengths": False, "order": "tokens"},
        # A training batch, gate and input side by side as one projection leaves them.
        {"name": "recurrence_8x4096x4096", "kind": "recurrence", "dtype": "bf16", "batch": 8, "tokens": 4096,
         "channels": 4096, "lengths": False, "order": "packed"},
        # Sequences of their own lengths in f32, an odd number of channels.
        {"name": "recurrence_grad_5x1000x1027_f32", "kind": "recurrence_grad", "dtype": "f32", "batch": 5,
         "tokens": 1000, "channels": 1027, "lengths": True, "order": "tokens"},
        # One long sequence with few channels: the tokens have to be split over the card.
        {"name": "recurrence_grad_1x65536x2048", "kind": "recurrence_grad", "dtype": "bf16", "batch": 1,
         "tokens": 65536, "channels": 2048, "lengths": False, "order": "tokens"},
        # A few tokens scored: the vocabulary's weights are read once.
        {"name": "loss_16x32000x2048", "kind": "loss", "dtype": "bf16", "rows": 16, "vocab": 32000, "width": 2048,
         "pad": 0},
        # A held-out batch: matrix instructions alone.
        {"name": "loss_8192x32768x4096", "kind": "loss", "dtype": "bf16", "rows": 8192, "vocab": 32768, "width": 4096,
         "pad": 0},
        # Odd sizes all round in f32: rows of the operands lie off any vector's boundary.
        {"name": "loss_grad_1000x5003x1025_f32", "kind": "loss_grad", "dtype": "f32", "rows": 1000, "vocab": 5003,
         "width": 1025, "pad": 0},
        # A training step's head: three products of this size.
        {"name": "loss_grad_8192x32768x4096", "kind": "loss_grad", "dtype": "bf16", "rows": 8192, "vocab": 32768,
         "width": 4096, "pad": 0},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 64 or 16, at times any number."""
    n, unit = _log_int(rng, lo, hi), rng.choice((64, 64, 16, 1))
    return min(hi, max(lo, n // unit * unit))


def draw(rng):
    kind = rng.choice(("norm", "norm_grad", "recurrence", "recurrence_grad", "loss", "loss_grad"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    wide = dtype == "f32"
    if kind in ("norm", "norm_grad"):
        rows, cols = _log_int(rng, 1, 16384), _width(rng, 64, 16384)
        rows = min(rows, (1 << (26 - wide)) // cols)
        return {"kind": kind, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.7,
                "pad": rng.choice((0, 0, 0, 8, 3))}
    if kind in ("loss", "loss_grad"):
        rows, vocab, width = _log_int(rng, 1, 8192), _width(rng, 500, 131072), _width(rng, 64, 8192)
        rows = max(1, min(rows, (1 << (36 if wide else 39)) // (vocab * width), (1 << 28) // vocab))
        return {"kind": kind, "dtype": dtype, "rows": rows, "vocab": vocab, "width": width,
                "pad": rng.choice((0, 0, 0, 8, 3))}
    batch, channels = _log_int(rng, 1, 64), _width(rng, 64, 8192)
    tokens = 1 if kind == "recurrence" and rng.random() < 0.3 else _log_int(rng, 2, 65536)
    batch = max(1, min(batch, (1 << (26 - wide)) // (tokens * channels)))
    tokens = min(tokens, (1 << (26 - wide)) // (batch * channels))
    return {"kind": kind, "dtype": dtype, "batch": batch, "tokens": tokens, "channels": channels,
            "lengths": tokens > 1 and rng.random() < 0.3, "order": rng.choice(("tokens", "packed", "time"))}


# ----------------------------------------------------------------- inputs
def _rows(values, pad):
    """The same rows, `pad` elements further apart."""
    if not pad:
        return values
    wide = torch.empty((values.shape[0], values.shape[1] + pad), dtype=values.dtype, device=values.device)
    wide[:, :values.shape[1]] = values
    return wide[:, :values.shape[1]]


def _sequences(case, make):
    """Two arrays [batch, tokens, channels] that `make` makes, in the case's order."""
    b, t, c = case["batch"], case["tokens"], case["channels"]
    if case["order"] == "packed":  # one row of both for a token
        return make(b, t, 2 * c).split(c, dim=-1)
    if case["order"] == "time":  # tokens outside sequences
        return tuple(make(t, b, c).transpose(0, 1) for _ in range(2))
    return make(b, t, c), make(b, t, c)


def _inputs(case, seed):
    """The operands of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=g)

    def below(n, *shape):
        return torch.randint(0, n, shape, device="cuda", dtype=torch.int32, generator=g)

    if case["kind"] in ("norm", "norm_grad"):
        rows, cols, pad = case["rows"], case["cols"], case["pad"]
        x = {"x": _rows(normal(rows, cols) + uniform(-1.0, 1.0, rows, 1).to(dtype), pad), "r": None,
             "w": uniform(0.5, 1.5, cols).to(dtype), "b": normal(cols, std=0.2)}
        if case["residual"]:
            x["r"] = _rows(normal(rows, cols, std=3.0), pad)
        if case["kind"] == "norm_grad":  # x is what the forward pass normalised, r the gradient that passes it
            x["dy"] = _rows(normal(rows, cols, std=1e-3), pad)
            x["r"] = None if x["r"] is None else _rows(normal(rows, cols, std=1e-3), pad)
            wide = x["x"].float()
            x["mean"] = wide.mean(1)
            x["rstd"] = torch.rsqrt((wide - x["mean"][:, None]).square().mean(1) + EPSILON)
        return x
    if case["kind"] in ("recurrence", "recurrence_grad"):
        b, t, c = case["batch"], case["tokens"], case["channels"]
        gate, x = _sequences(case, normal)
        # Channels that remember 2 to 1000 tokens, a token's gate around its channel's.
        gate.add_(uniform(0.0, 7.0, c).to(dtype))
        state = {"gate": gate, "x": x, "first": torch.randn((b, c), device="cuda", generator=g),
                 "lengths": below(t + 1, b) if case["lengths"] else None}
        if case["kind"] == "recurrence_grad":
            # Outputs as large as the forward pass gives them, where each has its own inputs.
            state["h"] = normal(b, t, c, std=0.5)
            state["dy"] = normal(b, t, c, std=1e-3)
            state["dlast"] = torch.randn((b, c), device="cuda", generator=g) * 1e-3
        return state
    rows, vocab, width, pad = case["rows"], case["vocab"], case["width"], case["pad"]
    x = {"x": _rows(normal(rows, width), pad), "w": _rows(normal(vocab, width, std=2.0 / math.sqrt(width)), pad)}
    # One row in sixteen has no target: padding, or the text of a question.
    x["targets"] = torch.where(uniform(0.0, 1.0, rows) < 1 / 16, -1, below(vocab, rows))
    if case["kind"] == "loss_grad":  # of the mean over the rows that have one
        with_target = x["targets"] >= 0
        x["grad"] = with_target / with_target.sum().clamp(min=1)
        x["lse"] = _plain_lse(x["x"], x["w"])[1]
    return x


# ---------------------------------------------------------------- prepare
def prepare(case, seed):
    """The operands, and the buffers that a program's outputs go to."""
    state = {"case": case, **_inputs(case, seed)}
    dtype, kind = TYPES[case["dtype"]], case["kind"]

    def new(*shape, of=torch.float32):
        return torch.empty(shape, dtype=of, device="cuda")

    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        state["out"] = {"y": new(rows, cols, of=dtype), "h": new(rows, cols, of=dtype) if case["residual"] else None,
                        "mean": new(rows), "rstd": new(rows)}
    elif kind == "norm_grad":
        rows, cols = case["rows"], case["cols"]
        state["out"] = {"dx": new(rows, cols, of=dtype), "dw": new(cols), "db": new(cols)}
    elif kind == "recurrence":
        b, t, c = case["batch"], case["tokens"], case["channels"]
        h = new(t, b, c, of=dtype).transpose(0, 1) if case["order"] == "time" else new(b, t, c, of=dtype)
        state["out"] = {"h": h, "last": new(b, c)}
    elif kind == "recurrence_grad":
        dgate, dx = _sequences(case, lambda *shape: new(*shape, of=dtype))
        state["out"] = {"dgate": dgate, "dx": dx, "dfirst": new(case["batch"], case["channels"])}
    elif kind == "loss":
        state["out"] = {"loss": new(case["rows"]), "lse": new(case["rows"])}
    else:
        state["out"] = {"dx": new(case["rows"], case["width"], of=dtype),
                        "dw": new(case["vocab"], case["width"], of=dtype)}
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
    dtype = {torch.float32: "float32", torch.int32: "uint32"}.get(t.dtype) or hx.bfloat16
    size = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0
    return hx.StridedView(dev.borrow(t.data_ptr(), dtype, size, owner=t), hx.Layout.try_new(t.shape, t.stride()))


def _plan(state):
    """The case's plan: its operands and outputs bound once."""
    import hephaestus_amd as hx

    case, dev, out = state["case"], _dev(hx), state["out"]

    def view(name, of=state):
        return _view(hx, dev, of[name])

    def buffer(name, of=state):
        v = view(name, of)
        return None if v is None else v.buffer

    if case["kind"] == "norm":
        return hx.RocmLayerNormOps().prepare_layer_norm(
            dev, view("x"), buffer("w"), buffer("b"), EPSILON, view("y", out), residual=view("r"),
            residual_out=view("h", out), mean=buffer("mean", out), rstd=buffer("rstd", out))
    if case["kind"] == "norm_grad":
        return hx.RocmLayerNormOps().prepare_layer_norm_backward(
            dev, view("dy"), view("x"), buffer("w"), buffer("mean"), buffer("rstd"), view("dx", out),
            residual_grad=view("r"), grad_weight=buffer("dw", out), grad_bias=buffer("db", out))
    if case["kind"] == "recurrence":
        return hx.RocmRecurrenceOps().prepare_gated_recurrence(
            dev, view("gate"), view("x"), view("h", out), state_in=view("first"), state_out=view("last", out),
            lengths=buffer("lengths"))
    if case["kind"] == "recurrence_grad":
        return hx.RocmRecurrenceOps().prepare_gated_recurrence_backward(
            dev, view("gate"), view("x"), view("h"), view("dy"), view("dgate", out), view("dx", out),
            state_in=view("first"), grad_state_out=view("dlast"), grad_state_in=view("dfirst", out),
            lengths=buffer("lengths"))
    if case["kind"] == "loss":
        return hx.RocmLossOps().prepare_linear_cross_entropy(
            dev, view("x"), view("w"), buffer("targets"), buffer("loss", out), buffer("lse", out))
    return hx.RocmLossOps().prepare_linear_cross_entropy_backward(
        dev, view("x"), view("w"), buffer("targets"), buffer("lse"), buffer("grad"), grad_x=view("dx", out),
        grad_weight=view("dw", out))


# -------------------------------------------------------------------- run
def run(state):
    if own:
        if "plan" not in state:
            state["plan"] = _plan(state)
        state["plan"].dispatch()
        return state["out"]
    kind = state["case"]["kind"]
    if kind == "norm":
        return _plain_norm(state["x"], state["r"], state["w"], state["b"])
    if kind == "norm_grad":
        return _plain_norm_grad(state["dy"], state["x"], state["r"], state["w"], state["mean"], state["rstd"])
    if kind == "recurrence":
        return _plain_recurrence(state["gate"], state["x"], state["first"], state["lengths"])
    if kind == "recurrence_grad":
        return _plain_recurrence_grad(*(state[key] for key in ("gate", "x", "h", "dy", "first", "dlast", "lengths")))
    if kind == "loss":
        logits, lse = _plain_lse(state["x"], state["w"])
        at = state["targets"].long()
        picked = logits.gather(1, at.clamp(min=0)[:, None])[:, 0]
        return {"loss": torch.where(at >= 0, lse - picked, 0.0), "lse": lse}
    return _plain_loss_grad(state["x"], state["w"], state["targets"], state["lse"], state["grad"])


def _plain_norm(x, r, w, b):
    h = x.float() if r is None else x.float() + r.float()
    mean = h.mean(1, keepdim=True)
    rstd = torch.rsqrt((h - mean).square().mean(1, keepdim=True) + EPSILON)
    y = (h - mean) * rstd * w.float() + b.float()
    return {"y": y.to(x.dtype), "h": None if r is None else h.to(x.dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _plain_norm_grad(dy, h, past, w, mean, rstd):
    g = dy.float()
    unit = (h.float() - mean[:, None]) * rstd[:, None]
    gw = g * w.float()
    dx = (gw - gw.mean(1, keepdim=True) - unit * (gw * unit).mean(1, keepdim=True)) * rstd[:, None]
    if past is not None:
        dx = dx + past.float()
    return {"dx": dx.to(h.dtype), "dw": (g * unit).sum(0), "db": g.sum(0)}


def _alive(x, lengths):
    """Which tokens of [batch, tokens, channels] a sequence has."""
    if lengths is None:
        return None
    return (torch.arange(x.shape[1], device=x.device)[None] < lengths[:, None])[..., None]


def _scan(f, b, first):
    """h_t = f_t·h_{t-1} + b_t along the tokens: all parts of the sequences a token
    at a time, then the parts one after another.  (h, the last state)"""
    tokens = f.shape[1]
    size = math.isqrt(tokens - 1) + 1
    parts = -(-tokens // size)
    more = (0, 0, 0, parts * size - tokens)
    f = torch.nn.functional.pad(f, more, value=1.0).unflatten(1, (parts, size))
    b = torch.nn.functional.pad(b, more).unflatten(1, (parts, size))
    h, kept, before = torch.empty_like(b), torch.empty_like(f), torch.empty_like(f[:, :, 0])
    h[:, :, 0], kept[:, :, 0] = b[:, :, 0], f[:, :, 0]
    for j in range(1, size):
        torch.addcmul(b[:, :, j], f[:, :, j], h[:, :, j - 1], out=h[:, :, j])
        torch.mul(f[:, :, j], kept[:, :, j - 1], out=kept[:, :, j])
    state = first
    for i in range(parts):
        before[:, i] = state
        state = torch.addcmul(h[:, i, -1], kept[:, i, -1], state)
    h.addcmul_(kept, before[:, :, None])
    return h.flatten(1, 2)[:, :tokens], state


def _plain_recurrence(gate, x, first, lengths):
    alive, z = _alive(x, lengths), gate.float()
    f, b = torch.sigmoid(z), torch.sigmoid(-z) * x.float()
    if alive is not None:  # past its end a sequence keeps its state
        f, b = torch.where(alive, f, 1.0), torch.where(alive, b, 0.0)
    if x.shape[1] == 1:
        last = f[:, 0] * first + b[:, 0]
        h = last[:, None]
    else:
        h, last = _scan(f, b, first)
    return {"h": (h if alive is None else torch.where(alive, h, 0.0)).to(x.dtype), "last": last}


def _plain_recurrence_grad(gate, x, h, dy, first, dlast, lengths):
    alive, z = _alive(x, lengths), gate.float()
    f, new, dy = torch.sigmoid(z), torch.sigmoid(-z), dy.float()
    if alive is not None:
        f, new, dy = torch.where(alive, f, 1.0), torch.where(alive, new, 0.0), torch.where(alive, dy, 0.0)
    # From the last token on: g_t = dy_t + f_{t+1}·g_{t+1}, and after the last the state's own.
    back = torch.cat((torch.ones_like(f[:, :1]), f.flip(1)[:, :-1]), 1)
    g = _scan(back, dy.flip(1), dlast)[0].flip(1)
    before = torch.cat((first[:, None], h[:, :-1].float()), 1)
    dx = new * g
    return {"dgate": (f * dx * (before - x.float())).to(x.dtype), "dx": dx.to(x.dtype), "dfirst": f[:, 0] * g[:, 0]}


def _plain_lse(x, w):
    logits = x.float() @ w.float().t()
    top = logits.amax(1, keepdim=True)
    return logits, (top + torch.log(torch.exp(logits - top).sum(1, keepdim=True)))[:, 0]


def _plain_loss_grad(x, w, targets, lse, grad):
    wide_x, wide_w = x.float(), w.float()
    g = torch.exp(wide_x @ wide_w.t() - lse[:, None])
    at = targets.long()
    rows = torch.arange(x.shape[0], device=x.device)
    g[rows, at.clamp(min=0)] -= (at >= 0).float()
    g *= torch.where(at >= 0, grad, 0.0)[:, None]
    return {"dx": (g @ wide_w).to(x.dtype), "dw": (g.t() @ wide_x).to(x.dtype)}


# ------------------------------------------------------------------- work
def work(case):
    """Each operand read once, each result written once; the loss's backward
    pass has its logits again, which nothing keeps."""
    size, kind = 4 if case["dtype"] == "f32" else 2, case["kind"]
    if kind in ("norm", "norm_grad"):
        n, cols, rows = case["rows"] * case["cols"], case["cols"], case["rows"]
        if kind == "norm":
            return {"bytes": n * size * (4 if case["residual"] else 2) + 2 * size * cols + 8 * rows, "flops": 8 * n}
        return {"bytes": n * size * (4 if case["residual"] else 3) + (size + 8) * cols + 8 * rows, "flops": 14 * n}
    if kind in ("recurrence", "recurrence_grad"):
        states = case["batch"] * case["channels"]
        n = states * case["tokens"]
        if kind == "recurrence":
            return {"bytes": 3 * n * size + 8 * states, "flops": 8 * n}
        return {"bytes": 6 * n * size + 12 * states, "flops": 12 * n}
    rows, vocab, width = case["rows"], case["vocab"], case["width"]
    product, operands = 2 * rows * vocab * width, (rows + vocab) * width * size
    if kind == "loss":
        return {"bytes": operands + 12 * rows, "flops": product}
    return {"bytes": 2 * operands + 12 * rows, "flops": 3 * product}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    x, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        h = x["x"].double()
        if x["r"] is not None:
            h = h + x["r"].double()
        mean = h.sum(1) / h.shape[1]
        far = h - mean[:, None]
        root = ((far * far).sum(1) / h.shape[1] + EPSILON).sqrt()
        return {"y": far / root[:, None] * x["w"].double() + x["b"].double(), "h": None if x["r"] is None else h,
                "mean": mean, "rstd": 1 / root}
    if kind == "norm_grad":
        h, dy, rstd = x["x"].double(), x["dy"].double(), x["rstd"].double()[:, None]
        unit = (h - x["mean"].double()[:, None]) * rstd
        t = dy * x["w"].double()
        dx = rstd * (t - (t.sum(1, keepdim=True) + unit * (t * unit).sum(1, keepdim=True)) / h.shape[1])
        return {"dx": dx if x["r"] is None else dx + x["r"].double(), "dw": (dy * unit).sum(0), "db": dy.sum(0)}
    if kind in ("recurrence", "recurrence_grad"):
        return _exact_recurrence(case, x)
    rows, vocab = case["rows"], case["vocab"]
    w, targets = x["w"].double(), x["targets"].long()
    columns = w.t().contiguous()
    out = {name: [] for name in (("loss", "lse") if kind == "loss" else ("dx",))}
    dw = torch.zeros_like(w)
    for lo in range(0, rows, 2048):  # rows of logits at a time
        part, at = x["x"][lo:lo + 2048].double(), targets[lo:lo + 2048]
        logits = part @ columns
        if kind == "loss":
            lse = torch.logsumexp(logits, 1)
            picked = logits[torch.arange(len(at), device="cuda"), at.clamp(min=0)]
            out["loss"].append((lse - picked) * (at >= 0))
            out["lse"].append(lse)
        else:
            hot = at[:, None] == torch.arange(vocab, device="cuda")
            g = logits.sub_(x["lse"][lo:lo + 2048].double()[:, None]).exp_().sub_(hot.double())
            g.mul_((x["grad"][lo:lo + 2048].double() * (at >= 0))[:, None])
            out["dx"].append(g @ w)
            dw += g.t().contiguous() @ part
    out = {name: torch.cat(values) for name, values in out.items()}
    return out if kind == "loss" else {**out, "dw": dw}


def _exact_recurrence(case, x):
    """Token by token."""
    z, u = x["gate"].double(), x["x"].double()
    batch, tokens, _ = z.shape
    f, new = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
    ends = None if x["lengths"] is None else x["lengths"].long()

    def has(t):
        return torch.ones((batch, 1), dtype=torch.bool, device="cuda") if ends is None else (t < ends)[:, None]

    if case["kind"] == "recurrence":
        h, state = torch.zeros_like(u), x["first"].double()
        for t in range(tokens):
            state = torch.where(has(t), f[:, t] * state + new[:, t] * u[:, t], state)
            h[:, t] = state * has(t)
        return {"h": h, "last": state}
    dgate, dx, g = torch.zeros_like(u), torch.zeros_like(u), x["dlast"].double()
    for t in reversed(range(tokens)):  # g: the gradient of the state after token t
        total = g + x["dy"][:, t].double()
        before = x["h"][:, t - 1].double() if t else x["first"].double()
        dx[:, t] = total * new[:, t] * has(t)
        dgate[:, t] = total * (before - u[:, t]) * f[:, t] * new[:, t] * has(t)
        g = torch.where(has(t), total * f[:, t], g)
    return {"dgate": dgate, "dx": dx, "dfirst": g}
