"""The training operators written out plainly in 64 bits, each with a bound on
what roundings may make of its results."""
from __future__ import annotations

import numpy as np

import hephaestus_amd as hx
from layer_reference import EPS16, EPS32, as_float64

TYPES = {"f32": np.float32, "bf16": hx.bfloat16}


def rounding(dtype):
    """Half a step of a type, relative: what the last rounding of an output costs
    beyond the arithmetic in f32."""
    return EPS16 if dtype == hx.bfloat16 else EPS32


# ------------------------------------------------------------------- norm
def _depth(cols):
    """Additions in a row's sum that follow one another: up to 32 of a thread (more
    in rows beyond the registers, which 1024 threads share), 6 over the wave, 16
    over the waves."""
    return 54 + cols / 1024


def layer_norm(x, residual, weight, bias, epsilon):
    """({name: value}, {name: bound}) of h, mean, rstd and y."""
    dtype, cols = x.dtype, x.shape[1]
    r = 0.0 if residual is None else as_float64(residual)
    h = as_float64(x) + r
    w, b = as_float64(weight), np.zeros(cols) if bias is None else as_float64(bias)
    mean = h.mean(1, keepdims=True)
    d = h - mean
    var = (d * d).mean(1, keepdims=True)
    rstd = (var + epsilon)**-0.5
    u = d * rstd
    y = u * w + b
    depth, eps, fine = _depth(cols), EPS32, rounding(dtype)
    # Of h: one rounding of the sum.  What it leaves in the mean and the differences
    # is their own; the mean's first sum only shifts the differences, which are
    # corrected by what they sum up to.
    in_h = eps * (np.abs(as_float64(x)) + np.abs(r)) if residual is not None else 0 * h
    shift = depth * eps * np.abs(h).mean(1, keepdims=True)
    mean_off = in_h.mean(1, keepdims=True) + eps * (3 * np.abs(mean) + (depth + 2) * (np.abs(d).mean(1, keepdims=True) + shift))
    d_off = in_h + mean_off + eps * (np.abs(d) + shift)
    # Relative: of a sum of squares and of the difference of two such sums.
    var_off = 2 * (depth + 4) * eps * (var + shift * shift) + 2 * np.sqrt((d_off**2).mean(1, keepdims=True) * (var + d_off.max(1, keepdims=True)**2))
    rstd_off = rstd * (np.divide(0.5 * var_off, var + epsilon, out=np.zeros_like(var), where=var + epsilon > 0) + 4 * eps)
    y_off = (d_off * rstd + np.abs(d) * rstd_off + 3 * eps * np.abs(u)) * np.abs(w) + eps * (np.abs(u * w) + np.abs(b))
    value = {"h": h, "mean": mean[:, 0], "rstd": rstd[:, 0], "y": y}
    bound = {"h": in_h + fine * np.abs(h), "mean": mean_off[:, 0], "rstd": rstd_off[:, 0], "y": y_off + fine * np.abs(y)}
    return value, bound


def layer_norm_backward(dy, h, weight, mean, rstd, past):
    """The gradients of h, weight and bias, and their bounds."""
    dtype, (rows, cols) = h.dtype, h.shape
    g, w = as_float64(dy), as_float64(weight)
    mean, rstd = mean.astype(np.float64)[:, None], rstd.astype(np.float64)[:, None]
    u = (as_float64(h) - mean) * rstd
    t = g * w
    mt, mtu = t.mean(1, keepdims=True), (t * u).mean(1, keepdims=True)
    p = 0.0 if past is None else as_float64(past)
    dh = rstd * (t - mt - u * mtu) + p
    depth, eps, fine = _depth(cols) + 8, EPS32, rounding(dtype)
    terms = np.abs(t) + np.abs(t).mean(1, keepdims=True) + np.abs(u) * np.abs(t * u).mean(1, keepdims=True)
    # Rows that follow one another in a block's sums, the 16 groups of a block, and
    # the blocks in turns of 16.
    down = 100 + rows / 256
    value = {"dh": dh, "dw": (g * u).sum(0), "db": g.sum(0)}
    bound = {"dh": rstd * depth * eps * terms + eps * np.abs(p) + fine * np.abs(dh),
             "dw": down * eps * np.abs(g * u).sum(0), "db": down * eps * np.abs(g).sum(0)}
    return value, bound


# ------------------------------------------------------------- recurrence
def _gates(gate):
    z = as_float64(gate)
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))


def _lengths(lengths, batch, tokens):
    return [tokens] * batch if lengths is None else [min(tokens, int(n)) for n in lengths]


STEP = 12  # roundings of a token: the gate's exponential and quotient, two products, their sum, the joins


def gated_recurrence(gate, x, state=None, lengths=None):
    """Token by token: h and the last state, and their bounds: what a state is off
    decays with it, and each token adds its roundings."""
    dtype, (batch, tokens, channels) = x.dtype, x.shape
    f, rest, u = *_gates(gate), as_float64(x)
    h, off = np.zeros(u.shape), np.zeros(u.shape)
    last = np.zeros((batch, channels)) if state is None else state.astype(np.float64)
    last, last_off = last.copy(), np.zeros((batch, channels))
    for b, n in enumerate(_lengths(lengths, batch, tokens)):
        size = np.abs(last[b])
        for t in range(n):
            last[b] = f[b, t] * last[b] + rest[b, t] * u[b, t]
            size = f[b, t] * size + rest[b, t] * np.abs(u[b, t])
            last_off[b] = f[b, t] * last_off[b] + STEP * EPS32 * size
            h[b, t], off[b, t] = last[b], last_off[b]
    return {"h": h, "last": last}, {"h": off + rounding(dtype) * np.abs(h), "last": last_off}


def gated_recurrence_backward(gate, x, h, dy, state=None, dlast=None, lengths=None):
    """The gradients of gate, x and the first state, and their bounds."""
    dtype, (batch, tokens, channels) = x.dtype, x.shape
    f, rest, u, out, g = *_gates(gate), as_float64(x), as_float64(h), as_float64(dy)
    dgate, dx = np.zeros(u.shape), np.zeros(u.shape)
    gate_off, x_off = np.zeros(u.shape), np.zeros(u.shape)
    c = np.zeros((batch, channels)) if dlast is None else dlast.astype(np.float64)
    c, c_off = c.copy(), np.zeros((batch, channels))
    first = np.zeros((batch, channels)) if state is None else state.astype(np.float64)
    for b, n in enumerate(_lengths(lengths, batch, tokens)):
        size = np.abs(c[b])
        for t in reversed(range(n)):
            total, size = g[b, t] + c[b], np.abs(g[b, t]) + size
            off = c_off[b] + STEP * EPS32 * size
            before = out[b, t - 1] if t else first[b]
            dx[b, t], x_off[b, t] = rest[b, t] * total, rest[b, t] * (off + 4 * EPS32 * size)
            by = f[b, t] * rest[b, t]
            dgate[b, t] = by * total * (before - u[b, t])
            gate_off[b, t] = by * (off + 8 * EPS32 * size) * (np.abs(before) + np.abs(u[b, t]))
            c[b], c_off[b], size = f[b, t] * total, f[b, t] * off, f[b, t] * size
    fine = rounding(dtype)
    return ({"dgate": dgate, "dx": dx, "dfirst": c},
            {"dgate": gate_off + fine * np.abs(dgate), "dx": x_off + fine * np.abs(dx), "dfirst": c_off + 4 * EPS32 * np.abs(c)})


# ---------------------------------------------------------- cross entropy
def _logits(x, w):
    """Logits, and what sums of `width` products in f32 may be off."""
    x, w = as_float64(x), as_float64(w)
    return x @ w.T, (w.shape[1] / 4 + 16) * EPS32 * (np.abs(x) @ np.abs(w).T)


def cross_entropy(x, w, targets):
    """loss and lse, and their bounds."""
    logits, off = _logits(x, w)
    top = logits.max(1, keepdims=True)
    lse = (top + np.log(np.exp(logits - top).sum(1, keepdims=True)))[:, 0]
    has = targets < w.shape[0]
    at = np.where(has, targets, 0).astype(np.int64)
    picked = logits[np.arange(len(at)), at]
    # The softmax weighs the logits' errors: at most their largest.  An exponential
    # errs by its argument's rounding, which weighs as the term does; the sums of a lane,
    # its wave and the tiles follow one another in fewer than 600 additions.
    lse_off = off.max(1) + EPS32 * (600 + 4 * np.abs(lse) + 4 * np.abs(top[:, 0]))
    loss_off = lse_off + off[np.arange(len(at)), at] + 2 * EPS32 * (np.abs(lse) + np.abs(picked))
    return {"loss": np.where(has, lse - picked, 0.0), "lse": lse}, {"loss": np.where(has, loss_off, 0.0), "lse": lse_off}


def cross_entropy_backward(x, w, targets, lse, grad):
    """The gradients of x and w, and their bounds."""
    dtype = x.dtype
    logits, off = _logits(x, w)
    from_lse = logits - lse.astype(np.float64)[:, None]
    p = np.exp(from_lse)
    hot = targets.astype(np.int64)[:, None] == np.arange(w.shape[0])
    has = (targets < w.shape[0])[:, None]
    by = np.where(has[:, 0], grad.astype(np.float64), 0.0)[:, None]
    g = by * (p - hot)
    x64, w64 = np.where(has, as_float64(x), 0.0), as_float64(w)
    # Of a term: the logit's error and the exponential's; G's rounding to the
    # operands' type, and three more of its quotient, product and difference.
    g_off = np.abs(by) * p * (off + (4 + 2 * np.abs(from_lse)) * EPS32) + np.abs(g) * ((EPS16 if dtype == hx.bfloat16 else 0) + 4 * EPS32)
    dx, dw = g @ w64, g.T @ x64
    fine = rounding(dtype)
    dx_off = g_off @ np.abs(w64) + (w.shape[0] / 4 + 24) * EPS32 * (np.abs(g) @ np.abs(w64)) + (fine + 2 * EPS32) * np.abs(dx)
    dw_off = g_off.T @ np.abs(x64) + (x.shape[0] / 4 + 24) * EPS32 * (np.abs(g).T @ np.abs(x64)) + (fine + 2 * EPS32) * np.abs(dw)
    return {"dx": dx, "dw": dw}, {"dx": dx_off, "dw": dw_off}


def near(got, value, bound, what):
    """Each element within its bound (and below the least float, whose sums are whole)."""
    got = as_float64(got)
    off = np.abs(got - value) - bound
    assert got.shape == value.shape, what
    assert np.all(off <= 2.0**-126), f"{what}: {off.max()} beyond the bound at {np.unravel_index(off.argmax(), off.shape)}"
