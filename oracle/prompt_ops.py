"""Plain 64-bit forms of the operators of a prompt's encoder (embedding, root-mean-
square norm, causal attention over one sequence) and bounds on what a correct
implementation may differ by.  Build-defined operators: the formulas are the
textbook ones.  The bounds follow the model of image_ops: each fp32 operation has
a relative error of at most U32, a sum of n terms one of at most (n - 1) U32 of
the sum of magnitudes, and a value stored in a type its rounding."""
from __future__ import annotations

import numpy as np

from .image_ops import ROUNDING, U32, _stored

# ------------------------------------------------------------ embedding


def embedding(tokens, weight, scale):
    """y [n, dim] from tokens [n] and weight [vocab, dim]."""
    known = (tokens >= 0) & (tokens < weight.shape[0])
    return np.where(known[:, None], weight[np.where(known, tokens, 0)], 0.0) * scale


def embedding_bound(y, dtype):
    """One product in fp32, by a scale rounded to fp32, and the rounding."""
    return 2 * U32 * np.abs(y) + _stored(y, dtype)


def embedding_grad(grad, tokens, vocab, scale, dtype):
    """(dweight, bound): sums over all positions of a token."""
    dw, size, count = np.zeros((vocab, grad.shape[1])), np.zeros((vocab, grad.shape[1])), np.zeros((vocab, 1))
    for i, t in enumerate(tokens):
        if 0 <= t < vocab:
            dw[t] += grad[i]
            size[t] += np.abs(grad[i])
            count[t] += 1
    dw = dw * scale
    return dw, (count + 3) * U32 * size * abs(scale) + _stored(dw, dtype)


# ------------------------------------------------------------ root-mean-square norm

# Terms that one thread adds one after the other where a row is in registers (4 pieces of 8), and the tree above them.
ROW_TERMS = 32 + 10


def rms_norm(h, weight, eps, dtype, grad=None, grad_sum=None):
    """h [rows, width] float64, as it is stored.  Returns y, stats and their bounds, the row's scale for 8 bits, and with
    grad dx, dweight and theirs."""
    w = np.ones(h.shape[1]) if weight is None else weight
    rstd = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    xhat = h * rstd
    y = xhat * w
    e = (ROW_TERMS + 8) * U32  # of the mean of squares (all of one sign), half of it in rstd; eps, division, root
    out = dict(y=y, stats=rstd[:, 0], stats_err=e * rstd[:, 0], raw_err=(e + 4 * U32) * np.abs(y),
               scale=np.abs(y).max(1) / 448.0)
    out["y_err"] = out["raw_err"] + _stored(y, dtype)
    out["scale_err"] = (e + 6 * U32) * out["scale"] + 2.0 ** -126
    if grad is None:
        return out
    n = grad * w
    m = (n * xhat).mean(1, keepdims=True)
    size = np.abs(n * xhat).mean(1, keepdims=True)
    dx = rstd * (n - xhat * m)
    # e: of rstd and of xhat; the sum of n xhat has magnitude `size` where m may cancel
    dx_err = rstd * (e + 6 * U32) * (np.abs(n) + np.abs(xhat) * (np.abs(m) + size) * 3)
    if grad_sum is not None:
        dx = dx + grad_sum
        dx_err = dx_err + U32 * np.abs(dx)
    out.update(dx=dx, dx_err=dx_err + _stored(dx, dtype), dweight=(grad * xhat).sum(0),
               dweight_err=(h.shape[0] + ROW_TERMS + 16) * U32 * np.abs(grad * xhat).sum(0))
    return out


def e4m3_bound(ratio):
    """Half a step of e4m3 at y / scale: 2^-4 of the value, 2^-10 below its normal range; a value near the middle of two
    may go to either, which is still within half a step and the fp32 errors of both sides."""
    return 2.0 ** -4 * np.abs(ratio) + 2.0 ** -10 + 2.0 ** -16 * np.abs(ratio)


# ------------------------------------------------------------ causal attention


def causal_attention(q, k, v, scale, dtype="f32", grad=None):
    """One head of one sequence: q [T, D], k, v [S, D] float64; token i sees the states up to i + S - T.  Returns a dict of
    out, lse, out_err and with grad dq, dk, dv and their bounds, as image_ops.attention does; 16-bit types: softmax terms
    and dS are rounded to the type before a product."""
    t, d = q.shape
    n = k.shape[0]
    sees = np.arange(n)[None] <= np.arange(t)[:, None] + n - t
    res = dict(out=np.zeros((t, d)), lse=np.full(t, -np.inf), out_err=np.zeros((t, d)), lse_err=np.zeros(t))
    if grad is not None:
        for name, rows in (("dq", t), ("dk", n), ("dv", n)):
            res[name], res[name + "_err"] = np.zeros((rows, d)), np.zeros((rows, d))
    at = sees.any(1)
    if not at.any():
        return res
    q, sees = q[at], sees[at]
    ut = 0.0 if dtype == "f32" else 2 * ROUNDING[dtype]  # a rounding and the difference it makes to the denominator
    tiny = 0.0 if dtype == "f32" else 2.0 ** -24          # fp16 terms below the normal range
    s = np.where(sees, q @ k.T * scale, -np.inf)
    top = s.max(1, keepdims=True)
    below = np.where(sees, s - top, 0.0)
    e = np.where(sees, np.exp(below), 0.0)
    total = e.sum(1, keepdims=True)
    p = e / total
    out = p @ v
    # relative error of p: twice the absolute error of s (its own and the denominator's) and a few operations
    ds_abs = np.where(sees, (d + 8) * U32 * (np.abs(q) @ np.abs(k).T) * abs(scale) + 8 * U32 * (1 + np.abs(below)), 0.0)
    p_rel = ds_abs + ds_abs.max(1, keepdims=True) + (n + 16) * U32
    p_err = np.where(sees, p * (p_rel + ut) + tiny / total, 0.0)
    lse = top + np.log(total)
    lse_err = ds_abs.max(1, keepdims=True) + (n + 16) * U32 * (1 + np.abs(lse))
    res["out"][at], res["lse"][at], res["lse_err"][at] = out, lse[:, 0], lse_err[:, 0]
    out_err = p_err @ np.abs(v) + (n + 4) * U32 * (p @ np.abs(v)) + _stored(out, dtype)
    res["out_err"][at] = out_err
    if grad is None:
        return res
    g = grad[at]
    delta = (g * out).sum(1, keepdims=True)
    dp = g @ v.T
    delta_err = (np.abs(g) * out_err).sum(1, keepdims=True) + (d + 4) * U32 * (np.abs(g) * np.abs(out)).sum(1, keepdims=True)
    dp_err = (d + 4) * U32 * (np.abs(g) @ np.abs(v).T)
    ds = p * (dp - delta)
    pb_rel = ds_abs + lse_err + 8 * U32 * (2 + np.abs(below) + np.abs(np.log(total)))
    ds_err = np.abs(ds) * (pb_rel + 8 * U32 + ut) + p * (dp_err + delta_err) \
        + np.where(sees, ut * 2.0 ** -10 * np.abs(ds).max(), 0.0)
    dq = ds @ k * scale
    res["dq"][at] = dq
    res["dq_err"][at] = abs(scale) * (ds_err @ np.abs(k) + (n + 8) * U32 * (np.abs(ds) @ np.abs(k))) + _stored(dq, dtype)
    dk = ds.T @ q * scale
    res["dk"] = dk
    res["dk_err"] = abs(scale) * (ds_err.T @ np.abs(q) + (t + 8) * U32 * (np.abs(ds).T @ np.abs(q))) + _stored(dk, dtype)
    dv = p.T @ g
    res["dv"] = dv
    res["dv_err"] = np.where(sees, p * (pb_rel + ut) + tiny, 0.0).T @ np.abs(g) + (t + 8) * U32 * (p.T @ np.abs(g)) \
        + _stored(dv, dtype)
    return res
