"""Plain 64-bit forms of the image-network operators (group normalisation,
cross attention, dropout) and bounds on what a correct implementation may
differ by.  Build-defined operators: the formulas are the textbook ones.

The bounds are elementwise and first order, from the standard model of rounding
(each fp32 operation has a relative error of at most U32 = 2^-24; a sum of n
terms in any order one of at most (n - 1) U32 of the sum of magnitudes), with
the type's own rounding where a value is stored in 16 bits."""
from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24
ROUNDING = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # 24, 11 and 8 significant bits, to nearest
# Absolute part of a rounding: half of the smallest fp16 number, and what the model leaves out of fp32 and bf16, the
# underflow of terms below 2^-126 (sums of up to 64 of them).
SMALLEST = {"f32": 2.0 ** -120, "f16": 2.0 ** -25, "bf16": 2.0 ** -120}


def _stored(ref, dtype):
    return ROUNDING[dtype] * np.abs(ref) + SMALLEST[dtype]


# ------------------------------------------------------------ group normalisation


def _act(z, activation):
    """activation(z) and its slope."""
    if activation == "relu":
        return np.maximum(z, 0.0), (z > 0).astype(np.float64)
    if activation == "silu":
        s = 1.0 / (1.0 + np.exp(-z))
        return z * s, s + z * s * (1.0 - s)
    return z, np.ones_like(z)


def group_norm(x, weight, bias, groups, eps=1e-5, activation="none", grad=None):
    """x [images, rows, channels] float64.  Returns y, or with grad a dict of y, dx, dweight, dbias and the magnitudes
    that the bounds need."""
    n, rows, c = x.shape
    w = np.ones(c) if weight is None else weight
    b = np.zeros(c) if bias is None else bias
    xg = x.reshape(n, rows, groups, c // groups)
    mean = xg.mean(axis=(1, 3), keepdims=True)
    std = np.sqrt(xg.var(axis=(1, 3), keepdims=True) + eps)
    xhat = ((xg - mean) / std).reshape(n, rows, c)
    z = xhat * w + b
    y, slope = _act(z, activation)
    # |x|, |mean| and the group's mean |x| over std: what an absolute error of the mean or of x - mean is relative to
    size = ((np.abs(xg) + np.abs(xg).mean(axis=(1, 3), keepdims=True)) / std).reshape(n, rows, c)
    out = dict(y=y, z=z, xhat=xhat, size=size, stats=np.stack([mean, 1.0 / std], -1).reshape(n, groups, 2))
    if grad is None:
        return out
    dz = grad * slope
    dn = (dz * w).reshape(n, rows, groups, c // groups)
    xh = xhat.reshape(dn.shape)
    m1, m2 = dn.mean(axis=(1, 3), keepdims=True), (dn * xh).mean(axis=(1, 3), keepdims=True)
    out.update(dx=((dn - m1 - xh * m2) / std).reshape(n, rows, c), dweight=(dz * xhat).sum((0, 1)),
               dbias=dz.sum((0, 1)))
    # bounds: `e` is the relative error of xhat's parts and of the slope, `n_seq` terms summed one after the other
    e = NORM_TERMS * U32
    z_err = e * (np.abs(w) * (np.abs(xhat) + size) + np.abs(b))
    dz_err = np.abs(grad) * (1.0 * z_err * (activation == "silu") + e)  # |silu''| <= 1
    xh_err = e * (np.abs(xhat) + size)
    mean_abs = lambda t: np.broadcast_to(t.reshape(dn.shape).mean(axis=(1, 3), keepdims=True), dn.shape).reshape(x.shape)
    dna = np.abs(dz * w)
    m2b = np.broadcast_to(np.abs(m2), dn.shape).reshape(x.shape)
    err = (np.abs(w) * dz_err + e * dna + mean_abs(np.abs(w) * dz_err + e * dna) + xh_err * m2b
           + np.abs(xhat) * mean_abs(np.abs(w * xhat) * dz_err + dna * xh_err + e * np.abs(dna * xhat)))
    istd = np.broadcast_to(1.0 / std, dn.shape).reshape(x.shape)
    out.update(dx_err=istd * err, dweight_err=(np.abs(xhat) * dz_err + np.abs(dz) * xh_err + e * np.abs(dz * xhat)).sum((0, 1)),
               dbias_err=(dz_err + e * np.abs(dz)).sum((0, 1)))
    return out


# Terms of a sum that one thread may take one after the other, plus the depth of the tree above them.
NORM_TERMS = 128


def group_norm_bound(ref, weight, bias, dtype):
    """Bound on |y - ref["y"]|: z = w (x - mean) rstd + b with relative errors of NORM_TERMS U32 in the mean, the
    variance and the line, activations of slope at most 1.1, one rounding to the type."""
    c = ref["y"].shape[-1]
    w = np.ones(c) if weight is None else weight
    b = np.zeros(c) if bias is None else bias
    e = NORM_TERMS * U32
    return 1.1 * e * (np.abs(w) * (np.abs(ref["xhat"]) + ref["size"]) + np.abs(b)) + e * np.abs(ref["y"]) \
        + _stored(ref["y"], dtype)


# ------------------------------------------------------------ cross attention


def attention(q, k, v, valid, scale, dtype="f32", grad=None):
    """One head: q [Lq, D], k, v [Lk, D] float64, valid [Lk] bool.  Returns a dict of out, lse, out_err and with grad
    dq, dk, dv and their bounds.  16-bit types: softmax terms and dS are rounded to the type before a product."""
    lq, d = q.shape
    lk = k.shape[0]
    res = dict(out=np.zeros((lq, d)), lse=np.full(lq, -np.inf), out_err=np.zeros((lq, d)), lse_err=np.zeros(lq))
    if grad is not None:
        for name, n in (("dq", lq), ("dk", lk), ("dv", lk)):
            res[name], res[name + "_err"] = np.zeros((n, d)), np.zeros((n, d))
    if not valid.any():
        return res
    ut = 0.0 if dtype == "f32" else 2 * ROUNDING[dtype]  # a rounding and the difference it makes to the denominator
    tiny = 0.0 if dtype == "f32" else 2.0 ** -24          # fp16 terms below the normal range
    kv, vv = k[valid], v[valid]
    n = kv.shape[0]
    s = q @ kv.T * scale
    top = s.max(1, keepdims=True)
    e = np.exp(s - top)
    total = e.sum(1, keepdims=True)
    p = e / total
    out = p @ vv
    # relative error of p: twice the absolute error of s (its own and the denominator's) and a few operations
    ds_abs = (d + 8) * U32 * (np.abs(q) @ np.abs(kv).T) * abs(scale) + 8 * U32 * (1 + np.abs(s - top))
    p_rel = ds_abs + ds_abs.max(1, keepdims=True) + (n + 16) * U32
    p_err = p * (p_rel + ut) + tiny / total
    res["out"], res["lse"] = out, (top + np.log(total))[:, 0]
    res["lse_err"] = (ds_abs.max(1) + (n + 16) * U32 * (1 + np.abs(res["lse"])))
    out_err = p_err @ np.abs(vv) + (n + 4) * U32 * (p @ np.abs(vv))
    res["out_err"] = out_err + _stored(out, dtype)
    if grad is None:
        return res
    g = grad
    delta = (g * out).sum(1, keepdims=True)
    dp = g @ vv.T
    delta_err = (np.abs(g) * (res["out_err"])).sum(1, keepdims=True) + (d + 4) * U32 * (np.abs(g) * np.abs(out)).sum(1, keepdims=True)
    dp_err = (d + 4) * U32 * (np.abs(g) @ np.abs(vv).T)
    ds = p * (dp - delta)
    lse_err = res["lse_err"][:, None]
    pb_rel = ds_abs + lse_err + 8 * U32 * (2 + np.abs(s - top) + np.abs(np.log(total)))
    ds_err = np.abs(ds) * (pb_rel + 8 * U32 + ut) + p * (dp_err + delta_err) + ut * 2.0 ** -10 * np.abs(ds).max()
    scale_abs = abs(scale)
    dq = ds @ kv * scale
    res["dq"] = dq
    res["dq_err"] = scale_abs * (ds_err @ np.abs(kv) + (n + 8) * U32 * (np.abs(ds) @ np.abs(kv))) + _stored(dq, dtype)
    dk = ds.T @ q * scale
    res["dk"][valid] = dk
    res["dk_err"][valid] = scale_abs * (ds_err.T @ np.abs(q) + (lq + 8) * U32 * (np.abs(ds).T @ np.abs(q))) + _stored(dk, dtype)
    pb_err = p * (pb_rel + ut) + tiny
    dv = p.T @ g
    res["dv"][valid] = dv
    res["dv_err"][valid] = pb_err.T @ np.abs(g) + (lq + 8) * U32 * (p.T @ np.abs(g)) + _stored(dv, dtype)
    return res


# ------------------------------------------------------------ dropout


def philox4x32(counter, key, rounds=10):
    """Philox4x32 (Salmon, Moraes, Dror, Shaw, 2011) in Python integers: four words in, two words of key, four out."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_keep(index, p, seed, subsequence):
    """Whether element `index` is kept."""
    block = index // 4
    word = philox4x32([block & 0xFFFFFFFF, block >> 32, subsequence & 0xFFFFFFFF, subsequence >> 32],
                      [seed & 0xFFFFFFFF, seed >> 32])[index % 4]
    return word >= int(p * 2.0 ** 32)


def dropout(x, p, seed, subsequence, residual=None):
    """x float64 of any shape; element by element."""
    keep = np.array([dropout_keep(i, p, seed, subsequence) for i in range(x.size)], bool).reshape(x.shape)
    y = np.where(keep, x / (1.0 - p) if p < 1.0 else 0.0, 0.0)
    return y if residual is None else y + residual
