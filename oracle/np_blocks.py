"""The layer-level operators for blocks of language models (include/qcnn.h: qcnn_op_matvec_w4, qcnn_op_grouped_matmul,
qcnn_op_norm_res) from their definitions, in 64 bits, each with a bound on what a float32 evaluation in any order may be off.

Every function returns (value, bound): `bound` is the first-order error of a float32 evaluation (unit roundoff U = 2^-24 an
operation; a sum of k terms in any order is off by at most k U sum |terms|), doubled for the higher orders.  Half a step of the
output type comes on top, see half_step.
"""
import numpy as np

U = 2.0 ** -24


def half_step(value, eps, tiny):
    """Half a step of the output type at `value`: eps = torch.finfo(t).eps, tiny = its smallest subnormal."""
    return np.maximum(np.abs(value) * eps / 2, tiny / 2)


def matvec_w4(x, w, scale, zero, bias, k, group):
    """x [rows][k]; w uint8 [n][(k + 1) // 2]; scale [groups][n]; zero uint8 [groups][n] or None."""
    n = w.shape[0]
    q = np.empty((n, 2 * w.shape[1]), np.int64)
    q[:, 0::2], q[:, 1::2] = w & 15, w >> 4
    q = q[:, :k]
    of = np.arange(k) // group
    z = np.full((n, k), 8) if zero is None else zero.astype(np.int64)[of].T
    s = scale.astype(np.float64)[of].T
    x = x.astype(np.float64)
    y = x @ (s * (q - z)).T
    # a kernel may sum (q - 8) x and (8 - z) x apart; x in three bfloat16 parts is off by U |x|
    size = np.abs(x) @ (np.abs(s) * (np.abs(q - 8) + np.abs(8 - z))).T
    if bias is not None:
        y = y + bias.astype(np.float64)
        size = size + np.abs(bias.astype(np.float64))
    return y, 2 * (k + 8) * U * size


def act_of(v, act):
    if act == 1:
        return np.maximum(v, 0)
    if act == 2:
        return v / (1 + np.exp(-np.clip(v, -700, 700)))
    return v


def grouped_matmul(x, w, offsets, src, x_scale, w_scale, bias, row_scale, act, y):
    """y [rows][n]: what stands there before; rows outside the offsets keep it.  bound is 0 there."""
    rows, n = y.shape
    experts, _, k = w.shape
    out, bound = y.astype(np.float64).copy(), np.zeros((rows, n))
    w8, x8 = w.astype(np.float64), x.astype(np.float64)
    for e in range(experts):
        lo, hi = max(0, int(offsets[e])), min(rows, int(offsets[e + 1]))
        if lo >= hi:
            continue
        s = np.arange(lo, hi) if src is None else src[lo:hi].astype(np.int64)
        have = (s >= 0) & (s < x.shape[0])
        at = np.where(have, s, 0)
        xv = np.where(have[:, None], x8[at], 0) if x.shape[0] else np.zeros((hi - lo, k))
        v, size = xv @ w8[e].T, np.abs(xv) @ np.abs(w8[e]).T
        if x.dtype == np.int8:
            size = np.abs(v) * 4 / (k + 8)  # exact sums, one rounding to float32
        for f in (w_scale[e][None, :] if w_scale is not None else None, np.where(have, x_scale[at], 1)[:, None] if x_scale is not None else None):
            if f is not None:
                v, size = v * f.astype(np.float64), size * np.abs(f.astype(np.float64))
        if bias is not None:
            v, size = v + bias[e], size + np.abs(bias[e])
        b = 2 * (k + 8) * U * size
        if act == 2:  # |silu'| <= 1.1; e^-v in float32 is off by a few U relative, more where |v| is large
            b = 1.1 * b + (8 + np.abs(v)) * 2 * U * np.abs(act_of(v, 2))
        v = act_of(v, act)
        f = np.ones((hi - lo, 1)) if row_scale is None else row_scale[lo:hi].astype(np.float64)[:, None]
        out[lo:hi], bound[lo:hi] = v * f, (b + 2 * U * np.abs(v)) * np.abs(f)
    return out, bound


def _norm(v, b, kind, w, bias, offset, eps):
    if kind == 0:
        return v, b
    d = v.shape[1]
    if kind == 2:
        m = v.mean(1, keepdims=True)
        b = b + b.mean(1, keepdims=True) + (d + 2) * U * np.abs(v).mean(1, keepdims=True)
        v = v - m
        b = b + U * np.abs(v)
    q = (v * v).mean(1, keepdims=True) + eps
    bq = (2 * np.abs(v) * b).mean(1, keepdims=True) + (d + 4) * U * q  # what the mean of the squares is off by
    inv = 1 / np.sqrt(q)
    rel = 0.5 * bq / q + 4 * U
    f = np.ones(d) if w is None else w.astype(np.float64) + offset
    out = v * inv * f
    bound = b * inv * np.abs(f) + np.abs(out) * (rel + 4 * U)
    if bias is not None:
        out = out + bias.astype(np.float64)
        bound = bound + 2 * U * np.abs(out)
    return out, bound


def gate_of(g, act):
    s = 1 / (1 + np.exp(-np.clip(g, -700, 700)))
    return (g, s, np.tanh(g), g * s)[act]


def norm_res(x, y, index, gate, gate_rows, post, post_w, post_b, pre, pre_w, pre_b, act, alpha, beta, post_eps, pre_eps, w_offset):
    """-> (h, bound, n, bound)."""
    x = x.astype(np.float64)
    rows = x.shape[0]
    alpha, beta, post_eps, pre_eps, w_offset = (float(np.float32(v)) for v in (alpha, beta, post_eps, pre_eps, w_offset))
    h, bh = beta * x, 2 * U * np.abs(beta * x)
    if y is not None:
        y = y.astype(np.float64)
        if index is None:
            v, b = y[:rows], np.zeros_like(x)
        else:
            ok = (index >= 0) & (index < y.shape[0])
            part = np.where(ok[:, :, None], y[np.where(ok, index, 0)], 0)
            v, b = part.sum(1), index.shape[1] * U * np.abs(part).sum(1)
        v, b = _norm(v, b, post, post_w, post_b, w_offset, post_eps)
        if gate is not None:
            g = gate.astype(np.float64)[np.arange(rows) // gate_rows]
            f = gate_of(g, act)
            b = b * np.abs(f) + np.abs(v) * np.abs(f) * (8 + np.abs(g)) * 2 * U + np.abs(v) * (4 * U if act == 2 else 0)
            v = v * f
        h, bh = h + alpha * v, bh + abs(alpha) * (b + 2 * U * np.abs(v)) + 2 * U * np.abs(h + alpha * v)
    n, bn = _norm(h, bh, pre, pre_w, pre_b, w_offset, pre_eps)
    return h, 2 * bh, n, 2 * bn
