"""float64 restatements of the feed-forward operators and of the 8-bit checkpoint format, for the tests: formulas as
include/soliton_b200.h states them, in numpy, with nothing of the kernels' blocking, scaling or order."""
import math

import numpy as np

GROUP = 32
_erf = np.vectorize(math.erf, otypes=[np.float64])
ACTS = {"none": 0, "gelu": 1, "silu": 2}


def act(v, kind):
    v = np.asarray(v, np.float64)
    if kind == "gelu":
        return 0.5 * v * (1.0 + _erf(v / math.sqrt(2.0)))
    return v / (1.0 + np.exp(-v)) if kind == "silu" else v.copy()


def act_grad(v, kind):
    v = np.asarray(v, np.float64)
    if kind == "gelu":
        return 0.5 * (1.0 + _erf(v / math.sqrt(2.0))) + v * np.exp(-0.5 * v * v) / math.sqrt(2.0 * math.pi)
    if kind == "silu":
        sig = 1.0 / (1.0 + np.exp(-v))
        return sig * (1.0 + v * (1.0 - sig))
    return np.ones_like(v)


def linear(x, w, bias=None, residual=None, kind="none"):
    """(y, pre)"""
    pre = np.asarray(x, np.float64) @ np.asarray(w, np.float64).T
    pre = pre if bias is None else pre + np.asarray(bias, np.float64)
    y = act(pre, kind)
    return (y if residual is None else y + np.asarray(residual, np.float64)), pre


def linear_bwd(dy, x, w, pre=None, kind="none"):
    """(dx, dw, db, d) with d the gradient of the pre-activations"""
    d = np.asarray(dy, np.float64)
    if kind != "none":
        d = d * act_grad(pre, kind)
    return d @ np.asarray(w, np.float64), d.T @ np.asarray(x, np.float64), d.sum(0), d


def gated(x, wg, wu, bg=None, bu=None, kind="silu"):
    """(h, g, u)"""
    g, u = linear(x, wg, bg)[1], linear(x, wu, bu)[1]
    return act(g, kind) * u, g, u


def gated_bwd(dh, x, wg, wu, g, u, kind="silu"):
    """(dx, dwg, dwu, dbg, dbu, dg, du)"""
    dh, g, u, x = (np.asarray(t, np.float64) for t in (dh, g, u, x))
    dg, du = dh * u * act_grad(g, kind), dh * act(g, kind)
    dx = dg @ np.asarray(wg, np.float64) + du @ np.asarray(wu, np.float64)
    return dx, dg.T @ x, du.T @ x, dg.sum(0), du.sum(0), dg, du


# ---------------------------------------------------------------- checkpoints

def ck8_exp_offset(rows, cols):
    return (rows * cols + 15) // 16 * 16


def ck8_bytes(rows, cols):
    return ck8_exp_offset(rows, cols) + rows * ((cols + GROUP - 1) // GROUP)


def ck8_save(x):
    """The checkpoint of a float32 matrix: (q int8 rows x cols, exponent bytes rows x groups)."""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    groups = (cols + GROUP - 1) // GROUP
    v = np.zeros((rows, groups * GROUP), np.float64)
    v[:, :cols] = x
    v = v.reshape(rows, groups, GROUP)
    bad = ~np.isfinite(v).all(-1)
    top = np.where(bad, 0.0, np.abs(np.where(np.isfinite(v), v, 0.0)).max(-1))
    e = np.full(top.shape, -126)
    while True:  # the least exponent that fits, one step at a time
        short = 127.0 * np.exp2(e.astype(np.float64)) < top
        if not short.any():
            break
        e = e + short
    q = np.where(bad[..., None], 0.0, np.rint(np.where(np.isfinite(v), v, 0.0) * np.exp2(-e.astype(np.float64))[..., None]))
    return q.reshape(rows, -1)[:, :cols].astype(np.int8), np.where(bad, 255, e + 127).astype(np.uint8)


def ck8_pack(q, eb):
    """One buffer, as the library lays it out."""
    rows, cols = q.shape
    buf = np.zeros(ck8_bytes(rows, cols), np.uint8)
    buf[:rows * cols] = q.reshape(-1).view(np.uint8)
    buf[ck8_exp_offset(rows, cols):] = eb.reshape(-1)
    return buf


def ck8_unpack(buf, rows, cols):
    q = buf[:rows * cols].view(np.int8).reshape(rows, cols)
    return q, buf[ck8_exp_offset(rows, cols):].reshape(rows, -1)


def ck8_values(q, eb):
    step = np.where(eb == 255, np.nan, np.exp2(eb.astype(np.float64) - 127.0))
    return q.astype(np.float64) * np.repeat(step, GROUP, axis=1)[:, :q.shape[1]]
