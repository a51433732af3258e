"""Plain forms, in float64, of the language-model operators (embedding, RMS norm with residual, Linear with activation and
residual, gated recurrence, gradient clipping) and the rounding bounds that their tests hold the library to.

The bounds count roundings.  u(dtype) is half a step, eps / 2; an operation that rounds once is off by at most u times its result, a
sum of n terms by at most (n - 1) u times the sum of their magnitudes whatever its order, and the device's exp by 1 ulp = 2 u, its
erfc by less than 8 ulp = 16 u."""
import numpy as np


def u(dtype):
    return np.finfo(dtype).eps / 2


def erfc(v):
    from scipy.special import erfc as f
    return f(v)


def sigmoid(v):
    e = np.exp(-np.abs(v))
    return np.where(v < 0, e / (1 + e), 1 / (1 + e))


def act(v, name):
    if name == "relu":
        return np.where(v > 0, v, 0.0)
    if name == "gelu":
        return v * (0.5 * erfc(-v / np.sqrt(2.0)))
    if name == "silu":
        return v * sigmoid(v)
    return v


def act_grad(v, name):
    if name == "relu":
        return (v > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * erfc(-v / np.sqrt(2.0)) + v * np.exp(-0.5 * v * v) / np.sqrt(2 * np.pi)
    if name == "silu":
        s = sigmoid(v)
        return s * (1 + v * sigmoid(-v))
    return np.ones_like(v)


# ---- embedding ---------------------------------------------------------------------------------------------------------------
def embedding_fwd(w, ids, scale):
    """In w's own type: the lookup rounds once."""
    out = np.zeros((ids.size, w.shape[1]), w.dtype)
    live = (ids.ravel() >= 0) & (ids.ravel() < w.shape[0])
    out[live] = w[ids.ravel()[live]] * w.dtype.type(scale)
    return out.reshape(ids.shape + (w.shape[1],))


def embedding_bwd(g, ids, vocab, scale):
    """(dW, bound): c tokens of one id make c - 1 additions and one product."""
    g, ids = g.reshape(-1, g.shape[-1]), ids.ravel()
    live = np.flatnonzero((ids >= 0) & (ids < vocab))
    dw, mag, count = (np.zeros((vocab, g.shape[1])) for _ in range(3))
    np.add.at(dw, ids[live], g[live].astype(np.float64))
    np.add.at(mag, ids[live], np.abs(g[live]).astype(np.float64))
    np.add.at(count, ids[live], 1.0)
    s = float(g.dtype.type(scale))
    return dw * s, 1.01 * (count + 1) * u(g.dtype) * mag * abs(s)


# ---- RMS norm ------------------------------------------------------------------------------------------------------------------
def sum_depth(dim):
    """Additions between a term of a row's sum and the sum: at most 16 in a thread up to 16384 elements (dim / 1024 beyond), 6 in
    the wave's tree, 16 over the waves."""
    return max(16, -(-dim // 1024)) + 6 + 16


def rmsnorm_fwd(x, w, eps, res=None):
    """h in the tensors' own type (one rounding, the same on both sides), y and rstd in float64 from it."""
    h = x if res is None else x + res
    h64 = h.astype(np.float64)
    rstd = 1 / np.sqrt((h64 * h64).mean(-1) + eps)
    return h, h64 * rstd[..., None] * w, rstd


def rmsnorm_rel(dim, dtype):
    """Relative error of rstd: the sum of squares (positive terms: one rounding per square and addition), / dim, + eps, sqrt, 1 / x;
    the first four count half.  eps rounded to the type adds one more."""
    return ((sum_depth(dim) + 4) / 2 + 2) * u(dtype)


def rmsnorm_bwd(dy, h, w, rstd, dh=None):
    """(dx, dw, bound of dx, bound of dw)"""
    dt = dy.dtype
    dy, h, w, r = dy.astype(np.float64), h.astype(np.float64), w.astype(np.float64), rstd.astype(np.float64)[:, None]
    dim, n = h.shape[1], h.shape[0]
    g = dy * w
    q = (g * h).mean(1, keepdims=True) * r * r
    dx = r * (g - h * q)
    absq = np.abs(g * h).mean(1, keepdims=True) * r * r
    # q: 2 roundings per term, the tree, / dim, r * r and the product; then g: 1, h q: 1, the difference and the product with r: 2
    bdx = u(dt) * r * (4 * np.abs(g) + np.abs(h) * absq * (sum_depth(dim) + 8))
    if dh is not None:
        dx = dx + dh
        bdx = bdx + u(dt) * (np.abs(dh) + np.abs(dx))
    dw = (dy * (h * r)).sum(0)
    return dx, dw, 1.01 * bdx, 1.01 * u(dt) * (n + 2) * np.abs(dy * (h * r)).sum(0)


# ---- Linear with activation and residual -------------------------------------------------------------------------------------------
def linear_fwd(a, b, bias, name, res):
    """(C, pre, bound of C, bound of pre) for a [M, K], b [K, N]: K products and K - 1 additions in any order, the bias' addition.
    The activations' slopes stay below 1.13; forming their argument costs 2 u, their value 24 u (exp or erfc, sum, quotient, product)."""
    dt = a.dtype
    a64, b64 = a.astype(np.float64), b.astype(np.float64)
    pre = a64 @ b64
    mag = np.abs(a64) @ np.abs(b64)
    if bias is not None:
        pre = pre + bias
        mag = mag + np.abs(bias)
    bpre = (a.shape[1] + 1) * u(dt) * mag
    y = act(pre, name)
    by = bpre if name == "none" else 1.13 * (bpre + 2 * u(dt) * np.abs(pre)) + 24 * u(dt) * np.abs(y)
    if res is not None:
        y = y + res
        by = by + u(dt) * np.abs(y)
    return y, pre, 1.01 * by + np.finfo(dt).tiny, 1.01 * bpre


def linear_bwd(dy, w, x, pre, name):
    """((dx, dw, db, dpre), bounds).  The activations' derivatives lie in -0.2 .. 1.2; their terms are rounded to 30 u of 1.2."""
    dt = dy.dtype
    dy64, w64, x64, p = dy.astype(np.float64), w.astype(np.float64), x.astype(np.float64), pre.astype(np.float64)
    slope = act_grad(p, name)
    dpre = dy64 * slope
    bd = u(dt) * np.abs(dpre) if name in ("none", "relu") else np.abs(dy64) * 36 * u(dt)
    top = np.abs(dpre) + bd
    bx = bd @ np.abs(w64) + (w.shape[0] + 1) * u(dt) * (top @ np.abs(w64))
    bw = bd.T @ np.abs(x64) + (dy.shape[0] + 1) * u(dt) * (top.T @ np.abs(x64))
    bb = bd.sum(0) + (dy.shape[0] + 1) * u(dt) * top.sum(0)
    return (dpre @ w64, dpre.T @ x64, dpre.sum(0), dpre), tuple(1.01 * b + np.finfo(dt).tiny for b in (bx, bw, bb, bd))


# ---- gated recurrence ---------------------------------------------------------------------------------------------------------------
# A gate is off by at most 6 u (exp 2, sum 1, quotient 1, product 1, and one spare), its product 1 more, a step's addition 1; maps of
# pieces add a product and an addition per level, of which there is less than one per step.  12 u of the magnitudes per step.
STEP = 12


def recurrence_fwd(z, x, h0):
    dt = z.dtype
    f, k = sigmoid(z.astype(np.float64)), sigmoid(-z.astype(np.float64))
    B, T, D = z.shape
    h, bound = np.zeros((B, T, D)), np.zeros((B, T, D))
    state = np.zeros((B, D)) if h0 is None else h0.astype(np.float64)
    mag, err = np.abs(state), np.zeros((B, D))
    for t in range(T):
        state = f[:, t] * state + k[:, t] * x[:, t]
        mag = f[:, t] * mag + k[:, t] * np.abs(x[:, t])
        err = f[:, t] * err + STEP * u(dt) * mag
        h[:, t], bound[:, t] = state, err
    return h, 1.01 * bound + np.finfo(dt).tiny


def recurrence_bwd(dh, z, x, h, h0, dh_next):
    """((dz, dx, dh0), bounds)"""
    dt = z.dtype
    f, k = sigmoid(z.astype(np.float64)), sigmoid(-z.astype(np.float64))
    dh, x, h = dh.astype(np.float64), x.astype(np.float64), h.astype(np.float64)
    B, T, D = z.shape
    C = np.zeros((B, D)) if dh_next is None else dh_next.astype(np.float64)
    mag, err = np.abs(C), np.zeros((B, D))
    dz, dx, bz, bx = (np.zeros((B, T, D)) for _ in range(4))
    for t in reversed(range(T)):
        S, Smag = dh[:, t] + C, np.abs(dh[:, t]) + mag
        Serr = err + u(dt) * Smag
        before = h[:, t - 1] if t else (np.zeros((B, D)) if h0 is None else h0.astype(np.float64))
        e = before - x[:, t]
        dx[:, t], dz[:, t] = k[:, t] * S, S * e * f[:, t] * k[:, t]
        bx[:, t] = k[:, t] * (Serr + 8 * u(dt) * Smag)
        bz[:, t] = f[:, t] * k[:, t] * np.abs(e) * (Serr + 18 * u(dt) * Smag)
        C, mag = f[:, t] * S, f[:, t] * Smag
        err = f[:, t] * err + STEP * u(dt) * mag
    return (dz, dx, C), tuple(1.01 * b + np.finfo(dt).tiny for b in (bz, bx, err))


# ---- clipping ---------------------------------------------------------------------------------------------------------------------------
def clip(gs, max_norm):
    """(outs, norm) in float64; a norm that is not finite scales nothing."""
    norm = np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in gs))
    coef = max_norm / norm if np.isfinite(norm) and norm > max_norm else 1.0
    return [g.astype(np.float64) * coef for g in gs], norm


def norm_rel(n, dtype):
    """One rounding of the norm to the type, and n squares and additions in double."""
    return u(dtype) + (n + 4) * u(np.float64)
