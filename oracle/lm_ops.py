"""Definitions of the language-model operators in float64.

Plain NumPy restatements of the formulas in ``include/tlb200.h``, which
the GPU kernels are tested against, and the forward and VJP rules of ``OracleProgram`` for the
ops of the same names.  Arguments are float64 arrays; class indices are integer
arrays in which a value outside [0, classes) names no class.
"""
from __future__ import annotations

import numpy as np


def _hat(v, kind, eps):
    """(norm(v), 1 / scale) along the last axis."""
    if kind == "layer":
        v = v - v.mean(axis=1, keepdims=True)
    r = 1.0 / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)
    return v * r, r


def _hat_vjp(g, hat, r, kind):
    m0 = g.mean(axis=1, keepdims=True) if kind == "layer" else 0.0
    return r * (g - m0 - hat * (g * hat).mean(axis=1, keepdims=True))


def _gate_rows(gate, mode):
    if mode == "none":
        return 1.0
    return gate[:, None] if mode == "token" else gate


def residual_norm(x, u=None, w_post=None, gate=None, gate_mode="none", alpha=1.0, w_pre=None,
                  kind="rms", eps=1e-5):
    """(y, n) with y = alpha x + gate * (norm(u) w_post), n = norm(y) w_pre."""
    y = alpha * x
    if u is not None:
        post = _hat(u, kind, eps)[0]
        if w_post is not None:
            post = post * w_post
        y = y + _gate_rows(gate, gate_mode) * post
    n = _hat(y, kind, eps)[0]
    return y, n if w_pre is None else n * w_pre


def _hat_abs(v, va, r, kind):
    """Magnitudes of the terms of hat(v), va those of v (which cancel where v
    is near its mean)."""
    return r * (va + np.abs(v.mean(axis=1, keepdims=True)) if kind == "layer" else va)


def _hat_vjp_abs(g, hat, r, kind):
    """Magnitudes of _hat_vjp's terms (which cancel where g is near hat), from
    those of g and hat."""
    m0 = g.mean(axis=1, keepdims=True) if kind == "layer" else 0.0
    return r * (g + m0 + hat * (g * hat).mean(axis=1, keepdims=True))


def residual_norm_vjp(x, dy, dn, u=None, w_post=None, gate=None, gate_mode="none", alpha=1.0,
                      w_pre=None, kind="rms", eps=1e-5):
    """Gradients by name, and under ``<name>_abs`` the magnitudes of the terms
    each is the sum of (for error bounds)."""
    wa = 1.0 if w_post is None else w_post
    wb = 1.0 if w_pre is None else w_pre
    g = _gate_rows(gate, gate_mode)
    out = {}
    y, ya = alpha * x, np.abs(alpha * x)
    if u is not None:
        hu, ru = _hat(u, kind, eps)
        hua = _hat_abs(u, np.abs(u), ru, kind)
        y, ya = y + g * hu * wa, ya + np.abs(g * wa) * hua
    G = np.zeros_like(x) if dy is None else dy
    Ga = np.abs(G)
    if dn is not None:
        hy, ry = _hat(y, kind, eps)
        G = G + _hat_vjp(dn * wb, hy, ry, kind)
        hya = _hat_abs(y, ya, ry, kind)
        Ga = Ga + _hat_vjp_abs(np.abs(dn * wb), hya, ry, kind)
        out["dw_pre"] = (dn * hy).sum(axis=0)
        out["dw_pre_abs"] = (np.abs(dn) * hya).sum(axis=0)
    else:
        out["dw_pre"] = out["dw_pre_abs"] = np.zeros(x.shape[1])
    out["dx"], out["dx_abs"] = alpha * G, abs(alpha) * Ga
    if u is None:
        return out
    P, Pa = G * g, Ga * np.abs(g)
    out["dw_post"], out["dw_post_abs"] = (P * hu).sum(axis=0), (Pa * hua).sum(axis=0)
    out["du"] = _hat_vjp(P * wa, hu, ru, kind)
    out["du_abs"] = _hat_vjp_abs(Pa * np.abs(wa), hua, ru, kind)
    t, ta = G * hu * wa, Ga * hua * np.abs(wa)
    if gate_mode in ("channel", "token"):
        axis = 0 if gate_mode == "channel" else 1
        out["dgate"], out["dgate_abs"] = t.sum(axis=axis), ta.sum(axis=axis)
    elif gate_mode == "full":
        out["dgate"], out["dgate_abs"] = t, ta
    return out


def _log_softmax(z):
    """(log softmax, log sum exp) along rows; a row of -inf has lse = -inf and
    no support (its log softmax is -inf)."""
    m = z.max(axis=1, keepdims=True)
    base = np.where(np.isneginf(m), 0.0, m)
    with np.errstate(divide="ignore"):
        log_s = np.log(np.exp(z - base).sum(axis=1, keepdims=True))
    # (z - m) - log s: z - lse would lose log s beside a z of the type's lowest value
    lp = np.where(np.isneginf(log_s), -np.inf, (z - base) - np.where(np.isneginf(log_s), 0.0, log_s))
    lse = base + log_s
    return lp, lse[:, 0]


def distill_topk(z, teacher, index, temperature=1.0, divisor=0.0, upstream=1.0):
    """{loss, row_loss, lse, dz}"""
    rows, classes = z.shape
    ok = (index >= 0) & (index < classes) & ~np.isneginf(teacher)
    some = ok.any(axis=1)
    lp, lse = _log_softmax(z / temperature)
    row_loss = np.zeros(rows)
    dz = np.exp(lp)
    for r in range(rows):
        k = np.nonzero(ok[r])[0]
        if not len(k):
            continue
        lq = teacher[r, k] / temperature
        lq = lq - lq.max()
        lq = lq - np.log(np.exp(lq).sum())
        q = np.exp(lq)
        c = index[r, k].astype(np.int64)
        row_loss[r] = temperature ** 2 * (q * (lq - lp[r, c])).sum()
        np.subtract.at(dz[r], c, q)
    div = divisor if divisor > 0 else max(1, int(some.sum()))
    dz *= np.where(some, temperature * upstream / div, 0.0)[:, None]
    dz[~some] = 0.0
    return {"loss": row_loss.sum() / div, "row_loss": row_loss, "lse": lse, "dz": dz}


def linear_ce(x, w, target, bias=None, divisor=0.0, upstream=1.0):
    """Cross entropy of z = x @ w (+ bias), w [width, classes]:
    {loss, row_loss, lse, dx, dw, dbias}"""
    z = x @ w
    if bias is not None:
        z = z + bias
    rows, classes = z.shape
    ok = (target >= 0) & (target < classes)
    lp, lse = _log_softmax(z)
    r = np.nonzero(ok)[0]
    c = target[r].astype(np.int64)
    row_loss = np.zeros(rows)
    row_loss[r] = -lp[r, c]
    div = divisor if divisor > 0 else max(1, len(r))
    g = np.exp(lp)
    g[r, c] -= 1.0
    g *= np.where(ok, upstream / div, 0.0)[:, None]
    g[~ok] = 0.0
    return {"loss": row_loss.sum() / div, "row_loss": row_loss, "lse": lse,
            "dx": g @ w.T, "dw": x.T @ g, "dbias": g.sum(axis=0), "g": g}
