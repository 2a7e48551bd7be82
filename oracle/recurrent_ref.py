"""CPU ORACLE — test infrastructure only.

float64 numpy definitions of the layer norm and the gated linear recurrence
of kmamba_b200.h, forward and adjoint, and for each output a bound on the
error of an fp32 evaluation.  The bounds are first-order: a relative error
per elementary step (U = 2^-24, half a step of fp32) carried through the
same sums and recurrences as the values, on absolute values.

Elementary steps.  A special function (exp2, reciprocal, square root) is
allowed 4 U, its rounded argument |z| U per unit of relative sensitivity;
sigmoid(z) then has (16 + 2 |z|) U, the decay exponent u the same, and the
input term b = root i x, with two gates and a root, (32 + 2 |z_r| + 2 |z_i|)
U.  A sum of n terms whose longest chain of additions is `depth` has depth U
times the sum of absolute values.
"""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24


def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def softplus(v):
    return np.logaddexp(0.0, v)


# ------------------------------------------------------------- layer norm
def ln_fwd(x, w, b, eps):
    """x [rows, D]; w, b [D] or None.  Returns (y, mean, rstd) and their bounds."""
    D = x.shape[1]
    w = np.ones(D) if w is None else w
    b = np.zeros(D) if b is None else b
    mean = x.mean(1, keepdims=True)
    c = x - mean
    rstd = 1.0 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    y = c * rstd * w + b
    # chains of at most D / 32 additions in a lane, 5 + 5 across lanes and warps
    depth = D / 32 + 16
    e_mean = depth * U * np.abs(x).mean(1, keepdims=True)
    # the squares' mean: its own sum, and the mean's error (first order: 2 avg(c) = 0, second: e_mean^2)
    rel = (depth + 8) * U + 0.5 * (e_mean * rstd) ** 2
    e_y = np.abs(w) * (rstd * (e_mean + 2 * U * np.abs(x)) + np.abs(c * rstd) * (rel + 4 * U)) \
        + 2 * U * (np.abs(y) + np.abs(b))
    return (y, mean[:, 0], rstd[:, 0]), (e_y, e_mean[:, 0] + U * np.abs(mean[:, 0]), (rstd * rel)[:, 0])


def ln_bwd(x, w, dy, eps, dres=None, mean=None, rstd=None):
    """(dx, dweight, dbias) and their bounds.  mean / rstd given: taken as exact."""
    rows, D = x.shape
    given = mean is not None
    (_, m, r), (_, e_m, e_r) = ln_fwd(x, None, None, eps)
    m, r = (mean, rstd) if given else (m, r)
    if given:
        e_m, e_r = 0 * e_m, 0 * e_r
    m, r, e_m, e_r = (v[:, None] for v in (m, r, e_m, e_r))
    w = np.ones(D) if w is None else w
    xh = (x - m) * r
    e_xh = r * (e_m + U * (np.abs(x) + np.abs(m))) + np.abs(xh) * (e_r / r + 2 * U)
    g = dy * w
    s1, s2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    depth = D / 32 + 20
    e_s1 = depth * U * np.abs(g).mean(1, keepdims=True)
    e_s2 = depth * U * np.abs(g * xh).mean(1, keepdims=True) + (np.abs(g) * e_xh).mean(1, keepdims=True)
    dx = r * (g - s1 - xh * s2)
    e_dx = r * (4 * U * (np.abs(g) + np.abs(s1) + np.abs(xh * s2)) + e_s1 + np.abs(xh) * e_s2
                + np.abs(s2) * e_xh) + np.abs(dx) * (e_r / r + 2 * U)
    if dres is not None:
        dx = dx + dres
        e_dx = e_dx + U * (np.abs(dx) + np.abs(dres))
    rdepth = min(rows, 2048) + 16
    dw, db = (dy * xh).sum(0), dy.sum(0)
    e_dw = (np.abs(dy) * e_xh).sum(0) + rdepth * U * np.abs(dy * xh).sum(0)
    e_db = rdepth * U * np.abs(dy).sum(0)
    return (dx, dw, db), (e_dx, e_dw, e_db)


# ------------------------------------------------ gated linear recurrence
def glr_gates(x, gr, gi, decay, scale):
    r, i = sigmoid(gr), sigmoid(gi)
    u = scale * softplus(decay) * r
    one = -np.expm1(-2 * u)
    root = np.sqrt(one)
    kappa = np.where(u > 1e-8, u * np.exp(-2 * u) / np.where(one > 0, one, 1.0), 0.5)
    e_u = (16 + 2 * np.minimum(np.abs(gr), 200)) * U
    e_b = (32 + 2 * np.minimum(np.abs(gr), 200) + 2 * np.minimum(np.abs(gi), 200)) * U
    return {"r": r, "i": i, "r1": sigmoid(-gr), "i1": sigmoid(-gi), "u": u, "a": np.exp(-u), "root": root, "b": root * i * x, "kappa": kappa,
            "e_u": e_u, "e_b": e_b}


def glr_fwd(x, gr, gi, decay, scale, h0, first=None):
    """One sequence: x, gr, gi [L, D], h0 [D].  Returns (h [L, D], bound)."""
    q = glr_gates(x, gr, gi, decay, scale)
    h, e = h0.astype(np.float64), np.zeros_like(h0, dtype=np.float64)
    hs, es = np.empty_like(q["b"]), np.empty_like(q["b"])
    for t in range(x.shape[0]):
        e = q["a"][t] * e + q["a"][t] * q["u"][t] * q["e_u"][t] * np.abs(h) + q["e_b"][t] * np.abs(q["b"][t])
        h = q["a"][t] * h + q["b"][t]
        e = e + 4 * U * np.abs(h)
        hs[t], es[t] = h, e
    return hs, es


def glr_bwd(x, gr, gi, decay, scale, h0, dy, dh_last):
    """One sequence.  Returns ({dx, dgate_r, dgate_i, udu, dh0}, the same of
    bounds); ddecay = sigmoid(decay) / softplus(decay) sum_t udu."""
    L = x.shape[0]
    q = glr_gates(x, gr, gi, decay, scale)
    hs, es = glr_fwd(x, gr, gi, decay, scale, h0)
    hp = np.concatenate([h0[None], hs[:-1]]) if L else hs
    ep = np.concatenate([np.zeros_like(h0)[None], es[:-1]]) if L else es
    c, ec = dh_last.astype(np.float64), np.zeros_like(dh_last, dtype=np.float64)
    out = {k: np.empty_like(q["b"]) for k in ("dx", "dgate_r", "dgate_i", "udu")}
    err = {k: np.empty_like(q["b"]) for k in out}
    for t in range(L - 1, -1, -1):
        a, u, b = q["a"][t], q["u"][t], q["b"][t]
        G = dy[t] + c
        eG = ec + 2 * U * (np.abs(G) + np.abs(c))
        share, mem = q["kappa"][t] * b, u * a * hp[t]
        udu = G * (share - mem)
        # a relative error e of u is (1 - u) e of u a = u e^-u, and at most
        # (1 + 2 u) e of kappa = u / (e^2u - 1)
        e = (1 + 2 * u) * q["e_u"][t] + q["e_b"][t]
        e_udu = eG * np.abs(share - mem) + np.abs(G) * (e * (np.abs(share) + np.abs(mem)) + u * a * ep[t])
        out["udu"][t], err["udu"][t] = udu, e_udu
        out["dx"][t] = G * q["root"][t] * q["i"][t]
        err["dx"][t] = (eG + np.abs(G) * q["e_b"][t]) * q["root"][t] * q["i"][t]
        out["dgate_r"][t] = udu * q["r1"][t]
        err["dgate_r"][t] = e_udu * q["r1"][t] + np.abs(udu) * (q["r"][t] * q["e_u"][t] + 2 * U)
        out["dgate_i"][t] = G * b * q["i1"][t]
        err["dgate_i"][t] = (eG + np.abs(G) * q["e_b"][t]) * np.abs(b) * q["i1"][t] \
            + np.abs(G * b) * (q["i"][t] * q["e_b"][t] + 2 * U)
        c = a * G
        ec = a * eG + np.abs(c) * (u * q["e_u"][t] + 2 * U)
    out["dh0"], err["dh0"] = c, ec
    return out, err


def decay_ratio(decay):
    return np.where(decay < -30, 1.0, sigmoid(decay) / np.maximum(softplus(decay), 1e-300))


def sequences(batch, L, offsets=None):
    """(first row, row after the last) of each sequence in the flat rows."""
    if offsets is None:
        return [(b * L, (b + 1) * L) for b in range(batch)]
    return [(int(offsets[b]), int(offsets[b + 1])) for b in range(batch)]


def glr(x, gr, gi, decay, scale, seqs, h0=None, dy=None, dh_last=None):
    """All sequences over flat rows [rows, D]; rows outside every sequence
    are NaN in the results.  Returns (values, bounds) dicts."""
    rows, D = x.shape
    n = len(seqs)
    h0 = np.zeros((n, D)) if h0 is None else h0
    names = ["y"] + (["dx", "dgate_r", "dgate_i"] if dy is not None else [])
    val = {k: np.full((rows, D), np.nan) for k in names}
    bnd = {k: np.full((rows, D), np.nan) for k in names}
    for d in (val, bnd):
        d["h_last"] = np.zeros((n, D))
        if dy is not None:
            d["dh0"], d["ddecay"] = np.zeros((n, D)), np.zeros(D)
    total = np.zeros(D)
    ratio = decay_ratio(decay)
    for s, (lo, hi) in enumerate(seqs):
        sl = slice(lo, hi)
        h, e = glr_fwd(x[sl], gr[sl], gi[sl], decay, scale, h0[s])
        val["y"][sl], bnd["y"][sl] = h, e
        val["h_last"][s], bnd["h_last"][s] = (h[-1], e[-1]) if hi > lo else (h0[s], 0.0)
        if dy is None:
            continue
        dl = np.zeros(D) if dh_last is None else dh_last[s]
        o, eo = glr_bwd(x[sl], gr[sl], gi[sl], decay, scale, h0[s], dy[sl], dl)
        for k in ("dx", "dgate_r", "dgate_i"):
            val[k][sl], bnd[k][sl] = o[k], eo[k]
        val["dh0"][s], bnd["dh0"][s] = o["dh0"], eo["dh0"]
        val["ddecay"] += ratio * o["udu"].sum(0)
        bnd["ddecay"] += ratio * eo["udu"].sum(0)
        total += ratio * np.abs(o["udu"]).sum(0)
    if dy is not None:
        # chains of sums: rows of a tile, then tiles; the ratio's own functions
        bnd["ddecay"] += (min(rows, 2048) + 64) * U * total
    return val, bnd
