"""How far fp32 results of the gated recurrence may be off, element by element, from a
float64 recurrence of the rounding errors -- TEST INFRASTRUCTURE ONLY.

u = 2^-24.  z is an argument of a sigmoid, s = sigmoid(z), m = sigmoid(-z).
* e = 2^(-z log2 e): the constant and the product round by 1.25 |z| u relative to e, the
  base-2 exponential by 2^-22 = 4 u.  s = 1 / (1 + e) takes over the share m of that, plus
  the sum (u) and the reciprocal (1 ulp = 2 u); m = e s takes over the share s, plus u more:
      es = m (1.25 |z| + 4) u + 3 u,   em = s (1.25 |z| + 4) u + 4 u     (relative).
* a = lower + (1 - lower) s is off by da = (1 - lower) s (es + u) + a u; (1 - lower) m x
  relatively by em + 3 u.
* Every way of composing the recurrence sums the same products of a's and one input, each
  bounded in sum by M_t = a_t M_{t-1} + i_t |x_t|, M_0 = |h_0|.  Per token such a product
  takes one more rounding, the sum another, and joining runs of 16 tokens at most 3 per run:
      E_t = a_t E_{t-1} + (da_t + 4 u a_t) M_{t-1} + (em + 5 u) i_t |x_t|.
  A range that is summed from its far end rounds its sum once per token without the sum
  decaying, and a state passes a few joins more: ENDS u M_t on top, for ranges of up to 32
  tokens (two runs: calls of up to 75776 tokens x blocks of 32 or 64 channels).  Second-order terms: a
  factor 1.05.
* The gradient that reaches h_t obeys the same recurrence from the end, in |dy sigmoid(g)|.
* dlower's sum: fp32 within a run of 16 tokens, at most 24 u of its terms' magnitudes.
Results far below the normal range flush: FLOOR.
"""

import numpy as np

from .gated import _sigmoid, gated_scan, gated_scan_grads, pieces

U = 2.0**-24
FLOOR = 1e-36
MORE = 1.05
ENDS = 48


def _factors(z):
    z = np.asarray(z, np.float64)
    s, m = _sigmoid(z), _sigmoid(-z)
    grow = (1.25 * np.minimum(np.abs(z), 90) + 4) * U
    return s, m, m * grow + 3 * U, s * grow + 4 * U


def gated_scan_bounds(x, forget, gate, lower, state, cu, dy=None, dlast=None):
    """``(values, bounds)``, dicts of y, last and, with dy, the gradients x, forget, gate,
    lower and state: what the definition gives, and how far fp32 may be from it before the
    rounding to a narrower type."""
    x, f = np.asarray(x, np.float64), np.asarray(forget, np.float64)
    B, T, D = x.shape
    low = np.zeros(D) if lower is None else np.asarray(lower, np.float64)
    om = 1 - low
    rows = B if cu is None else len(cu) - 1
    h0 = np.zeros((rows, D)) if state is None else np.asarray(state, np.float64)
    y, last, h = gated_scan(x, f, gate, lower, state, cu)
    s, m, es, em = _factors(f)
    a, i = low + om * s, om * m
    da = om * s * (es + U) + a * U
    if gate is None:
        sg, mg, esg, emg = np.ones_like(x), np.zeros_like(x), 0.0, 0.0
    else:
        sg, mg, esg, emg = _factors(gate)
    M, E = np.zeros((B, T, D)), np.zeros((B, T, D))
    Mp, Ep = np.zeros((B, T, D)), np.zeros((B, T, D))  # of the state before the token
    end = np.zeros((rows, D))
    for b, lo, hi, r in pieces(B, T, cu):
        mt, et = np.abs(h0[r]), np.zeros(D)
        for t in range(lo, hi):
            Mp[b, t], Ep[b, t] = mt, et
            ix = i[b, t] * np.abs(x[b, t])
            et = a[b, t] * et + (da[b, t] + 4 * U * a[b, t]) * mt + (em[b, t] + 5 * U) * ix
            mt = a[b, t] * mt + ix
            M[b, t], E[b, t] = mt, et
        end[r] = et + ENDS * U * mt if hi > lo else 0.0
    E, Ep = MORE * (E + ENDS * U * M), MORE * (Ep + ENDS * U * Mp)
    value = {"y": y, "last": last}
    bound = {"y": sg * (E + np.abs(h) * (esg + U)) + FLOOR, "last": MORE * end + FLOOR}
    if dy is None:
        return value, bound
    dy = np.asarray(dy, np.float64)
    w = gated_scan_grads(x, f, gate, lower, state, cu, dy, dlast)
    value.update({k: w[k] for k in ("x", "forget", "gate", "lower", "state")})
    value["dh"], value["prev"] = w["dh"], w["prev"]
    live = np.zeros((B, T, 1))
    Dm, Ed = np.zeros((B, T, D)), np.zeros((B, T, D))
    es0 = np.zeros((rows, D))
    for b, lo, hi, r in pieces(B, T, cu):
        gm, eg = (np.zeros(D) if dlast is None else np.abs(np.asarray(dlast[r], np.float64))), np.zeros(D)
        for t in range(hi - 1, lo - 1, -1):
            live[b, t] = 1
            p = np.abs(dy[b, t]) * sg[b, t]
            dm = p + gm
            ed = eg + (esg if gate is None else esg[b, t] + U) * p + U * dm
            Dm[b, t], Ed[b, t] = dm, ed
            eg = a[b, t] * ed + (da[b, t] + 4 * U * a[b, t]) * dm
            gm = a[b, t] * dm
        es0[r] = MORE * (eg + ENDS * U * gm) if hi > lo else 0.0
    Ed = MORE * (Ed + ENDS * U * Dm)
    gap = np.abs(w["prev"] - x) * live
    term = m * ((Ed + Dm * (em + 3 * U)) * gap + Dm * (Ep + U * gap)) * live
    bound["x"] = i * (Ed + Dm * (em + 4 * U)) + FLOOR
    bound["forget"] = i * s * ((Ed + Dm * (em + es + 6 * U)) * gap + Dm * (Ep + U * gap)) * live + FLOOR
    bound["gate"] = np.abs(dy) * sg * mg * (E + np.abs(h) * (esg + emg + 4 * U)) * live + FLOOR
    bound["lower"] = term.sum((0, 1)) + 24 * U * w["lower_terms"] + FLOOR
    bound["state"] = es0 + FLOOR
    return value, bound


def beyond(got, want, bound, half=0.0, floor=0.0):
    """Largest excess over the bound, <= 0 where got holds; ``half`` and ``floor`` of a
    rounding to a narrower type.  What is not finite is beyond."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    off = np.abs(got - want) - (bound * (1 + half) + half * np.abs(want) + floor)
    return float(np.where(np.isfinite(got), off, np.inf).max(initial=-np.inf))
