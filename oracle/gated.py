"""The gated recurrence and dropout in float64 numpy, token by token -- TEST
INFRASTRUCTURE ONLY.  The reference has neither; the definitions are those of
``include/yufb200.h`` (``yuf_gated_scan_forward``, ``yuf_dropout``).
"""

import numpy as np

from .philox import M0, M1, MASK, W0, W1


def _sigmoid(z):
    return np.where(z >= 0, 1.0 / (1.0 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1.0 + np.exp(-np.abs(z))))


def pieces(B, T, cu):
    """(batch row, first token, end, state row) of every sequence."""
    if cu is None:
        return [(b, 0, T, b) for b in range(B)]
    return [(0, int(cu[s]), int(cu[s + 1]), s) for s in range(len(cu) - 1)]


def gated_scan(x, forget, gate=None, lower=None, state=None, cu=None):
    """``(y, final_state, history h)``; rows of no sequence have y = h = 0."""
    x, f = np.asarray(x, np.float64), np.asarray(forget, np.float64)
    B, T, D = x.shape
    low = np.zeros(D) if lower is None else np.asarray(lower, np.float64)
    rows = B if cu is None else len(cu) - 1
    end = np.zeros((rows, D)) if state is None else np.array(state, np.float64)
    s, m = _sigmoid(f), _sigmoid(-f)
    h = np.zeros((B, T, D))
    for b, lo, hi, r in pieces(B, T, cu):
        cur = end[r].copy()
        for t in range(lo, hi):
            cur = (low + (1 - low) * s[b, t]) * cur + (1 - low) * m[b, t] * x[b, t]
            h[b, t] = cur
        end[r] = cur
    return (h if gate is None else h * _sigmoid(np.asarray(gate, np.float64))), end, h


def gated_scan_grads(x, forget, gate, lower, state, cu, dy, dlast):
    """Gradients as a dict: x, forget, gate, lower, state (those of absent inputs too), and
    ``dh``, the gradient that reaches each h."""
    x, f, dy = (np.asarray(t, np.float64) for t in (x, forget, dy))
    B, T, D = x.shape
    low = np.zeros(D) if lower is None else np.asarray(lower, np.float64)
    rows = B if cu is None else len(cu) - 1
    h0 = np.zeros((rows, D)) if state is None else np.asarray(state, np.float64)
    s, m = _sigmoid(f), _sigmoid(-f)
    sg = np.ones_like(x) if gate is None else _sigmoid(np.asarray(gate, np.float64))
    mg = np.zeros_like(x) if gate is None else _sigmoid(-np.asarray(gate, np.float64))
    h = gated_scan(x, forget, gate, lower, state, cu)[2]
    dh = np.zeros((B, T, D))
    dstate = np.zeros((rows, D)) if dlast is None else np.array(dlast, np.float64)
    prev = np.zeros((B, T, D))
    live = np.zeros((B, T, 1))
    for b, lo, hi, r in pieces(B, T, cu):
        G = dstate[r]
        for t in range(hi - 1, lo - 1, -1):
            live[b, t] = 1
            prev[b, t] = h0[r] if t == lo else h[b, t - 1]
            dh[b, t] = dy[b, t] * sg[b, t] + G
            G = (low + (1 - low) * s[b, t]) * dh[b, t]
        dstate[r] = G
    da = dh * (prev - x) * live
    return {"x": dh * (1 - low) * m, "forget": da * (1 - low) * m * s, "gate": live * dy * h * sg * mg,
            "lower": (da * m).sum((0, 1)), "lower_terms": np.abs(da * m).sum((0, 1)), "state": dstate, "dh": dh,
            "prev": prev}


def philox_words(first, n, seed, step):
    """Words first .. first + n - 1 of the dropout stream of (seed, step)."""
    q = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    c = [q & np.uint64(MASK), q >> np.uint64(32), np.full_like(q, step & MASK), np.full_like(q, (step >> 32) & MASK)]
    k0, k1 = seed & MASK, (seed >> 32) & MASK
    for _ in range(10):
        p0, p1 = np.uint64(M0) * c[0], np.uint64(M1) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & np.uint64(MASK),
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & np.uint64(MASK)]
        k0, k1 = (k0 + W0) & MASK, (k1 + W1) & MASK
    return np.stack(c, 1).reshape(-1)[first % 4:first % 4 + n].astype(np.int64)


def dropout(x, p, seed, step=0, residual=None):
    x = np.asarray(x, np.float64)
    keep = (philox_words(0, x.size, seed, step) >= int(p * 2**32)).reshape(x.shape)
    y = np.where(keep, x / (1.0 - p) if p < 1 else 0.0, 0.0)
    return y if residual is None else y + np.asarray(residual, np.float64)
