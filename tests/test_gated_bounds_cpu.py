"""That the bounds of ``oracle/gated_bounds.py`` hold for fp32 arithmetic and see what they
are there to see: shares, rows and elements that are lost, small ones too."""

import numpy as np
import pytest

from oracle import gated_bounds as gb

NAMES = ("y", "last", "x", "forget", "gate", "lower", "state")
SHAPES = [(2, 1025, 33, None), (1, 2048, 64, None), (2, 2060, 72, None), (37, 300, 32, None), (80, 530, 8, None),
          (1, 9000, 32, [0, 5000, 5001, 8990])]


def sample(B, T, D, cu, seed=0):
    rng = np.random.default_rng(seed)
    rows = B if cu is None else len(cu) - 1

    def t(*shape):
        return np.clip(rng.standard_normal(shape), -4, 4).astype(np.float32)

    return (t(B, T, D), (t(B, T, D) * 1.5 + 2).astype(np.float32), t(B, T, D),
            (rng.random(D) * 0.95).astype(np.float32), t(rows, D), cu, t(B, T, D), t(rows, D))


def in_fp32(x, f, g, low, h0, cu, dy, dlast):
    """The definition token by token in fp32, for one sequence per batch row."""
    one = np.float32(1)
    e, eg = np.exp(-f), np.exp(-g)
    s, sg = one / (one + e), one / (one + eg)
    m, mg = e * s, eg * sg
    om = one - low
    a, i = om * s + low, om * m
    h, prev, dh = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
    cur = h0.copy()
    for t in range(x.shape[1]):
        prev[:, t] = cur
        cur = a[:, t] * cur + i[:, t] * x[:, t]
        h[:, t] = cur
    last, G = cur, dlast.copy()
    for t in range(x.shape[1] - 1, -1, -1):
        dh[:, t] = dy[:, t] * sg[:, t] + G
        G = a[:, t] * dh[:, t]
    d = dh * m * (prev - x)
    return {"y": h * sg, "last": last, "x": dh * i, "forget": dh * i * (prev - x) * s, "gate": dy * h * sg * mg,
            "lower": d.sum((0, 1), dtype=np.float64).astype(np.float32), "state": G}


@pytest.mark.parametrize("B,T,D,cu", [s for s in SHAPES if s[3] is None])
def test_fp32_holds(B, T, D, cu):
    v = sample(B, T, D, cu)
    want, bound = gb.gated_scan_bounds(*v)
    got = in_fp32(*v)
    off = {k: gb.beyond(got[k], want[k], bound[k]) for k in NAMES}
    assert all(o <= 0 for o in off.values()), off


@pytest.mark.parametrize("B,T,D,cu", SHAPES)
def test_what_is_lost_is_seen(B, T, D, cu):
    v = sample(B, T, D, cu)
    want, bound = gb.gated_scan_bounds(*v)

    def seen(name, got):
        return gb.beyond(got, want[name], bound[name]) > 0

    for k in NAMES:
        assert not seen(k, want[k]), k
        assert seen(k, np.zeros_like(want[k])) and seen(k, -want[k]), k
        if k in ("lower", "last", "state"):
            continue
        # at least 99 of 100 elements are above their bound
        at = np.abs(want[k]) > 0
        assert (np.abs(want[k])[at] > bound[k][at]).mean() > 0.99, k
        small = want[k].copy()
        small[np.abs(small) < np.quantile(np.abs(small[at]), 0.05)] = 0
        assert seen(k, small), k
        # the last token of a run of 16, or a whole run, of one row
        for part in (slice(T // 32 * 16 + 15, T // 32 * 16 + 16), slice(T // 32 * 16, T // 32 * 16 + 16)):
            cut = want[k].copy()
            cut[-1, part] = 0
            assert seen(k, cut), k
    # dlower without one batch row's share, without 64 tokens', without 16
    x, f = v[0].astype(np.float64), v[1].astype(np.float64)
    term = want["dh"] * (want["prev"] - x) / (1 + np.exp(f))
    if cu is not None:
        term[:, cu[-1]:] = 0
    np.testing.assert_allclose(term.sum((0, 1)), want["lower"], rtol=1e-6, atol=1e-9)
    if B > 1:
        assert seen("lower", want["lower"] - term[B // 2].sum(0))
    for n in (64, 16):
        at = T // 64 // 2 * 64
        assert seen("lower", want["lower"] - term[0, at:at + n].sum(0)), n
        assert seen("lower", want["lower"] + term[0, at:at + n].sum(0)), n


def test_small_elements_at_both_ends_of_a_gate():
    """sigmoid(-z) as 1 - sigmoid(z) in fp32, and sigmoid(z) as 1 - sigmoid(-z), are seen."""
    x, f, g, low, h0, cu, dy, dl = sample(2, 64, 40, None)
    rng = np.random.default_rng(1)
    wide = rng.uniform(-20, 20, x.shape).astype(np.float32)
    one = np.float32(1)
    v = (x, f, wide, low, h0, cu, dy, dl)
    want, bound = gb.gated_scan_bounds(*v)
    good, s = in_fp32(*v), one / (one + np.exp(-wide))
    assert gb.beyond(good["gate"], want["gate"], bound["gate"]) <= 0
    assert gb.beyond(good["y"] * dy * (one - s), want["gate"], bound["gate"]) > 0
    v = (x, wide, g, low, h0, cu, dy, dl)
    want, bound = gb.gated_scan_bounds(*v)
    good, s = in_fp32(*v), one / (one + np.exp(-wide))
    assert gb.beyond(good["forget"], want["forget"], bound["forget"]) <= 0
    with np.errstate(invalid="ignore"):
        bad = good["forget"] / s * (one - np.exp(-wide) * s)
    assert gb.beyond(bad, want["forget"], bound["forget"]) > 0
