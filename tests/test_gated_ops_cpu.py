"""Gated recurrence and dropout without a GPU: the float64 oracle against
differences and the published generator, and every refusal of the C ABI and of
the Python callables (made on the host, before any CUDA call)."""

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import gated  # noqa: E402
from oracle.philox import philox4x32_10  # noqa: E402
from yufmusicgen_b200 import _lib  # noqa: E402
from yufmusicgen_b200._torch import ops  # noqa: E402
from yufmusicgen_b200.dropout import dropout  # noqa: E402
from yufmusicgen_b200.gated_scan import gated_scan, gated_scan_step  # noqa: E402


@pytest.mark.parametrize("cu", [None, [0, 3, 3, 8]])
def test_oracle_gradients_against_differences(cu):
    rng = np.random.default_rng(5)
    B, T, D = (1, 9, 3) if cu else (2, 7, 3)
    rows = len(cu) - 1 if cu else B
    v = {"x": rng.standard_normal((B, T, D)), "forget": rng.standard_normal((B, T, D)),
         "gate": rng.standard_normal((B, T, D)), "lower": rng.random(D) * 0.9, "state": rng.standard_normal((rows, D))}
    dy, dl = rng.standard_normal((B, T, D)), rng.standard_normal((rows, D))

    def loss(v):
        y, last, _ = gated.gated_scan(v["x"], v["forget"], v["gate"], v["lower"], v["state"], cu)
        return (y * dy).sum() + (last * dl).sum()

    g = gated.gated_scan_grads(v["x"], v["forget"], v["gate"], v["lower"], v["state"], cu, dy, dl)
    for k in v:
        d = rng.standard_normal(v[k].shape)
        e = 1e-5
        diff = (loss({**v, k: v[k] + e * d}) - loss({**v, k: v[k] - e * d})) / (2 * e)
        assert abs(diff - (g[k] * d).sum()) < 1e-7 * max(1.0, abs(diff)), k


def test_oracle_dropout_words_are_the_published_generator():
    seed, step = 0x0123456789ABCDEF, 0xFEDCBA9876543210
    got = gated.philox_words(5, 9, seed, step)
    want = [w for q in range(4) for w in philox4x32_10((q, 0, step & 0xFFFFFFFF, step >> 32),
                                                       (seed & 0xFFFFFFFF, seed >> 32))]
    assert got.tolist() == want[5:14]
    far = gated.philox_words(2**34 + 4, 4, seed, step)  # the counter's second word
    assert far.tolist() == list(philox4x32_10((1, 1, step & 0xFFFFFFFF, step >> 32), (seed & 0xFFFFFFFF, seed >> 32)))


P = 64  # a fake aligned address: the refusals come before any access


def _fwd(x=P, f=P, g=P, strides=None, lower=None, h0=None, cu=None, n=0, y=P, last=P, ck=None, ws=P, dt=0, B=1, T=4,
         D=8):
    return _lib.load().yuf_gated_scan_forward(x, f, g, strides, lower, h0, cu, n, y, last, ck, ws, dt, B, T, D, None)


def _bwd(x=P, f=P, g=P, dy=P, strides=None, cu=None, n=0, ck=P, dx=P, df=P, dg=P, dlower=None, dh0=None, ws=P,
         dt=0, B=1, T=4, D=8):
    return _lib.load().yuf_gated_scan_backward(x, f, g, dy, strides, None, None, cu, n, ck, None, dx, df, dg, dlower,
                                               dh0, ws, dt, B, T, D, None)


@pytest.mark.parametrize("kw, word", [
    (dict(dt=3), "type"), (dict(dt=-1), "type"), (dict(B=-1), "size"), (dict(T=-1), "size"), (dict(D=0), "size"),
    (dict(T=2**30 + 1), "2^30"), (dict(B=2**27, D=64), "too large"), (dict(cu=P, n=2, B=2), "packed"),
    (dict(cu=P, n=-1), "packed"), (dict(x=None), "required"), (dict(f=None), "required"), (dict(y=None), "required"),
    (dict(x=66), "aligned"), (dict(g=65, dt=1), "aligned"), (dict(y=65, dt=2), "aligned"), (dict(last=66), "aligned"),
    (dict(ck=66), "aligned"), (dict(cu=66, n=1), "aligned"), (dict(lower=66), "aligned"), (dict(h0=66), "aligned"),
    (dict(ws=None, T=10**6, D=64), "workspace"), (dict(ws=P + 4), "workspace"),
    (dict(strides=(ctypes.c_int64 * 6)(32, -8, 32, 8, 32, 8)), "negative stride"),
])
def test_forward_refuses_on_the_host(kw, word):
    assert _fwd(**kw) == 1
    assert word in _lib.load().yuf_last_error().decode()


@pytest.mark.parametrize("kw, word", [
    (dict(dt=7), "type"), (dict(D=-4), "size"), (dict(dy=None), "required"), (dict(dx=None), "required"),
    (dict(df=None), "required"), (dict(ck=None), "required"), (dict(dg=None), "dgate"), (dict(ws=None), "workspace"), (dict(ws=P + 8), "workspace"),
    (dict(dx=66), "aligned"), (dict(dg=66), "aligned"), (dict(dh0=66), "aligned"), (dict(cu=P, n=1, B=3), "packed"),
    (dict(strides=(ctypes.c_int64 * 8)(32, 8, 32, 8, 32, 8, -1, 8)), "negative stride"),
])
def test_backward_refuses_on_the_host(kw, word):
    assert _bwd(**kw) == 1
    assert word in _lib.load().yuf_last_error().decode()


def test_step_and_dropout_refuse_on_the_host():
    lib = _lib.load()

    def step(x=P, f=P, g=None, strides=None, lower=None, state=P, ss=8, y=P, dt=0, B=2, D=8):
        return lib.yuf_gated_scan_step(x, f, g, strides, lower, state, ss, y, dt, B, D, None)

    for kw, word in [(dict(dt=9), "type"), (dict(B=-1), "size"), (dict(D=0), "size"), (dict(x=None), "required"),
                     (dict(state=None), "required"), (dict(ss=7), "overlap"), (dict(ss=0), "overlap"),
                     (dict(x=65, dt=1), "aligned"), (dict(state=66), "aligned"),
                     (dict(strides=(ctypes.c_int64 * 3)(8, -8, 8)), "negative stride"), (dict(B=2**30, D=2**30), "large")]:
        assert step(**kw) == 1, kw
        assert word in lib.yuf_last_error().decode(), kw
    assert step(B=0, x=None, state=None) == 0

    def drop(x=P, xs=8, xt=0, r=None, rs=8, out=P, ot=0, rows=2, cols=8, p=0.5, step=None):
        return lib.yuf_dropout(x, xs, xt, r, rs, out, ot, rows, cols, p, 1, 2, step, None)

    for kw, word in [(dict(xt=5), "type"), (dict(p=-0.1), "outside"), (dict(p=1.5), "outside"),
                     (dict(p=float("nan")), "outside"), (dict(rows=-1), "negative"), (dict(cols=-1), "negative"),
                     (dict(rows=2**40, cols=2**40), "too large"), (dict(x=None), "required"), (dict(out=None), "required"),
                     (dict(xs=-8), "stride"), (dict(x=66), "aligned"), (dict(r=66), "aligned"), (dict(step=68), "aligned")]:
        assert drop(**kw) == 1, kw
        assert word in lib.yuf_last_error().decode(), kw
    assert drop(rows=0) == 0 and drop(cols=0, x=None) == 0
    for kw in [dict(xt=1, ot=2), dict(xt=0, ot=1, r=P), dict(xt=2, ot=1)]:  # pairs of types without a kernel
        assert drop(**kw) == 2, kw
        assert "no kernel" in lib.yuf_last_error().decode()


def test_empty_batches_need_no_gpu_and_sizes_are_told():
    lib = _lib.load()
    assert _fwd(B=0, x=None, f=None, y=None) == 0
    assert [lib.yuf_gated_scan_block(d) > 0 for d in (0, 1, 2)] == [True] * 3
    assert [lib.yuf_gated_scan_block(d) for d in (3, -1)] == [0, 0]
    assert lib.yuf_gated_scan_workspace_bytes(3, 100, 64, 1, 1) >= 4 * 3 * 64
    assert lib.yuf_gated_scan_workspace_bytes(1, 10**6, 64, 1, 0) > 0
    for bad in [(3, 100, 64, 9), (-1, 100, 64, 0), (3, -1, 64, 0), (3, 100, 0, 0)]:
        assert lib.yuf_gated_scan_workspace_bytes(*bad, 1) == 0


def test_python_callables_refuse_what_is_not_on_the_gpu():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        gated_scan(x, x)
    with pytest.raises(ValueError, match="shape"):
        gated_scan(x[0], x[0])
    with pytest.raises(ValueError, match="CUDA"):
        gated_scan_step(x[0], x[0], x[0])
    with pytest.raises(ValueError, match="CUDA"):
        dropout(x, 0.1, 1)
    for bad in (None, 3, "x", [1.0]):
        with pytest.raises(TypeError, match="tensor"):
            gated_scan(bad, x)
        with pytest.raises(TypeError, match="tensor"):
            gated_scan(x, x if bad is None else bad, bad if bad is not None else 5)
        with pytest.raises((TypeError, ValueError)):
            dropout(bad, 0.1, 1)
        with pytest.raises(TypeError):
            ops.gated_scan(x, bad)


def test_row_strides():
    """The row stride that dropout's kernel is given, or None where rows have none."""
    t = torch.zeros(4, 6, 10)
    assert ops.row_stride(t) == 10
    assert ops.row_stride(t[:, :, 2:5]) == 10
    assert ops.row_stride(t[:, 1:3]) is None            # two strides
    assert ops.row_stride(t[:, 1:2, :4]) == 60          # axes of one row are not rows
    assert ops.row_stride(t[0, 0]) == 10 and ops.row_stride(t[0, 0, 2:5]) == 3
    assert ops.row_stride(t.transpose(1, 2)) is None
    assert ops.row_stride(t[:, :, :1]) == 10
    assert ops.row_stride(torch.zeros(1, 1, 8).expand(4, 6, 8)) == 0
    assert ops.row_stride(torch.zeros(1, 6, 8).expand(4, 6, 8)) is None
