"""GPU parity of the gated recurrence (yufmusicgen_b200/gated_scan.py) with its
definition in float64 (oracle/gated.py) on the very inputs the kernel gets.

Tolerance.  u = 2^-24.  In sigmoid(z) and sigmoid(-z): rounding z log2(e) gives a
relative error of at most |z| u in e^-z (|z| <= 8 here), the base-2 exponential 2 ulp
= 4 u, the sum, the reciprocal (1 ulp = 2 u) and the product 4 u: 16 u relative.  A
state is h + i (x - h) with i = (1 - lower) sigmoid(-f) off by 17 u relatively, which
moves the steady state by at most 17 u (|x| + |h|), and a step rounds 4 times (a twice,
i x, the FMA): 4 u max(|x|, |h|) each, summed over the n = min(T, 1 / min i) steps that
a state remembers.  With X = max |x| + max |h|:
    |h error| <= (17 + 4 n) u X,
runs joined in another order (block maps) at most double the roundings, so
    K = (64 + 8 n) u is the bound used, times the magnitudes each output is made of:
    y, h_last: X;  dx, dh0: max |dh|;  dforget: max |dh| max |h_{t-1} - x|;
    dgate: max |dy| X;  dlower: the sum of its terms' magnitudes (+ 64 u for the sum).
dforget and dlower also carry h's own error times dh: X instead of |h - x|.
Outputs of a 16-bit type are rounded once: half a step, eps / 2 relative (fp16 below
its normal range: 2^-25 absolute).
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from oracle import gated  # noqa: E402
from yufmusicgen_b200.gated_scan import gated_scan, gated_scan_step  # noqa: E402

DEV = "cuda:0"
U = 2.0**-24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def near(got, want, bound, what):
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    g, floor = f64(got), 2.0**-25 if got.dtype == torch.float16 else 0.0
    assert g.shape == want.shape, what
    off = np.abs(g - want) - (np.asarray(bound) * (1 + half) + half * np.abs(want) + floor)
    assert np.isfinite(g).all() and (off <= 0).all(), f"{what}: beyond the bound by {np.nanmax(off):.3g}"


def make(B, T, D, dtype, gate=True, lower=True, state=True, cu=None, seed=0):
    rng = np.random.default_rng(seed)
    rows = B if cu is None else len(cu) - 1

    def t(*shape, scale=1.0, shift=0.0, dt=DT[dtype]):
        a = np.clip(rng.standard_normal(shape), -4, 4) * scale + shift
        return torch.from_numpy(a.astype(np.float32)).to(DEV).to(dt)

    return {"x": t(B, T, D), "forget": t(B, T, D, scale=1.5, shift=2.0), "gate": t(B, T, D) if gate else None,
            "lower": torch.from_numpy((rng.random(D) * 0.95).astype(np.float32)).to(DEV) if lower else None,
            "state": t(rows, D, dt=torch.float32) if state else None,
            "cu": None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV),
            "dy": t(B, T, D), "dlast": t(rows, D, dt=torch.float32)}


def check(v, got, grads=None):
    """got = (y, last); grads by name; v the inputs as the kernel got them."""
    cu = None if v["cu"] is None else v["cu"].tolist()
    a = [f64(v[k]) for k in ("x", "forget", "gate", "lower", "state")]
    y, last, h = gated.gated_scan(*a, cu)
    T, D = h.shape[1:]
    low = 0.0 if a[3] is None else a[3]
    share = ((1 - low) / (1 + np.exp(a[1]))).reshape(-1, D).min(0) if h.size else np.ones(D)
    K = (64 + 8 * np.minimum(T, 1 / share)) * U  # per channel
    X = max(np.abs(t).max() if t is not None and t.size else 0.0 for t in (a[0], h, a[4])) * 2
    near(got[0], y, K * X, "y")
    near(got[1], last, K * X, "final state")
    if grads is None:
        return
    dy, dl = f64(v["dy"]), f64(v["dlast"])
    w = gated.gated_scan_grads(*a, cu, dy, dl)
    dh = max(np.abs(w["dh"]).max() if w["dh"].size else 0.0, np.abs(dl).max() if dl.size else 0.0)
    near(grads["x"], w["x"], K * dh, "dx")
    near(grads["forget"], w["forget"], 2 * K * dh * X, "dforget")
    if a[2] is not None:
        near(grads["gate"], w["gate"], K * np.abs(dy).max(initial=0.0) * X, "dgate")
    if a[3] is not None:
        n = h.shape[0] * T
        near(grads["lower"], w["lower"], w["lower_terms"] * 64 * U + 2 * K * n * dh * X, "dlower")
    if a[4] is not None:
        near(grads["state"], w["state"], K * dh, "dstate")


NAMES = ("x", "forget", "gate", "lower", "state")


def train(v):
    leaves = {k: v[k].detach().clone().requires_grad_(True) for k in NAMES if v[k] is not None}
    y, last = gated_scan(leaves["x"], leaves["forget"], leaves.get("gate"), leaves.get("lower"), leaves.get("state"),
                         v["cu"])
    g = torch.autograd.grad((y, last), list(leaves.values()), (v["dy"], v["dlast"]))
    return (y, last), dict(zip(leaves, g))


def infer(v):
    return gated_scan(v["x"], v["forget"], v["gate"], v["lower"], v["state"], v["cu"])


SHAPES = [(1, 1, 1), (2, 7, 33), (3, 16, 64), (1, 17, 2), (2, 129, 40), (1, 300, 130), (2, 1025, 66), (1, 2048, 640),
          (5, 64, 31), (300, 3, 10), (1, 1100, 64), (2, 2060, 72), (37, 300, 64), (80, 530, 16), (150, 290, 8),
          (80, 300, 17)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_forward_and_gradients(B, T, D, dtype):
    v = make(B, T, D, dtype, seed=B + T + D)
    got, grads = train(v)
    check(v, got, grads)
    y, last = infer(v)  # without saved states: the same values
    assert torch.equal(y, got[0]) and torch.equal(last, got[1])


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("lower", [False, True])
@pytest.mark.parametrize("state", [False, True])
def test_optional_inputs(gate, lower, state):
    v = make(2, 145, 70, "fp32", gate, lower, state, seed=3)
    check(v, *train(v))


PACKED = [([0, 5, 5, 40, 41, 300], 300), ([0, 0, 0, 64], 64), ([0, 0], 7), ([0, 1, 2, 3], 3), ([0, 128, 256], 256),
          ([0, 127, 129, 129, 129, 1000], 1100), ([0], 5), ([0, 0, 0], 0), ([0, 700], 700), ([0, 5000, 5001, 9000], 9000), ([0, 200, 200, 257, 260], 270)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 37])
@pytest.mark.parametrize("cu,T", PACKED)
def test_packed_sequences(cu, T, D, dtype):
    v = make(1, T, D, dtype, cu=cu, seed=T + D)
    got, grads = train(v)
    check(v, got, grads)
    end = cu[-1]
    for t in (got[0], grads["x"], grads["forget"], grads["gate"]):
        assert not t[:, end:].any()


@pytest.mark.parametrize("gate,state", [(False, False), (True, False), (False, True)])
def test_packed_without_optional_inputs(gate, state):
    v = make(1, 500, 66, "fp16", gate, False, state, cu=[0, 100, 100, 355, 480], seed=8)
    check(v, *train(v))


@pytest.mark.parametrize("T", [40, 700])
def test_many_short_and_empty_sequences(T):
    """Sequences of one token, and dozens of empty ones at one place."""
    cu = sorted(list(range(0, 30)) + [17] * 40 + [31] * 33 + [33, 38])
    v = make(1, T, 24, "fp32", cu=cu, seed=T)
    check(v, *train(v))


@pytest.mark.parametrize("D", [2600, 2601])
def test_packed_wide_rows(D):
    """So many columns that a block walks a packed row by itself, in several steps."""
    cu = [0, 100, 100, 430, 590]
    v = make(1, 600, D, "bf16", cu=cu, seed=D)
    got, grads = train(v)
    check(v, got, grads)
    assert not got[0][:, 590:].any() and not grads["gate"][:, 590:].any()


def test_packed_equals_each_sequence_alone_and_shields_it():
    """An infinite state, or NaN and infinities behind the last row, stay where they are."""
    cu = [0, 37, 37, 300, 513]
    v = make(1, 600, 48, "fp32", cu=cu, seed=9)
    clean, cgrads = train(v)
    for s in range(4):
        one = {**v, "cu": None, "state": v["state"][s:s + 1], "dlast": v["dlast"][s:s + 1],
               **{k: v[k][:, cu[s]:cu[s + 1]] for k in ("x", "forget", "gate", "dy")}}
        y, last = infer(one)
        torch.testing.assert_close(clean[0][:, cu[s]:cu[s + 1]], y, rtol=1e-4, atol=1e-5)
        torch.testing.assert_close(clean[1][s:s + 1], last, rtol=1e-4, atol=1e-5)
    for k in ("x", "forget", "gate", "dy"):
        v[k][:, 513:] = float("nan")
        v[k][:, 550:] = float("inf")
    got, grads = train(v)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    for k in NAMES:
        assert torch.equal(grads[k], cgrads[k]), k
    v["x"][0, 36] = float("inf")          # ends the first sequence with an infinite state
    v["state"][2, 0] = float("nan")       # and the third starts with NaN in one channel
    got, grads = train(v)
    assert torch.isinf(got[1][0]).all() and torch.equal(got[1][1], clean[1][1])
    assert torch.equal(got[0][:, 37:300, 1:], clean[0][:, 37:300, 1:])
    assert torch.equal(got[0][:, 300:], clean[0][:, 300:]) and torch.equal(got[1][3], clean[1][3])
    assert torch.equal(grads["x"][:, 300:], cgrads["x"][:, 300:])
    assert torch.equal(grads["forget"][:, 300:], cgrads["forget"][:, 300:])
    v["dy"][0, 300] = float("nan")        # the fourth sequence's gradient does not reach the third
    grads = train(v)[1]
    assert torch.equal(grads["x"][:, 37:300, 1:], cgrads["x"][:, 37:300, 1:])


def test_a_short_packed_row_shields_its_sequences():
    """As above at a length where one block walks the whole row, the cut inside a warp's tokens
    and at a warp's first."""
    cu = [0, 21, 48, 150]
    v = make(1, 160, 48, "bf16", cu=cu, seed=30)
    clean, cgrads = train(v)
    v["x"][0, 20], v["x"][0, 47] = float("inf"), float("-inf")
    for k in ("x", "forget", "gate", "dy"):
        v[k][:, 150:] = float("nan")
    got, grads = train(v)
    assert torch.equal(got[0][:, 48:], clean[0][:, 48:]) and torch.equal(got[1][2], clean[1][2])
    assert torch.isinf(got[1][:2]).all() and torch.equal(got[0][:, 21:47], clean[0][:, 21:47])
    for k in ("x", "forget", "gate"):
        assert torch.equal(grads[k][:, 48:], cgrads[k][:, 48:]), k
    assert torch.equal(grads["state"][2], cgrads["state"][2])


def test_gradients_are_not_differentiable_themselves():
    v = make(1, 20, 8, "fp32", seed=31)
    x, w = v["x"].clone().requires_grad_(True), torch.ones(8, device=DEV, requires_grad=True)
    y, _ = gated_scan(x * w, v["forget"])
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)   # allowed: a graph around the operator
    check_x, = torch.autograd.grad(gated_scan(x * w, v["forget"])[0].sum(), x)
    assert torch.equal(gx, check_x)
    with pytest.raises(RuntimeError, match="not differentiable themselves"):
        gx.sum().backward()


def test_a_channel_of_nan_stays_alone():
    v = make(2, 200, 6, "bf16", seed=10)
    clean, cg = train(v)
    v["x"][0, 50, 2] = v["forget"][1, 60, 3] = v["gate"][0, 70, 4] = float("nan")
    got, g = train(v)
    bad = torch.isnan(got[0])
    assert bad[0, 50:, 2].all() and bad[1, 60:, 3].all() and bad[0, 70, 4]
    assert int(bad.sum()) == 150 + 140 + 1
    for t, c in ((got[0], clean[0]), (g["x"], cg["x"]), (g["gate"], cg["gate"])):
        assert torch.equal(t[:, :, [0, 1, 5]], c[:, :, [0, 1, 5]])


def test_extreme_gates():
    """sigmoid at both ends and infinite gate inputs: the state is kept or replaced."""
    T, D = 40, 8
    v = make(1, T, D, "fp32", gate=True, lower=False, seed=11)
    v["forget"][:] = torch.tensor([-200.0, 200.0, -90.0, 90.0, float("inf"), float("-inf"), 0.0, -30.0], device=DEV)
    v["gate"][:, :, ::2] = 1000.0
    v["gate"][:, :, 1] = -1000.0
    (y, last), grads = train(v)
    x, h0 = v["x"], v["state"]
    for c in (0, 2, 5):
        assert torch.equal(last[0, c], x[0, -1, c])   # retention 0
    for c in (1, 3, 4):
        torch.testing.assert_close(last[0, c], h0[0, c], rtol=1e-6, atol=0)
    assert (y[:, :, 1].abs() < 1e-37).all() and torch.isfinite(y).all()
    assert all(torch.isfinite(t).all() for t in grads.values())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 33])
def test_strided_inputs(D, dtype):
    """Column ranges of one projection, a time-major layout, rows shared by a batch, a
    transposed tensor, and a strided output gradient."""
    B, T = 3, 150
    v = make(B, T, D, dtype, seed=12)
    want = infer(v)
    proj = torch.cat([v["x"], v["forget"], v["gate"]], -1)
    px, pf, pg = proj.split(D, -1)
    y, last = gated_scan(px, pf, pg, v["lower"], v["state"])
    assert torch.equal(y, want[0]) and torch.equal(last, want[1])
    tm = v["x"].transpose(0, 1).contiguous().transpose(0, 1)
    cf = v["forget"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(gated_scan(tm, cf, v["gate"], v["lower"], v["state"])[0], want[0])
    shared = v["forget"][:1].expand(B, T, D)
    v2 = {**v, "forget": shared}
    leaves = [v[k].detach().clone().requires_grad_(True) for k in ("x", "gate", "lower", "state")]
    f1 = v["forget"][:1].detach().clone().requires_grad_(True)
    y, last = gated_scan(leaves[0], f1.expand(B, T, D), *leaves[1:])
    wide = torch.zeros(B, T, 2 * D + 1, device=DEV, dtype=y.dtype)
    wide[:, :, 1:D + 1] = v["dy"]
    g = torch.autograd.grad((y, last), leaves + [f1], (wide[:, :, 1:D + 1], v["dlast"]))
    full, fg = train(v2)
    check(v2, full, fg)
    # another layout may take another kernel, whose sums associate differently
    check(v2, (y, last), {**dict(zip(("x", "gate", "lower", "state"), g)), "forget": fg["forget"]})
    # the gradient of the shared rows is the sum over the batch, made by autograd in f1's type
    torch.testing.assert_close(g[4], fg["forget"].float().sum(0, keepdim=True).to(g[4].dtype), rtol=2e-2, atol=1e-3)


def test_misaligned_rows():
    """Element-aligned views that no pair access may touch."""
    B, T, D = 2, 90, 64
    v = make(B, T, D, "bf16", seed=13)
    want = infer(v)
    off = {k: torch.empty(B * T * D + 1, device=DEV, dtype=torch.bfloat16)[1:].view(B, T, D).copy_(v[k])
           for k in ("x", "forget", "gate")}
    flat = torch.empty(D + 1, device=DEV)[1:].copy_(v["lower"])
    st = torch.empty(B * D + 1, device=DEV)[1:].view(B, D).copy_(v["state"])
    for w in ({**v, "x": off["x"]}, {**v, **off}, {**v, "lower": flat}, {**v, "state": st}):
        got, grads = train(w)
        check(v, got, grads)
        torch.testing.assert_close(got[1], want[1], rtol=1e-5, atol=1e-5)


def test_only_one_output_is_differentiated():
    v = make(2, 77, 34, "fp32", seed=14)
    zero = {**v, "dlast": torch.zeros_like(v["dlast"])}
    x = v["x"].clone().requires_grad_(True)
    y, last = gated_scan(x, v["forget"], v["gate"], v["lower"], v["state"])
    (gy,) = torch.autograd.grad(y, x, v["dy"], retain_graph=True)
    check(zero, (y, last), {**train(zero)[1], "x": gy})
    (gl,) = torch.autograd.grad(last, x, v["dlast"], retain_graph=True)
    z2 = {**v, "dy": torch.zeros_like(v["dy"])}
    check(z2, (y, last), {**train(z2)[1], "x": gl})
    (gs,) = torch.autograd.grad(y.sum(), x)  # an expanded gradient
    z3 = {**zero, "dy": torch.ones_like(v["dy"])}
    check(z3, (y, last), {**train(z3)[1], "x": gs})


def test_gradient_against_differences():
    """The directional derivative of an fp32 loss: a central difference of step e of a
    smooth function is off by O(e^2) and by rounding of about K X sqrt(terms) / e."""
    v = make(2, 60, 20, "fp32", seed=15)
    y_w = v["dy"].double()

    def loss(w):
        y, last = infer(w)
        return float((y.double() * y_w).sum() + (last.double() * v["dlast"].double()).sum())

    grads = train(v)[1]
    for k in NAMES:
        d = torch.randn(v[k].shape, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
        if k == "lower":
            d = d * 0.01
        e = 1e-2
        diff = (loss({**v, k: v[k] + e * d}) - loss({**v, k: v[k] - e * d})) / (2 * e)
        want = float((grads[k].double() * d.double()).sum())
        assert abs(diff - want) <= 2e-3 * (abs(want) + float((grads[k].double() * d.double()).abs().sum()) * 0.05), k


def test_two_calls_continue_one_sequence():
    v = make(2, 700, 50, "fp32", seed=16)
    y, last = infer(v)
    cut = 333
    parts = [{**v, **{k: v[k][:, a:b] for k in ("x", "forget", "gate")}} for a, b in ((0, cut), (cut, 700))]
    y1, s1 = infer(parts[0])
    y2, s2 = infer({**parts[1], "state": s1})
    torch.testing.assert_close(torch.cat([y1, y2], 1), y, rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(s2, last, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,D", [(1, 1), (1, 640), (256, 640), (7, 33), (1000, 17)])
def test_step(B, D, dtype):
    v = make(B, 1, D, dtype, seed=B + D)
    pool = torch.full((B + 4, D), 7.0, device=DEV)
    pool[2:B + 2] = v["state"]
    view = pool[2:B + 2]
    y = gated_scan_step(v["x"][:, 0], v["forget"][:, 0], view, v["gate"][:, 0], v["lower"])
    check(v, (y[:, None], view))
    assert (pool[:2] == 7).all() and (pool[B + 2:] == 7).all()
    st = v["state"].clone()
    y = gated_scan_step(v["x"][:, 0], v["forget"][:, 0], st)
    check({**v, "gate": None, "lower": None}, (y[:, None], st))


def test_steps_follow_a_prefill():
    """Prefill, then single tokens, as the whole sequence in one call."""
    v = make(3, 100, 96, "bf16", seed=17)
    y, last = infer(v)
    head = {**v, **{k: v[k][:, :60] for k in ("x", "forget", "gate")}}
    y1, st = infer(head)
    ys = [y1] + [gated_scan_step(v["x"][:, t], v["forget"][:, t], st, v["gate"][:, t], v["lower"])[:, None]
                 for t in range(60, 100)]
    check(v, (torch.cat(ys, 1), st))
    torch.testing.assert_close(st, last, rtol=1e-4, atol=1e-5)


def test_step_strides_and_refusals():
    v = make(4, 1, 30, "fp16", seed=18)
    proj = torch.cat([v["x"], v["forget"], v["gate"]], -1)[:, 0]
    wide = torch.zeros(4, 47, device=DEV)
    wide[:, 3:33] = v["state"]
    y = gated_scan_step(proj[:, :30], proj[:, 30:60], wide[:, 3:33], proj[:, 60:], v["lower"])
    check(v, (y[:, None], wide[:, 3:33]))
    assert not wide[:, :3].any() and not wide[:, 33:].any()
    x = v["x"][:, 0]
    with pytest.raises(ValueError, match="overlap"):
        gated_scan_step(x, x, v["state"][:1].expand(4, 30))
    with pytest.raises(ValueError, match="overlap"):
        gated_scan_step(x, x, v["state"].t().contiguous().t())
    with pytest.raises(TypeError, match="float32"):
        gated_scan_step(x, x, x.clone())
    with pytest.raises(ValueError, match="state"):
        gated_scan_step(x, x, v["state"][:3])
    with pytest.raises(NotImplementedError):
        gated_scan_step(x.clone().requires_grad_(True), x, v["state"])
    st = v["state"].clone()
    leaf = v["x"].clone().requires_grad_(True)
    y, _ = gated_scan(leaf, v["forget"], state=st)
    gated_scan_step(x, x, st)  # changes a tensor that the graph above has saved
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals():
    v = make(2, 5, 8, "bf16", seed=19)
    x, f = v["x"], v["forget"]
    cu = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    bad = [
        (ValueError, "forget", (x, f[:, :4])), (ValueError, "forget", (x, f.float())), (ValueError, "gate", (x, f, f[:1])),
        (TypeError, "float32, bfloat16", (x.double(), f.double())), (TypeError, "lower", (x, f, None, v["lower"].half())),
        (ValueError, "lower", (x, f, None, v["lower"][:4])), (ValueError, "lower", (x, f, None, v["lower"].cpu())),
        (TypeError, "state", (x, f, None, None, v["state"].half())), (ValueError, "state", (x, f, None, None, v["state"][:1])),
        (ValueError, "packed", (x, f, None, None, None, cu)), (ValueError, "cu_seqlens", (x[:1], f[:1], None, None, None, cu.long())),
        (ValueError, "cu_seqlens", (x[:1], f[:1], None, None, None, cu.cpu())),
        (ValueError, "state", (x[:1], f[:1], None, None, v["state"], cu)), (ValueError, "D must", (x[:, :, :0], f[:, :, :0])),
        (ValueError, "CUDA", (x.cpu(), f.cpu())), (ValueError, "forget", (x, f.cpu())),
    ]
    for err, word, args in bad:
        with pytest.raises(err, match=word):
            gated_scan(*args)


def test_no_tokens_and_no_sequences():
    for B, T in ((2, 0), (0, 5), (0, 0)):
        v = make(B, T, 12, "fp32", seed=20)
        (y, last), g = train(v)
        assert y.shape == (B, T, 12) and torch.equal(last, v["state"])
        assert torch.equal(g["state"], v["dlast"]) and not g["lower"].any() and g["x"].shape == (B, T, 12)


def test_wrong_cu_seqlens_stay_in_bounds():
    """Boundaries that decrease or pass the last row give some values and touch nothing else."""
    for cu in ([5, 3, 90, 2], [0, 500, 1000, 70], [-7, 20, 30, 64], [64, 64, 64, 64], [2**31 - 1, -2**31, 0, 64]):
        v = make(1, 64, 40, "bf16", cu=[0, 1, 2, 3], seed=21)
        v["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
        (y, last), g = train(v)
        assert y.shape == (1, 64, 40) and last.shape == (3, 40)
    torch.cuda.synchronize()


def test_same_bits_again_on_another_stream():
    v = make(2, 1500, 130, "bf16", seed=22)
    torch.cuda.synchronize()
    a = train(v)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = train(v)
    s.synchronize()
    for p, q in zip((*a[0], *a[1].values()), (*b[0], *b[1].values())):
        assert torch.equal(p, q)


def test_two_streams_at_once():
    vs = [make(1, 3000, 260, "fp32", seed=s) for s in (23, 24)]
    want = [train(v) for v in vs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in vs], []
    for _ in range(5):
        got = []
        for v, s in zip(vs, streams):
            with torch.cuda.stream(s):
                got.append(train(v))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            for k in NAMES:
                assert torch.equal(w[1][k], g[1][k])


def test_captured_training_step_and_decode():
    v = make(1, 400, 64, "bf16", cu=[0, 150, 390], seed=25)
    new = make(1, 400, 64, "bf16", cu=[0, 150, 390], seed=26)
    want = train({**new, "cu": torch.tensor([0, 10, 400], dtype=torch.int32, device=DEV)})
    leaves = {k: v[k].detach().clone().requires_grad_(True) for k in NAMES}
    dy, dl = v["dy"].clone(), v["dlast"].clone()

    def step():
        y, last = gated_scan(*(leaves[k] for k in NAMES), v["cu"])
        return (y, last), torch.autograd.grad((y, last), list(leaves.values()), (dy, dl))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, grads = step()
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        out2, grads2 = step()
    with torch.no_grad():
        for k in NAMES:
            leaves[k].copy_(new[k])
    dy.copy_(new["dy"])
    dl.copy_(new["dlast"])
    v["cu"].copy_(torch.tensor([0, 10, 400], dtype=torch.int32))
    g.replay()
    g2.replay()
    torch.cuda.synchronize()
    for o, gr in ((out, grads), (out2, grads2)):
        assert torch.equal(o[0], want[0][0]) and torch.equal(o[1], want[0][1])
        for k, t in zip(NAMES, gr):
            assert torch.equal(t, want[1][k]), k


def test_offsets_beyond_32_bits():
    """Inputs whose token stride alone passes 2^31 elements, and an output of more."""
    big = torch.empty(2**31 + 64, dtype=torch.bfloat16, device=DEV)
    v = make(1, 2, 64, "bf16", seed=27)
    big[:64], big[2**31:] = v["x"][0, 0], v["x"][0, 1]
    far = big.as_strided((1, 2, 64), (0, 2**31, 1))
    got, _ = train({**v, "x": v["x"]})
    y, last = gated_scan(far, v["forget"], v["gate"], v["lower"], v["state"])
    assert torch.equal(y, got[0]) and torch.equal(last, got[1])
    del big, far
    D, T = 64, 2**25 + 33                     # B T D = 2^31 + 2112
    one = make(1, 1, D, "bf16", gate=False, lower=False, state=False, seed=28)
    x, f = one["x"].expand(1, T, D), torch.full_like(one["x"], -3.0).expand(1, T, D)
    y, last = gated_scan(x, f)                # forgets fast: the state settles at x
    torch.testing.assert_close(y[0, -200:].float(), one["x"][0].float().expand(200, D), rtol=1e-2, atol=1e-3)
    torch.testing.assert_close(last, one["x"][0].float(), rtol=1e-5, atol=1e-6)
