"""The gated recurrence against its definition in float64, element by element, within
the rounding errors that ``oracle/gated_bounds.py`` derives: a bound for each element
from its own factors, so that small elements count as much as large ones."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from oracle import gated_bounds as gb  # noqa: E402
from yufmusicgen_b200.gated_scan import gated_scan  # noqa: E402

DEV = "cuda:0"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NAMES = ("x", "forget", "gate", "lower", "state")


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def make(B, T, D, dtype, cu=None, seed=0, forget=(1.5, 2.0), gate=(1.0, 0.0), ends=None):
    """Inputs as a layer meets them; ``ends``: that input spread evenly over [-20, 20]."""
    rng = np.random.default_rng(seed)
    rows = B if cu is None else len(cu) - 1

    def t(*shape, scale=1.0, shift=0.0, dt=DT[dtype], even=False):
        a = rng.uniform(-20, 20, shape) if even else np.clip(rng.standard_normal(shape), -4, 4) * scale + shift
        return torch.from_numpy(a.astype(np.float32)).to(DEV).to(dt)

    return {"x": t(B, T, D), "forget": t(B, T, D, scale=forget[0], shift=forget[1], even=ends == "forget"),
            "gate": t(B, T, D, scale=gate[0], shift=gate[1], even=ends == "gate"),
            "lower": torch.from_numpy((rng.random(D) * 0.95).astype(np.float32)).to(DEV),
            "state": t(rows, D, dt=torch.float32),
            "cu": None if cu is None else torch.tensor(cu, dtype=torch.int32, device=DEV),
            "dy": t(B, T, D), "dlast": t(rows, D, dt=torch.float32)}


def train(v):
    leaves = {k: v[k].detach().clone().requires_grad_(True) for k in NAMES if v[k] is not None}
    y, last = gated_scan(*(leaves.get(k) for k in NAMES), v["cu"])
    g = torch.autograd.grad((y, last), list(leaves.values()), (v["dy"], v["dlast"]))
    return {"y": y, "last": last, **dict(zip(leaves, g))}


def check(v, names=("y", "last", *NAMES)):
    got = train(v)
    cu = None if v["cu"] is None else v["cu"].tolist()
    want, bound = gb.gated_scan_bounds(*(f64(v[k]) for k in NAMES), cu, f64(v["dy"]), f64(v["dlast"]))
    off = {}
    for k in names:
        if k not in got:
            continue
        half = torch.finfo(got[k].dtype).eps / 2 if got[k].dtype != torch.float32 else 0.0
        floor = 2.0**-25 if got[k].dtype == torch.float16 else 0.0
        off[k] = gb.beyond(f64(got[k]), want[k], bound[k], half, floor)
    assert all(o <= 0 for o in off.values()), off


# few columns (ranges), many (a block walks the time axis), rows of whole 16-byte pieces or not
FORMS = [(1, 60, 64), (2, 77, 33), (2, 2060, 72), (80, 130, 16), (80, 100, 17)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,T,D", FORMS)
def test_output_gate_at_both_ends(B, T, D, dtype):
    """The gradient of a saturated gate keeps its relative accuracy on both sides."""
    check(make(B, T, D, dtype, seed=T, ends="gate"), ("y", "gate"))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,T,D", FORMS)
def test_forget_gate_at_both_ends(B, T, D, dtype):
    """Every gradient where the state is all but kept or all but replaced: a retention near 0
    keeps its relative accuracy as much as an input share near 0."""
    check(make(B, T, D, dtype, seed=T, ends="forget"))


@pytest.mark.parametrize("copies", [False, True])
def test_dlower_sums_many_equal_terms(copies):
    """2.6 million terms of nearly the same size per channel: an fp32 sum of them drops the
    same bits of each one again and again.  The rows of the batch are alike, so the sum is
    B times that of one row (``copies``: rows of their own, or shared ones)."""
    B, T, D = 80, 32768, 32
    size = torch.arange(1, D + 1, device=DEV) / D + 0.37
    sign = 1 - 2.0 * (torch.arange(T, device=DEV) % 2)
    x = (sign[:, None] * size)[None]
    v = {"x": x, "forget": torch.linspace(-2, 2, D, device=DEV).expand(1, T, D), "gate": None,
         "lower": torch.zeros(D, device=DEV), "state": None, "dy": x, "dlast": torch.zeros(1, D, device=DEV)}
    want, bound = gb.gated_scan_bounds(*(f64(v[k]) for k in NAMES), None, f64(v["dy"]), f64(v["dlast"]))
    rows = {k: v[k].expand(B, T, D) for k in ("x", "forget", "dy")}
    if copies:
        rows = {k: t.contiguous() for k, t in rows.items()}
    lower = v["lower"].requires_grad_(True)
    y, _ = gated_scan(rows["x"], rows["forget"], None, lower)
    (g,) = torch.autograd.grad(y, lower, rows["dy"])
    assert gb.beyond(f64(g), B * want["lower"], B * bound["lower"]) <= 0


SHAPES = [(1, 1, 1), (2, 129, 40), (2, 1025, 66), (1, 2048, 640), (5, 64, 31), (300, 3, 10), (2, 2060, 72),
          (37, 300, 64), (80, 530, 16), (150, 290, 8), (80, 300, 17)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_every_element(B, T, D, dtype):
    """Both forms, one and several steps and ranges, many batch rows."""
    check(make(B, T, D, dtype, seed=B + T + D))


PACKED = [([0, 5000, 5001, 8990], 9000), ([0, 200, 200, 257, 260], 270), ([0, 1, 2, 3], 3), ([0, 127, 129, 129, 1000], 1100)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 37])
@pytest.mark.parametrize("cu,T", PACKED)
def test_every_element_of_packed_rows(cu, T, D, dtype):
    check(make(1, T, D, dtype, cu=cu, seed=T + D))


@pytest.mark.parametrize("D", [2600, 2601])
def test_every_element_of_wide_packed_rows(D):
    """So many columns that a block walks a packed row by itself; dlower's shares lie elsewhere."""
    v = make(1, 600, D, "bf16", cu=[0, 100, 100, 430, 590], seed=D)
    check(v)
    check({**v, "dy": v["dy"][:, :, 1:2].expand(1, 600, D).contiguous(), "lower": torch.zeros_like(v["lower"])})


def test_every_element_at_both_ends_of_all_gates():
    for cu in (None, [0, 40, 41, 333]):
        v = make(1, 350, 96, "fp32", cu=cu, seed=7, ends="forget")
        check({**v, "gate": make(1, 350, 96, "fp32", seed=8, ends="gate")["gate"]})
