"""GPU parity of dropout (yufmusicgen_b200/dropout.py) with its definition in
float64 (oracle/gated.py).  A kept element is one fp32 FMA of exact inputs and the
rounded 1 / (1 - p): 2 u relative to x / (1 - p) and u to the sum (u = 2^-24), then
half a step of the output's type.  Which elements are kept is exact."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from oracle import gated  # noqa: E402
from yufmusicgen_b200.dropout import dropout  # noqa: E402
from yufmusicgen_b200.gated_scan import gated_scan  # noqa: E402

DEV = "cuda:0"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0**-24


def rnd(shape, dtype, seed):
    a = np.random.default_rng(seed).standard_normal(shape).astype(np.float32)
    return torch.from_numpy(a).to(DEV).to(dtype)


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def near(got, want, terms):
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    bound = 3 * U * terms * (1 + half) + half * np.abs(want) + (2.0**-25 if got.dtype == torch.float16 else 0.0)
    g = f64(got)
    assert g.shape == want.shape and (np.abs(g - want) <= bound).all()


def check(x, p, seed, step, r, dy):
    xl = x.detach().requires_grad_(True)
    rl = None if r is None else r.detach().requires_grad_(True)
    y = dropout(xl, p, seed, step, rl)
    assert y.dtype == (x.dtype if r is None else r.dtype) and y.is_contiguous()
    plain = gated.dropout(f64(x), p, seed, step)
    terms = np.abs(plain) + (0 if r is None else np.abs(f64(r)))
    near(y, plain + (0 if r is None else f64(r)), terms)
    g = torch.autograd.grad(y, [xl] if r is None else [xl, rl], dy)
    want = gated.dropout(f64(dy), p, seed, step)
    assert g[0].dtype == x.dtype
    near(g[0], want, np.abs(want))
    if r is not None:
        assert torch.equal(g[1], dy)
    with torch.no_grad():
        assert torch.equal(dropout(x, p, seed, step, r), y)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("res", ["none", "same", "fp32"])
@pytest.mark.parametrize("shape", [(1,), (3,), (8,), (5, 7), (2, 9, 64), (1000, 33), (2049,), (2, 3, 5, 24)])
def test_against_the_definition(shape, res, dtype):
    n = int(np.prod(shape))
    x = rnd(shape, DT[dtype], n)
    r = None if res == "none" else rnd(shape, DT[dtype] if res == "same" else torch.float32, n + 1)
    check(x, 0.3, 0x123456789ABCDEF0, 2**40 + n, r, rnd(shape, x.dtype if r is None else r.dtype, n + 2))


@pytest.mark.parametrize("p", [0.0, 1.0, 0.5, 2.0**-32, 1 - 2.0**-32, 1e-12])
def test_probabilities(p):
    x, r = rnd((40, 50), torch.float32, 1), rnd((40, 50), torch.float32, 2)
    y = dropout(x, p, 5, 6)
    if p == 1.0:
        assert not y.any() and torch.equal(dropout(x, p, 5, 6, r), r)
    else:
        check(x, p, 5, 6, r, rnd((40, 50), torch.float32, 3))
    if p == 0.0:
        assert torch.equal(y, x)


def test_share_of_dropped_elements():
    """n Bernoulli draws: the share lies within 6 standard deviations of p."""
    n, p = 1 << 20, 0.2
    y = dropout(torch.ones(n, device=DEV), p, 11, 0)
    assert abs(float((y == 0).float().mean()) - p) < 6 * (p * (1 - p) / n) ** 0.5
    z = dropout(torch.ones(n, device=DEV), p, 11, 1)  # another step: an independent mask
    both = float(((y == 0) & (z == 0)).float().mean())
    assert abs(both - p * p) < 6 * (p * p * (1 - p * p) / n) ** 0.5


def test_dropped_infinities_and_nan_do_not_get_through():
    x = torch.full((64, 64), float("inf"), device=DEV)
    x[::2] = float("nan")
    r = rnd((64, 64), torch.float32, 4)
    keep = torch.from_numpy(gated.philox_words(0, 4096, 7, 8) >= int(0.5 * 2**32)).reshape(64, 64).to(DEV)
    y = dropout(x, 0.5, 7, 8, r)
    assert torch.equal(y[~keep], r[~keep])
    assert not torch.isfinite(y[keep]).any()
    assert torch.equal(dropout(x, 1.0, 7, 8, r), r)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("cols", [64, 40, 13])
def test_strided_tensors(cols, dtype):
    """Column ranges, a slice of the middle axis, shared rows, a transposed tensor: the mask goes by
    the logical index."""
    B, T, dt = 3, 10, DT[dtype]
    base, rbase = rnd((B, T, 2 * cols + 8), dt, 1), rnd((B, T + 3, cols), dt, 2)
    x, r = base[:, :, 8:8 + cols], rbase[:, 1:T + 1]
    dy = rnd((B, T, 3 * cols), dt, 3)[:, :, :cols]
    check(x, 0.4, 9, 10, r, dy)
    check(x, 0.4, 9, 10, None, dy)
    check(base[:, :, 1:1 + cols], 0.4, 9, 10, rbase[:1, :1].expand(B, T, cols), dy)
    check(x.transpose(0, 2), 0.4, 9, 10, None, dy.transpose(0, 2))
    odd = torch.empty(B * T * cols + 1, device=DEV, dtype=dt)[1:].view(B, T, cols).copy_(x)
    check(odd, 0.4, 9, 10, odd, dy)


def test_step_on_the_device():
    x = rnd((20, 24), torch.bfloat16, 5).requires_grad_(True)
    step = torch.tensor([2**33 + 5], device=DEV)
    y = dropout(x, 0.3, -1, step)
    assert torch.equal(y, dropout(x, 0.3, 2**64 - 1, 2**33 + 5))
    step += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    z = dropout(x, 0.3, -1, step)
    assert not torch.equal(y, z) and torch.equal(z, dropout(x, 0.3, -1, 2**33 + 6))


def test_captured_graph_draws_new_masks():
    x, r = rnd((300, 40), torch.bfloat16, 6).requires_grad_(True), rnd((300, 40), torch.float32, 7)
    dy = rnd((300, 40), torch.float32, 8)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)

    def run():
        y = dropout(x, 0.25, 77, step, r)
        return y, torch.autograd.grad(y, x, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, dx = run()
        step += 1
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert int(step) == k + 1
        want = dropout(x, 0.25, 77, k, r)
        assert torch.equal(y, want) and torch.equal(dx, torch.autograd.grad(want, x, dy)[0])


def test_gradients_are_not_differentiable_themselves():
    x = rnd((8, 8), torch.float32, 9).requires_grad_(True)
    (gx,) = torch.autograd.grad((dropout(x, 0.5, 1) ** 2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable themselves"):
        gx.sum().backward()


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    for err, word, kw in [
        (ValueError, "CUDA", dict(x=x.cpu())), (TypeError, "float32, bfloat16", dict(x=x.double())),
        (ValueError, "0, 1", dict(p=1.5)), (ValueError, "0, 1", dict(p=-0.1)), (ValueError, "0, 1", dict(p=float("nan"))),
        (ValueError, "residual", dict(residual=x[:2])), (ValueError, "residual", dict(residual=x.cpu())),
        (TypeError, "residual", dict(residual=x.half())), (TypeError, "residual", dict(x=x.half(), residual=x.bfloat16())),
        (ValueError, "step", dict(step=torch.zeros(1, device=DEV))), (ValueError, "step", dict(step=torch.zeros(1, dtype=torch.int64))),
        (ValueError, "step", dict(step=torch.zeros(2, dtype=torch.int64, device=DEV))),
    ]:
        with pytest.raises(err, match=word):
            dropout(**{"x": x, "p": 0.5, "seed": 1, **kw})
    assert dropout(x[:0], 0.5, 1).shape == (0, 8) and dropout(x[:, :0], 0.5, 1).shape == (4, 0)
    scalar = torch.tensor(2.0, device=DEV)
    assert dropout(scalar, 0.0, 1).shape == ()


def test_beyond_32_bit_indexes():
    n = 2**31 + 4099
    x = torch.ones(1, dtype=torch.bfloat16, device=DEV).expand(n // 11, 11)  # shared rows: nothing is read twice
    y = dropout(x, 0.5, 3, 4)
    tail = (y.reshape(-1)[-4096:] != 0).cpu().numpy()
    total = y.numel()
    assert (tail == (gated.philox_words(total - 4096, 4096, 3, 4) >= 2**31)).all()


def test_a_block_trained_with_both():
    """Projection -> gated scan over packed sequences -> output projection -> dropout onto an fp32
    residual stream, forward and backward, against the same block in float64."""
    D, T, cu = 48, 200, [0, 60, 60, 190]
    gen = torch.Generator(DEV).manual_seed(0)
    u = torch.randn(1, T, D, device=DEV, generator=gen)
    w_in = (torch.randn(3 * D, D, device=DEV, generator=gen) * D**-0.5).requires_grad_(True)
    w_out = (torch.randn(D, D, device=DEV, generator=gen) * D**-0.5).requires_grad_(True)
    low = (torch.rand(D, device=DEV, generator=gen) * 0.9).requires_grad_(True)
    s0 = torch.randn(3, D, device=DEV, generator=gen).requires_grad_(True)
    dy, dl = (torch.randn(*s, device=DEV, generator=gen) for s in ((1, T, D), (3, D)))
    cut = torch.tensor(cu, dtype=torch.int32, device=DEV)
    leaves = [w_in, w_out, low, s0]
    p, seed, step = 0.2, 5, 6

    x, f, g = (u @ w_in.t()).split(D, -1)
    y, last = gated_scan(x, f, g, low, s0, cut)
    out = dropout(y @ w_out.t(), p, seed, step, residual=u)
    got = torch.autograd.grad((out, last), leaves, (dy, dl))

    dbl = [t.detach().double().requires_grad_(True) for t in leaves]
    x, f, g = (u.double() @ dbl[0].t()).split(D, -1)
    a = dbl[2] + (1 - dbl[2]) * torch.sigmoid(f)
    rows, ends = [None] * T, []
    for s in range(3):
        h = dbl[3][s]
        for t in range(cu[s], cu[s + 1]):
            h = a[0, t] * h + (1 - a[0, t]) * x[0, t]
            rows[t] = h * torch.sigmoid(g[0, t])
        ends.append(h)
    zero = torch.zeros(D, device=DEV, dtype=torch.float64)
    yd = torch.stack([zero if r is None else r for r in rows])[None]
    keep = torch.from_numpy(gated.philox_words(0, T * D, seed, step) >= int(p * 2**32)).reshape(1, T, D).to(DEV)
    outd = u.double() + torch.where(keep, (yd @ dbl[1].t()) / (1 - p), 0.0)
    want = torch.autograd.grad((outd, torch.stack(ends)), dbl, (dy.double(), dl.double()))
    # fp32 products of D = 48 terms and sums over T = 200 rows: (D + T) u of the magnitudes, with
    # the recurrence's own error (tests/test_gated_scan_gpu.py): within 5e-4 of the largest entry
    torch.testing.assert_close(out.double(), outd, rtol=0, atol=5e-4 * float(outd.abs().max()))
    for a_, b_ in zip(got, want):
        torch.testing.assert_close(a_.double(), b_, rtol=0, atol=5e-4 * float(b_.abs().max()))
