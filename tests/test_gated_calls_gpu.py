"""Calls of the gated recurrence and of dropout that torch allows and that have to be
answered rightly or refused."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

import torch.autograd.forward_ad as fw  # noqa: E402

from yufmusicgen_b200.dropout import dropout  # noqa: E402
from yufmusicgen_b200.gated_scan import gated_scan, gated_scan_step  # noqa: E402

DEV = "cuda:0"


def test_forward_mode_tangents_are_refused():
    """Of an input, and of a gradient that comes back (forward over reverse)."""
    x, f = torch.randn(1, 9, 8, device=DEV), torch.randn(1, 9, 8, device=DEV)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: gated_scan(dual, f), lambda: gated_scan(x, f, lower=fw.make_dual(x[0, 0], x[0, 1])),
                     lambda: gated_scan_step(dual[:, 0], f[:, 0], torch.zeros(1, 8, device=DEV)),
                     lambda: dropout(dual, 0.5, 1), lambda: dropout(x, 0.5, 1, residual=dual)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
        leaf = x.clone().requires_grad_(True)
        for y in (gated_scan(leaf, f)[0], gated_scan(leaf, f)[1], dropout(leaf, 0.5, 1)):
            loss = (y * fw.make_dual(torch.ones_like(y), torch.ones_like(y))).sum()
            with pytest.raises(NotImplementedError, match="tangent"):
                torch.autograd.grad(loss, leaf)
    assert torch.isfinite(gated_scan(x, f)[0]).all()


def lazily_negated(*shape):
    """A float32 tensor that torch negates only when it is read (the imaginary part of a
    conjugate), with a last axis of one element: no copy for the sake of its strides."""
    t = torch.randn(*shape, 1, dtype=torch.complex64, device=DEV).conj().imag
    assert t.is_neg() and t.dtype == torch.float32
    return t


def test_lazily_negated_tensors():
    x, f, g, h0, dy, dl = *(lazily_negated(2, 40) for _ in range(3)), lazily_negated(2), lazily_negated(2, 40), lazily_negated(2)
    low = torch.full((1,), -0.5j, device=DEV).conj().imag
    plain = [t.clone() for t in (x, f, g, low, h0)]
    assert float(low) == 0.5 and low.is_neg() and not any(t.is_neg() for t in plain)
    for a, b in zip(gated_scan(x, f, g, low, h0), gated_scan(*plain)):
        assert torch.equal(a, b)
    leaves = [t.requires_grad_(True) for t in plain]
    out = gated_scan(*leaves)
    for a, b in zip(torch.autograd.grad(out, leaves, (dy, dl), retain_graph=True),
                    torch.autograd.grad(out, leaves, (dy.clone(), dl.clone()))):
        assert torch.equal(a, b)
    s1, s2 = (torch.zeros(2, 1, device=DEV) for _ in range(2))
    y = gated_scan_step(x[:, 0], f[:, 0], s1, g[:, 0], low)
    assert torch.equal(y, gated_scan_step(*(t[:, 0].clone() for t in (x, f)), s2, g[:, 0].clone(), low.clone()))
    assert torch.equal(s1, s2)
    with pytest.raises(ValueError, match="negated"):
        gated_scan_step(x[:, 0], f[:, 0], h0)


def test_lazily_negated_tensors_in_dropout():
    x, r, dy = (lazily_negated(50) for _ in range(3))
    assert torch.equal(dropout(x, 0.25, 3, 4, r), dropout(x.clone(), 0.25, 3, 4, r.clone()))
    leaf = x.detach().clone().requires_grad_(True)
    (a,) = torch.autograd.grad(dropout(leaf, 0.25, 3), leaf, dy)
    (b,) = torch.autograd.grad(dropout(leaf, 0.25, 3), leaf, dy.clone())
    assert torch.equal(a, b)


def test_zeros_that_torch_does_not_store():
    """Whole and sliced, as inputs and as output gradients."""
    x, f = torch.randn(2, 9, 8, device=DEV), torch.randn(2, 9, 8, device=DEV)
    z = torch._efficientzerotensor((4, 9, 8), device=DEV)[2:]
    real = torch.zeros(2, 9, 8, device=DEV)
    assert z._is_zerotensor()
    for a, b in zip(gated_scan(x, z, z, z[0, 0], z[:, 0]), gated_scan(x, real, real, real[0, 0], real[:, 0])):
        assert torch.equal(a, b)
    assert torch.equal(dropout(z, 0.5, 1, residual=x), x) and torch.equal(dropout(x, 0.0, 1, residual=z), x)
    leaf = x.clone().requires_grad_(True)
    y, last = gated_scan(leaf, f)
    (g,) = torch.autograd.grad((y, last), leaf, (z, z[:, 0]))
    assert not g.any()
    (g,) = torch.autograd.grad(dropout(leaf, 0.5, 1), leaf, z)
    assert not g.any()


def test_fake_outputs_do_not_reach_a_kernel():
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, x1 = torch.randn(1, 9, 8, device=DEV), torch.randn(1, 8, device=DEV)
    state = torch.zeros(1, 8, device=DEV)
    with FakeTensorMode():
        for call in (lambda: gated_scan(x, x), lambda: gated_scan_step(x1, x1, state), lambda: dropout(x, 0.5, 1)):
            with pytest.raises((RuntimeError, TypeError), match="memory"):
                call()
    assert not state.any()


def test_a_step_may_take_its_state_as_input():
    """Each element with itself: x and forget are the state, in rows of their own."""
    pool = torch.randn(5, 40, device=DEV)
    want = pool[1:4].clone()
    y = gated_scan_step(want.clone(), want.clone(), want)
    state = pool[1:4]
    assert torch.equal(gated_scan_step(state, state, state), y) and torch.equal(state, want)
