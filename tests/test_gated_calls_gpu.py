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
