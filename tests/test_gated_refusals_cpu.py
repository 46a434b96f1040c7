"""Calls of the gated recurrence and of dropout that are refused on the host, before any
CUDA call, because their answer would be wrong."""

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fw  # noqa: E402

from yufmusicgen_b200.dropout import dropout  # noqa: E402
from yufmusicgen_b200.gated_scan import gated_scan, gated_scan_step  # noqa: E402


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_tangents_are_refused(requires_grad):
    """A tangent that no derivative carries on would be lost without a word."""
    plain = {"x": torch.ones(1, 3, 4), "forget": torch.ones(1, 3, 4), "gate": torch.ones(1, 3, 4),
             "lower": torch.zeros(4), "state": torch.zeros(1, 4)}
    token = {k: t[:, 0] if t.dim() == 3 else t for k, t in plain.items()}
    with fw.dual_level():
        for call, args in ((gated_scan, plain), (gated_scan_step, token),
                           (lambda x, residual: dropout(x, 0.5, 1, residual=residual),
                            {"x": torch.ones(3), "residual": torch.ones(3)})):
            for k, t in args.items():
                dual = fw.make_dual(t.clone().requires_grad_(requires_grad), torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="tangent"):
                    call(**{**args, k: dual})
                with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                    call(**{**args, k: dual})
