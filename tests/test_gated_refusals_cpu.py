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


def test_sizes_beyond_the_limits_are_value_errors():
    """Refused before an output is allocated (the tensors here are one element, shared)."""
    one = torch.zeros(1, 1, 1)
    for shape in ((1, 2**30 + 1, 1), (2**26 + 1, 1, 1), (1, 1, 2**31), (2**20, 1, 32 * 64 + 1)):
        with pytest.raises(ValueError, match="too large"):
            gated_scan(one.expand(shape), one.expand(shape))
    big = one[0].expand(2**20, 2**18 + 1)
    with pytest.raises(ValueError, match="too large"):
        gated_scan_step(big, big, big)
    with pytest.raises(ValueError, match="too large"):
        dropout(one.expand(2**20, 2**10, 2**10 + 1), 0.5, 1)
    for shape in ((1, 2**30, 1), (2**26, 1, 1), (2**20, 1, 32 * 64)):  # at the limits
        with pytest.raises(ValueError, match="CUDA"):
            gated_scan(one.expand(shape), one.expand(shape))
