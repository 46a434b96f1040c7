"""The compiled torch module ``_yuf_torch`` (``csrc/torch/binding.cpp``), built
in-tree by ``yufmusicgen_b200.build`` beside the library it calls."""

from __future__ import annotations

import torch  # noqa: F401  (its libraries come first)

try:
    from . import _yuf_torch as ops
except ImportError as exc:
    raise ImportError(
        f"yufmusicgen_b200._yuf_torch cannot be loaded ({exc}): build it with "
        "`python -m yufmusicgen_b200.build` (this package has no CPU fallback)"
    ) from exc
