"""Corners of the beam-search operators on the GPU."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_z_beams_gpu import check_reorder, filled, parents_of

pytestmark = pytest.mark.gpu


def test_reorder_tensors_without_elements():
    """A cache before its first position is written, alone and among others."""
    import torch

    beams = parents_of(2, 4, 5)
    empty = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    check_reorder([empty(8, 0, 16)], beams)
    check_reorder([empty(8, 2, 0, 16)], beams, lengths=[0, 3], dim=2)
    check_reorder([empty(8, 0, 16), filled((8, 5, 16), torch.bfloat16), empty(8, 0, 16)], beams, lengths=[2, 5], dim=1)
    check_reorder([filled((8, 5, 16), torch.int32), empty(8, 0, 16)], beams)
    check_reorder([empty(0, 16)], beams, rows=np.arange(8).reshape(2, 4))


def test_candidates_past_32_bits_are_refused():
    import torch

    from xgraph_b200.beams import beam_select

    logits, scores = torch.zeros((4, 100), device="cuda"), torch.zeros((1, 4), device="cuda")
    with pytest.raises(ValueError, match="candidates must be between 1 and 128"):
        beam_select(logits, scores, candidates=(1 << 32) + 2)
