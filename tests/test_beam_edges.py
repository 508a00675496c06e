"""Corners of the beam-search operators' host side, without a GPU."""

from __future__ import annotations

import pytest

from tests.test_beams import FAKE, GOOD, library, records, refused


@pytest.mark.parametrize("shape", [(0, 8), (3, 0), (0,), (2, 0, 4, 8)])
@pytest.mark.parametrize("lengths", [None, FAKE])
def test_tensors_without_elements_have_no_address(shape, lengths):
    lib = library()
    strides = (1,) * len(shape)
    empty = (8, 8, shape, strides, 4, 0, 0)
    assert lib.xg_beam_reorder(records(empty), 1, FAKE, 2, 4, lengths, None, None) == 0
    assert lib.xg_beam_reorder(records(empty, empty), 2, FAKE, 2, 4, lengths, None, None) == 0
    assert lib.xg_beam_reorder(records((0, 8, (8,), (1,), 4, 0, 0)), 1, FAKE, 2, 4, lengths, FAKE, None) == 0
    refused(lib.xg_beam_reorder(records((*GOOD[:5], 0, 0)), 1, FAKE, 2, 4, lengths, None, None), "null tensor")


def test_a_first_call_beside_another_finds_everything_loaded(monkeypatch):
    """The library is what a thread asks for to know that all is there, so it is set last."""
    from xgraph_b200 import beams

    seen = []

    class Types(dict):
        def update(self, *given):
            seen.append(beams._lib)
            super().update(*given)

    for name in ("_torch", "_lib", "_call_errors", "_get_device", "_get_stream"):
        monkeypatch.setattr(beams, name, None)
    monkeypatch.setattr(beams, "_dtypes", Types())
    beams._load()
    assert seen == [None] and beams._lib is not None
    assert beams._torch is not None and beams._get_device is not None and beams._get_stream is not None
