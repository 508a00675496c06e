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


@pytest.mark.parametrize("sizes,message", [
    (dict(beams=0), "1 to 64 beams, got 0"), (dict(beams=65), "1 to 64 beams"), (dict(beams=(1 << 32) + 4), "1 to 64 beams"),
    (dict(candidates=0), "candidates"), (dict(candidates=129), "candidates"), (dict(candidates=(1 << 32) + 8), "candidates"),
    (dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 20) + 1), "vocabulary"), (dict(vocab=(1 << 32) + 100), "vocabulary"),
    (dict(groups=(1 << 32) + 1), "too many groups"), (dict(steps=(1 << 32) + 1), "too many steps"),
])
def test_sizes_past_32_bits_are_refused_not_cut(sizes, message):
    from xgraph_b200.beams import _check_sizes

    _check_sizes(**{"groups": 0, "beams": 64, "vocab": 1 << 20, "candidates": 128, "steps": 1 << 30})
    with pytest.raises(ValueError, match=message):
        _check_sizes(**{"groups": 2, "beams": 4, **sizes})


def test_the_limits_are_the_headers():
    import re
    from pathlib import Path

    from xgraph_b200 import beams

    text = (Path(__file__).parents[1] / "include" / "xgraph_b200.h").read_text()
    for name in ("MAX_BEAMS", "MAX_CANDIDATES", "MAX_BEAM_VOCAB"):
        value = re.search(rf"#define XG_{name} (.*)", text).group(1)
        assert eval(value) == getattr(beams, name)  # noqa: S307 (a number or a shift of two)
