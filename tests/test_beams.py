"""The beam-search operators without a GPU: argument checks, and the host reference that the
GPU tests compare with, on worked examples."""

from __future__ import annotations

import ctypes
import struct

import numpy as np
import pytest

from tests import beam_reference as ref

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: every call below fails its host checks


def library():
    from xgraph_b200.engine import load_library

    return load_library()


def refused(rc, message):
    from xgraph_b200.engine import _check

    with pytest.raises(ValueError, match=message):
        _check(rc)


def select(lib, dtype=1, groups=2, beams=4, vocab=100, row_stride=100, scores=FAKE, mask=None, mask_stride=0,
           finished=None, candidates=8, end_token=-1, logits=FAKE, workspace=FAKE, workspace_bytes=1 << 30):
    return lib.xg_beam_select(logits, dtype, groups, beams, vocab, row_stride, scores, mask, mask_stride, finished,
                              candidates, end_token, 1, FAKE, FAKE, FAKE, FAKE, workspace, workspace_bytes, None)


@pytest.mark.parametrize("change,message", [
    ({"dtype": 3}, "float32, bfloat16 or float16"), ({"beams": 0}, "1 to 64 beams"), ({"beams": 65}, "1 to 64 beams"),
    ({"groups": -1}, "beams"), ({"candidates": 0}, "candidates"), ({"candidates": 129}, "candidates"),
    ({"vocab": 0}, "vocabulary"), ({"vocab": (1 << 20) + 1}, "vocabulary"), ({"end_token": 100}, "end_token"),
    ({"end_token": -2}, "end_token"), ({"finished": FAKE}, "end_token"), ({"row_stride": 99}, "contiguous row"),
    ({"mask": FAKE, "mask_stride": 3}, "4 words"), ({"logits": None}, "null"), ({"scores": None}, "null"),
    ({"logits": ctypes.c_void_p((1 << 20) + 1)}, "aligned"), ({"groups": 1 << 30}, "too many"),
])
def test_select_refusals(change, message):
    refused(select(library(), **change), message)


def test_an_empty_batch_is_nothing_to_do():
    lib = library()
    assert select(lib, groups=0, logits=None) == 0
    assert lib.xg_beam_reorder(None, 0, None, 0, 4, None, None, None) == 0
    assert lib.xg_beam_sequences(None, 0, 0, None, 0, 0, 0, 3, 4, None, -1, None, None) == 0


def test_sequences_refusals():
    lib = library()
    refused(lib.xg_beam_sequences(FAKE, 8, 4, FAKE, 8, 4, 5, 2, 65, None, -1, FAKE, None), "1 to 64 beams")
    refused(lib.xg_beam_sequences(FAKE, 8, 4, FAKE, 8, 4, -1, 2, 4, None, -1, FAKE, None), "beams")
    refused(lib.xg_beam_sequences(None, 8, 4, FAKE, 8, 4, 5, 2, 4, None, -1, FAKE, None), "null")


def records(*tensors):
    """XgRowTensor records of (rows, row_stride, shape, strides, element_bytes, position[, address])."""
    out = b""
    for rows, row_stride, shape, strides, size, position, *address in tensors:
        pad = (0,) * (4 - len(shape))
        out += struct.pack("<qqq4q4q4i", address[0] if address else 1 << 20, rows, row_stride, *shape, *pad, *strides,
                           *pad, len(shape), size, position, 0)
    return out


GOOD = (8, 60, (3, 20), (20, 1), 4, -1)


@pytest.mark.parametrize("tensor,message,lengths", [
    ((7, 60, (3, 20), (20, 1), 4, -1), "one row per beam", None),
    ((8, 60, (3, 20), (20, 1), 3, -1), "bytes", None),
    ((8, 60, (3, 20), (20, 1), 4, -1, 0), "null", None),
    ((8, 60, (3, 20), (20, 1), 4, -1, (1 << 20) + 2), "aligned", None),
    ((8, 60, (3, 20), (20, 1), 4, 2), "position", None),
    ((8, 60, (3, 20), (20, 1), 4, -1), "position", FAKE),
    ((8, 59, (3, 20), (20, 1), 4, -1), "overlap", None),
    ((8, 0, (3, 20), (20, 1), 4, -1), "overlap", None),
    ((8, 60, (3, 20), (0, 1), 4, -1), "overlaps itself", None),
    ((8, 60, (3, 20), (19, 1), 4, -1), "overlaps itself", None),
    ((8, 60, (3, 20), (-20, 1), 4, -1), "negative stride", None),
    ((8, 60, (-3, 20), (20, 1), 4, -1), "negative size", None),
    ((8, 1000, (3, 3, 3, 3), (300, 90, 29, 9), 4, -1), "two places", None),
])
def test_reorder_refusals(tensor, message, lengths):
    lib = library()
    for count, given in ((1, records(tensor)), (2, records((*GOOD[:5], 0), tensor))):
        rc = lib.xg_beam_reorder(given, count, FAKE, 2, 4, lengths, None, None)
        if message == "one row per beam" and count == 2:
            refused(rc, "same number of rows")
        else:
            refused(rc, message)
    refused(lib.xg_beam_reorder(None, 1, FAKE, 2, 4, None, None, None), "null")
    refused(lib.xg_beam_reorder(records(GOOD), 1, None, 2, 4, None, None, None), "null")
    refused(lib.xg_beam_reorder(records(GOOD), 1, FAKE, 2, 65, None, None, None), "1 to 64 beams")
    refused(lib.xg_beam_reorder(records(GOOD), 1, FAKE, 70000, 4, None, None, None), "groups")


@pytest.mark.parametrize("tables", [(1 << 20, None, None), ((1 << 20) + 8 * 240 - 4, None, None),
                                    ((1 << 20) - 28, None, None), (1, 1 << 20, None), (1, None, (1 << 20) + 100)])
def test_reorder_refuses_tables_inside_a_tensor(tables):
    """The parents, lengths or rows would change while they are read."""
    parents, lengths, rows = (ctypes.c_void_p(t) if t else None for t in tables)
    given = records((*GOOD[:5], 0, 1 << 24), (*GOOD[:5], 0))
    refused(library().xg_beam_reorder(given, 2, parents, 2, 4, lengths, rows, None), "share memory")


def test_null_engine():
    lib = library()
    refused(lib.xg_reorder_slots(None, FAKE, FAKE, 1, 4, None), "null engine")
    refused(lib.xg_engine_beam_select(None, FAKE, 1, 1, 4, 10, 10, FAKE, FAKE, None, 4, -1, 1, FAKE, FAKE, FAKE, FAKE,
                                      FAKE, 1 << 20, None), "null engine")


def test_tensors_must_be_on_the_gpu():
    import torch

    from xgraph_b200 import beam_reorder, beam_select, beam_sequences

    logits, scores = torch.zeros((4, 10)), torch.zeros((1, 4))
    with pytest.raises(ValueError, match="GPU"):
        beam_select(logits, scores)
    with pytest.raises(ValueError, match="GPU"):
        beam_reorder([logits], torch.zeros((1, 4), dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        beam_sequences(torch.zeros((3, 1, 4), dtype=torch.int32), torch.zeros((3, 1, 4), dtype=torch.int32))


def test_shared_memory_is_found():
    from xgraph_b200.beams import _check_apart

    _check_apart([(1000, 100, True), (1100, 50, True), (900, 100, True), (5, 0, True)])
    _check_apart([(1000, 200, False), (1050, 200, False)])  # interleaved halves of one buffer
    for spans in ([(1000, 100, True), (1000, 100, True)], [(1000, 100, True), (1099, 50, True)],
                  [(1000, 100, False), (1000, 10, False)]):
        with pytest.raises(ValueError, match="share memory"):
            _check_apart(spans)


def test_layouts_of_tensors():
    """The records have the C structure's layout, and say what the tensors' shapes say."""
    import torch

    from xgraph_b200.beams import _layout, _load, _row_tensors

    _load()
    cpu = torch.device("cpu")
    a, b = torch.zeros((8, 2, 5), dtype=torch.bfloat16), torch.zeros((8, 4))
    half = torch.zeros((8, 3, 5), dtype=torch.bfloat16)[:, 1:]
    found, rows = _row_tensors([a, b, half], [2, 1, -1], cpu)
    assert rows == 8 and len(found) == 3 * 104
    assert found == records((8, 10, (2, 5), (5, 1), 2, 1, a.data_ptr()), (8, 4, (4,), (1,), 4, 0, b.data_ptr()),
                            (8, 15, (2, 5), (5, 1), 2, 1, half.data_ptr()))
    assert [_layout(t, None, cpu)[1:] for t in (a, b, half)] == [(160, True), (128, True), (230, False)]
    with pytest.raises(ValueError, match="share memory"):
        _row_tensors([a, b, a], None, cpu)
    for tensor, dim in ((torch.zeros(()), None), (torch.zeros((1,) * 6), None), (a, 0), (a, 3), (a, -3),
                        (torch.zeros((4, 4)).to_sparse(), None), (torch.zeros((4, 4), requires_grad=True), None)):
        with pytest.raises((ValueError, RuntimeError)):
            _layout(tensor, dim, cpu)


def test_the_record_is_the_headers_structure(tmp_path):
    import subprocess
    from pathlib import Path

    fields = ("data", "rows", "row_stride", "size", "stride", "dims", "element_bytes", "position_dim", "reserved")
    prints = "\n".join(f'printf("%zu ", offsetof(XgRowTensor, {f}));' for f in fields)
    source = tmp_path / "offsets.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "xgraph_b200.h"\nint main(void) {\n'
                      + prints + '\nprintf("%zu", sizeof(XgRowTensor));\nreturn 0;\n}\n')
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-std=c11", "-I", str(include), str(source), "-o", str(tmp_path / "offsets")], check=True)
    printed = subprocess.run([str(tmp_path / "offsets")], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in printed.split()] == [0, 8, 16, 24, 56, 88, 92, 96, 100, 104]


def test_reference_select_on_a_worked_example():
    """Two beams, four tokens: the constrained probabilities are simple fractions."""
    logits = np.log(np.array([[1.0, 1.0, 2.0, 4.0], [3.0, 1.0, 9.0, 3.0]]))
    scores = np.array([[0.0, np.log(0.5)]])
    mask = np.array([[0b0111], [0b1011]], dtype=np.int32)
    (value, beam, token, done), _ = ref.select(logits, scores, 5, mask=mask, end_token=2)
    # beam 0 over {0, 1, 2}: 1/4, 1/4, 1/2; beam 1 over {0, 1, 3}, halved: 3/14, 1/14, 3/14
    assert list(zip(beam[0], token[0], done[0])) == [(0, 2, True), (0, 0, False), (0, 1, False), (1, 0, False), (1, 3, False)]
    np.testing.assert_allclose(np.exp(value[0]), [1 / 2, 1 / 4, 1 / 4, 3 / 14, 3 / 14])
    (value, beam, token, done), _ = ref.select(logits, scores, 3, mask=mask, end_token=2, renormalize=False,
                                               finished=np.array([[False, True]]))
    assert list(zip(beam[0], token[0], done[0])) == [(1, 2, True), (0, 2, True), (0, 0, False)]
    np.testing.assert_allclose(np.exp(value[0]), [1 / 2, 1 / 4, 1 / 8])


def test_reference_sequences_and_reorder():
    tokens = np.array([[[10, 11]], [[20, 21]], [[30, 31]]])
    beams = np.array([[[0, 0]], [[1, 0]], [[1, -1]]])
    assert ref.sequences(tokens, beams).tolist() == [[[10, 21, 30], [-1, -1, 31]]]
    assert ref.sequences(tokens, beams, lengths=[2]).tolist() == [[[11, 20, -1], [10, 21, -1]]]
    moved = ref.reorder(np.arange(4)[:, None] * [1, 1], np.array([[1, 0], [-1, 0]]), lengths=[1, 2], dim=1)
    assert moved.tolist() == [[1, 0], [0, 1], [2, 2], [2, 2]]
