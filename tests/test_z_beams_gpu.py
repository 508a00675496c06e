"""The beam-search operators on the GPU against their definitions in 64 bits.

Order (beams, tokens, finished) must be equal.  A score is one float32 rounding of a 64-bit
value: half a step, 2^-24 of it, plus the scan's log-sum error, below 1e-6 absolutely (its
exponentials are within 2^-22 of theirs, its 32-bit additions, 16 in a row, within 2^-20, and
the exponents' rounding moves a sum by 2^-24 times the sum's mean exponent, at most 18).
"""

from __future__ import annotations

import numpy as np
import pytest

from tests import beam_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")
STEP = 2.0**-24
LOG_SUM = 2.0**-22 + 2.0**-20 + 18 * 2.0**-24


def make(dtype, rows, cols, seed, *, stride=None, offset=0, scale=2.0):
    """Logits [rows, cols] with any row stride and first-element offset (both in elements)."""
    import torch

    stride = cols if stride is None else stride
    gen = torch.Generator().manual_seed(seed)
    flat = (torch.randn(offset + rows * stride, generator=gen) * scale).to(getattr(torch, dtype)).cuda()
    return torch.as_strided(flat, (rows, cols), (stride, 1), offset)


def make_mask(rows, vocab, seed, kinds=(1.0, 0.5, 0.02, 0.0)):
    import torch

    rng = np.random.default_rng(seed)
    words = (vocab + 31) // 32
    bits = np.zeros((rows, words * 32), dtype=bool)
    share = rng.choice(kinds, size=rows)
    bits[:, :vocab] = rng.random((rows, vocab)) < share[:, None]
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).cuda()


def check(logits, scores, candidates, *, mask=None, finished=None, ties_exact=True, **options):
    from xgraph_b200.beams import beam_select

    got = beam_select(logits, scores, mask=mask, finished=finished, candidates=candidates, **options)
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    want, gaps = ref.select(logits.float().cpu().numpy(), host(scores), candidates, mask=host(mask),
                            finished=host(finished), **options)
    near = gaps[(gaps > 0) & (gaps < 1e-11)]
    assert not len(near), "the inputs leave the order to 64-bit rounding"
    np.testing.assert_array_equal(host(got.beams), want[1])
    np.testing.assert_array_equal(host(got.tokens), want[2])
    np.testing.assert_array_equal(host(got.finished), want[3])
    found = host(got.scores).astype(np.float64)
    empty = np.isneginf(want[0])
    np.testing.assert_array_equal(np.isneginf(found), empty)
    error = np.abs(found[~empty] - want[0][~empty])
    assert (error <= STEP * np.abs(want[0][~empty]) + LOG_SUM).all(), error.max()
    return got


def random_scores(groups, beams, seed):
    import torch

    gen = torch.Generator().manual_seed(seed)
    return (-10 * torch.rand((groups, beams), generator=gen)).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 31, 33, 255, 256, 1000, 4097, 8192, 16384, 16389, 40001])
def test_vocabulary_sizes(dtype, vocab):
    for groups, beams, candidates in ((1, 1, 1), (2, 3, 6), (3, 4, 8)):
        logits = make(dtype, groups * beams, vocab, vocab + beams)
        check(logits, random_scores(groups, beams, vocab), candidates)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("beams,candidates", [(1, 128), (2, 1), (5, 10), (16, 32), (17, 17), (32, 64), (64, 128), (64, 1)])
def test_beam_and_candidate_counts(dtype, beams, candidates):
    logits = make(dtype, 2 * beams, 5003, beams)
    check(logits, random_scores(2, beams, beams), candidates, mask=make_mask(2 * beams, 5003, beams))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extra,offset", [(0, 1), (1, 0), (3, 5), (8, 0), (13, 7)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_strides_and_alignment(dtype, extra, offset, renormalize):
    vocab = 2001
    logits = make(dtype, 12, vocab + 2, 9, stride=vocab + 2 + extra, offset=offset)
    check(logits, random_scores(3, 4, 1), 8, vocab=vocab, renormalize=renormalize)
    check(logits, random_scores(3, 4, 2), 8, vocab=vocab, renormalize=renormalize, mask=make_mask(12, vocab, 3))


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("kinds", [(1.0,), (0.5,), (0.01,), (0.0,), (0.0005, 0.0, 1.0)])
def test_masks(kinds, renormalize):
    logits = make("bfloat16", 32, 33000, 5)
    mask = make_mask(32, 33000, 6, kinds)
    got = check(logits, random_scores(4, 8, 3), 16, mask=mask, renormalize=renormalize)
    if kinds == (0.0,):
        assert (got.tokens == -1).all() and (got.scores == -float("inf")).all()


def test_a_wide_mask_with_spare_words():
    logits = make("float32", 4, 100, 5)
    wide = make_mask(4, 640, 6, (0.5,))
    check(logits, random_scores(1, 4, 3), 4, mask=wide[:, :7])


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_go_to_the_lowest_token(dtype):
    import torch

    logits = torch.full((8, 20011), 1.25, dtype=getattr(torch, dtype), device="cuda")
    scores = torch.tensor([[0.0, 0.0, -1.0, 0.0], [-3.0, -2.0, -2.0, -9.0]], device="cuda")
    check(logits, scores, 8)
    logits[:, ::3] = 2.5
    check(logits, scores, 128, mask=make_mask(8, 20011, 4, (0.5,)))
    check(torch.zeros_like(logits), scores, 128, renormalize=False, mask=make_mask(8, 20011, 4, (0.9,)))


@pytest.mark.parametrize("dtype,vocab", [("float32", 140001), ("bfloat16", 270000)])
def test_a_row_of_several_rounds(dtype, vocab):
    """64 beams of 128 candidates leave one CTA to a row, which takes its best out in rounds:
    ties over all of them, and rows whose tokens lie in one."""
    import torch

    logits = torch.zeros((64, vocab), dtype=getattr(torch, dtype), device="cuda")
    logits[8:16] = make(dtype, 8, vocab, 3)
    logits[16:24, : vocab // 2] = -4.0
    logits[24:32, vocab - 9:] = 3.0
    logits[32:40, :5] = 2.0
    bits = np.ones((64, (vocab + 31) // 32 * 32), dtype=bool)
    bits[40:48, : vocab - 700] = False
    bits[48:56, 300:] = False
    bits[56] = False
    bits[57:60, 5:vocab - 5] = False
    mask = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).cuda()
    scores = random_scores(1, 64, 3)
    check(logits, scores, 128, mask=mask)
    check(logits, scores, 128, mask=mask, renormalize=False)
    check(logits, torch.zeros_like(scores), 128)


def test_scores_of_zero_tie_whatever_their_sign():
    import torch

    scores = torch.tensor([[-0.0, 0.0, -0.0, 0.0]], device="cuda")
    finished = torch.tensor([[True, False, True, True]], device="cuda")
    logits = torch.full((4, 7), -float("inf"), device="cuda")
    logits[:, 3] = 1.5
    check(logits, scores, 4, finished=finished, end_token=5)


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_sorted_logits(order):
    import torch

    x = torch.linspace(-9, 9, 30000, device="cuda")
    x = x if order == "rising" else x.flip(0)
    check(torch.stack([x, x * 0.5]).contiguous(), random_scores(1, 2, 3), 64)


def test_a_cluster_of_allowed_tokens():
    """Many allowed tokens in one place of the row: few of the scan's threads see any."""
    import torch

    vocab = 16384
    bits = np.zeros((4, vocab), dtype=bool)
    for r, (at, n) in enumerate([(0, 1300), (5000, 2000), (16383, 1), (8, 1100)]):
        bits[r, at: at + n] = True
    mask = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).cuda()
    check(make("float16", 4, vocab, 8), random_scores(2, 2, 3), 64, mask=mask)


def test_identical_beams_are_ordered_by_beam():
    """Equal rows at different alignments have equal scores."""
    row = make("bfloat16", 1, 5001, 3)
    logits = make("bfloat16", 8, 5001, 4, stride=5001)
    logits.copy_(row.expand(8, -1))
    import torch

    check(logits, torch.zeros((1, 8), device="cuda"), 32)


def test_near_ties_are_decided_in_64_bits():
    """Beams whose log-sums differ by less than the 32-bit sums can tell: the scores differ by
    one small change far down the row."""
    import torch

    row = make("float32", 1, 30000, 3)
    logits = row.repeat(6, 1)
    for b in range(6):
        logits[b, 100 + b] -= 0.01 * (b + 1)
    check(logits, torch.zeros((1, 6), device="cuda"), 24)
    check(logits.half(), torch.zeros((1, 6), device="cuda"), 24, renormalize=False,
          mask=make_mask(6, 30000, 5, (0.7,)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_do_not_count(dtype):
    """-inf logits are never taken; masked NaN and infinities do not matter; the type's lowest
    value is a value."""
    import torch

    t = getattr(torch, dtype)
    logits = make(dtype, 8, 4000, 3)
    mask = make_mask(8, 4000, 4, (0.5,))
    blocked = torch.from_numpy(~np.stack([ref.allowed_bits(m, 4000) for m in mask.cpu().numpy()])).cuda()
    noise = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(t).max], device="cuda").to(t)
    logits[blocked] = noise.repeat(int(blocked.sum()) // 4 + 1)[: int(blocked.sum())]
    logits[:, 7::5] = torch.where(blocked[:, 7::5], logits[:, 7::5], -float("inf"))
    check(logits, random_scores(2, 4, 3), 8, mask=mask)
    lowest = torch.full((4, 300), torch.finfo(t).min, dtype=t, device="cuda")
    lowest[1, 40] = 1.0
    lowest[2] = -float("inf")
    lowest[3, :299] = -float("inf")
    check(lowest, random_scores(1, 4, 3), 12)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_rows_that_offer_nothing(dtype, bad):
    import torch

    logits = make(dtype, 12, 3000, 3)
    logits[1, 77] = float(bad)
    logits[6, 2999] = float(bad)
    logits[9] = float("nan")
    scores = random_scores(3, 4, 3)
    scores[0, 0], scores[1, 3], scores[2, 0] = -float("inf"), float("nan"), float("inf")
    check(logits, scores, 8)
    check(logits, scores, 8, renormalize=False, mask=make_mask(12, 3000, 4, (0.5,)))
    scores[:] = -float("inf")
    got = check(logits, scores, 8)
    assert (got.beams == -1).all()


@pytest.mark.parametrize("scale", [1e-3, 30.0, 2e5, 1e30])
def test_magnitudes(scale):
    logits = make("float32", 8, 6007, 3, scale=scale)
    check(logits, random_scores(2, 4, 3), 16)
    if scale > 1:
        check(make("bfloat16", 8, 6007, 3, scale=scale), random_scores(2, 4, 3), 16, renormalize=False)


def test_finished_beams():
    import torch

    logits = make("bfloat16", 24, 9000, 3)
    logits[5] = float("nan")  # an ended beam's logits are not read
    scores = random_scores(6, 4, 3)
    finished = torch.zeros((6, 4), dtype=torch.bool, device="cuda")
    finished[0, 1] = finished[1] = finished[2, 3] = True
    scores[2, 3] = -float("inf")
    for end_token in (0, 4711, 8999):
        check(logits, scores, 8, finished=finished, end_token=end_token, mask=make_mask(24, 9000, 4))
    check(logits, scores, 4, end_token=17)


def test_first_step_has_one_live_beam():
    scores = random_scores(4, 8, 3)
    scores[:, 1:] = -float("inf")
    check(make("float32", 32, 32000, 3), scores, 16, mask=make_mask(32, 32000, 4, (1.0, 0.5)))


@pytest.mark.parametrize("groups,beams,vocab,dtype", [(32, 8, 128256, "bfloat16"), (1, 4, 128256, "bfloat16"),
                                                      (6, 16, 151936, "float16"), (1, 64, 151936, "float32")])
def test_serving_sizes(groups, beams, vocab, dtype):
    logits = make(dtype, groups * beams, vocab, 3)
    check(logits, random_scores(groups, beams, 3), 2 * beams, mask=make_mask(groups * beams, vocab, 4, (1.0, 0.5, 0.001)))


def test_select_in_a_graph_and_on_another_stream():
    import torch

    from xgraph_b200.beams import beam_select

    logits = make("bfloat16", 16, 40001, 3)
    scores = random_scores(4, 4, 3)
    want = beam_select(logits, scores, candidates=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = beam_select(logits, scores, candidates=8, stream=side.cuda_stream)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    static, graphs = logits.clone(), []
    for _ in range(2):  # two graphs over the same inputs, replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = beam_select(static, scores, candidates=8, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for seed in (5, 6):
        static.copy_(make("bfloat16", 16, 40001, seed))
        want = beam_select(static, scores, candidates=8)
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_select_refusals():
    import torch

    from xgraph_b200.beams import beam_select

    logits, scores = make("float32", 8, 100, 3), random_scores(2, 4, 3)
    mask, finished = make_mask(8, 100, 3), torch.zeros((2, 4), dtype=torch.bool, device="cuda")
    beam_select(logits, scores, mask=mask, finished=finished, end_token=3)
    for change, message in [
        (dict(logits=logits.double()), "float32, bfloat16 or float16"), (dict(logits=logits[0]), "2-D"),
        (dict(logits=logits.t()), "contiguous row|row per beam"), (dict(logits=logits[:7]), "one row per beam"),
        (dict(logits=logits[:1].expand(8, -1)), "overlap"), (dict(scores=scores[0]), "groups, beams"),
        (dict(scores=scores.half()), "float32"), (dict(scores=scores.cpu()), "on cuda"),
        (dict(scores=scores.t().contiguous().t()), "contiguous"), (dict(mask=mask.long()), "int32"),
        (dict(mask=mask[:, :3]), "words"), (dict(mask=mask[:7]), "rows"),
        (dict(mask=mask[:1].expand(8, -1)), "overlap"), (dict(mask=mask.t().contiguous().t()), "contiguous row"),
        (dict(finished=finished.int()), "bool"), (dict(finished=finished[:, :3]), "shape"),
        (dict(end_token=None), "end_token"), (dict(end_token=100), "end_token"), (dict(end_token=-1), "end_token"),
        (dict(candidates=0), "candidates"), (dict(candidates=129), "candidates"), (dict(vocab=101), "vocab"),
        (dict(vocab=0), "vocab"), (dict(scores=torch.zeros((8, 0), device="cuda"), logits=logits[:0]), "beams"),
    ]:
        call = {"logits": logits, "scores": scores, "mask": mask, "finished": finished, "end_token": 3, **change}
        if "scores" in change and change["scores"].numel() == 0:
            call.update(mask=None, finished=None, end_token=None)
        with pytest.raises(ValueError, match=message):
            beam_select(call.pop("logits"), call.pop("scores"), **call)
    empty = beam_select(logits[:0], scores[:0], candidates=5)
    assert empty.scores.shape == (0, 5) and empty.finished.shape == (0, 5)


def test_overlapping_calls_on_two_streams():
    """Calls in flight together keep their own workspaces."""
    import torch

    from xgraph_b200.beams import beam_select

    inputs = [(make("bfloat16", 32, 60000, k), random_scores(4, 8, k)) for k in range(2)]
    want = [beam_select(*i, candidates=16) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, stream in enumerate(streams):
            got[k].append(beam_select(*inputs[k], candidates=16, stream=stream.cuda_stream))
    torch.cuda.synchronize()
    for k in range(2):
        for result in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[k]))


# ---------------------------------------------------------------------------------------

def parents_of(groups, beams, seed, shape=()):
    rng = np.random.default_rng(seed)
    out = rng.integers(0, beams, size=(*shape, groups, beams)).astype(np.int32)
    out[rng.random(out.shape) < 0.05] = -1
    out[rng.random(out.shape) < 0.02] = beams
    return out


def check_reorder(tensors, beams, *, lengths=None, dim=None, rows=None):
    import torch

    from xgraph_b200.beams import beam_reorder

    device = lambda a: None if a is None else torch.from_numpy(np.asarray(a, dtype=np.int32)).cuda()  # noqa: E731
    dims = dim if isinstance(dim, list) else [dim] * len(tensors)
    raw = [t.contiguous().view(torch.uint8).cpu().numpy().reshape(*t.shape, t.element_size()) for t in tensors]
    want = [ref.reorder(r, beams, lengths=lengths, dim=d, rows=rows) for r, d in zip(raw, dims)]
    beam_reorder(tensors, device(beams), lengths=device(lengths), dim=dim, rows=device(rows))
    for t, w in zip(tensors, want):
        got = t.contiguous().view(torch.uint8).cpu().numpy().reshape(w.shape)
        np.testing.assert_array_equal(got, w)


def filled(shape, dtype, seed=0):
    import torch

    gen = torch.Generator().manual_seed(seed)
    size = torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * size), generator=gen, dtype=torch.uint8)
    return raw.view(dtype).cuda()


@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("type_name", ["uint8", "bfloat16", "int32", "float64", "complex128"])
def test_reorder_whole_rows(beams, type_name):
    import torch

    dtype = getattr(torch, type_name)
    for shape in ((1,), (7,), (3, 5), (2, 4, 64)):
        tensors = [filled((3 * beams, *shape), dtype, k) for k in range(2)]
        check_reorder(tensors, parents_of(3, beams, beams))


@pytest.mark.parametrize("beams", [3, 8, 40])
@pytest.mark.parametrize("shape,dim", [((2, 9, 16), 2), ((9, 2, 16), 1), ((9,), 1), ((4, 9), 2), ((2, 3, 16, 9), 4),
                                       ((1, 5, 8), 1), ((3, 1, 8), 2), ((2, 3, 5, 8), 2)])
def test_reorder_written_positions(beams, shape, dim):
    import torch

    lengths = [0, shape[dim - 1], 1, max(0, shape[dim - 1] - 1), 99, -4]
    for dtype in (torch.bfloat16, torch.int32):
        check_reorder([filled((6 * beams, *shape), dtype)], parents_of(6, beams, 3), lengths=lengths, dim=dim)


def test_reorder_strided_tensors():
    import torch

    beams = 4
    for base_shape, view in [
        ((12, 2, 6, 16), lambda t: t[:, 1]),                       # one half of an interleaved cache
        ((2, 12, 6, 16), lambda t: t[1]),
        ((6, 12, 16), lambda t: t.transpose(0, 1)),                 # rows not outermost
        ((6, 16, 12), lambda t: t.permute(2, 0, 1)),                # rows innermost
        ((12, 6, 20), lambda t: t[:, :, 3:19]),
        ((12, 6, 20), lambda t: t[:, ::2, :16]),
        ((12, 33), lambda t: t[:, 1:]),
        ((13, 32), lambda t: t[1:]),
        ((24, 8), lambda t: t[::2]),
    ]:
        for dtype in (torch.float16, torch.float32):
            base = filled(base_shape, dtype)
            tensor = view(base)
            before = base.clone()
            touched = view(torch.ones_like(base, dtype=torch.bool).logical_not_())
            check_reorder([tensor], parents_of(3, beams, 3))
            marks = torch.zeros_like(base, dtype=torch.bool)
            view(marks).fill_(True)
            del touched
            same = base.view(torch.int16 if dtype == torch.float16 else torch.int32) == before.view(
                torch.int16 if dtype == torch.float16 else torch.int32)
            assert bool((same | marks).all())  # nothing outside the view changed


def test_reorder_many_tensors_and_layouts():
    import torch

    tensors, dims = [], []
    for k in range(150):
        tensors.append(filled((8, 2, 5, 8) if k % 3 else (8, 5, 2, 4), torch.bfloat16 if k % 2 else torch.float32, k))
        dims.append(2 if k % 3 else 1)
    check_reorder(tensors, parents_of(2, 4, 5), lengths=[3, 5], dim=dims)


def test_reorder_named_rows():
    import torch

    rng = np.random.default_rng(3)
    rows = rng.permutation(40)[:24].reshape(3, 8)
    check_reorder([filled((40, 9), torch.int32)], parents_of(3, 8, 5), rows=rows)
    rows[1, 2], rows[2, 0] = -1, 40  # outside the tensor: left out, as parents too
    check_reorder([filled((40, 9), torch.int32)], parents_of(3, 8, 6), rows=rows)


def test_reorder_refusals():
    import torch

    from xgraph_b200.beams import beam_reorder

    beams = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    cache, lengths = filled((8, 3, 5), torch.float32), torch.zeros(2, dtype=torch.int32, device="cuda")
    beam_reorder([], beams)
    for args, options, message in [
        (([cache, cache], beams), {}, "share memory"), (([cache, cache[:, 1:]], beams), dict(rows=beams), "share memory"),
        (([cache[:7]], beams), {}, "8 rows"), (([cache, filled((9, 2), torch.int32)], beams), {}, "same number of rows"),
        (([cache.cpu()], beams), {}, "on cuda"), (([cache], beams.cpu()), {}, "GPU"), (([cache], beams.long()), {}, "int32"),
        (([cache], beams), dict(dim=1), "lengths"), (([cache], beams), dict(lengths=lengths), "dim"),
        (([cache], beams), dict(lengths=lengths, dim=3), "dim"), (([cache], beams), dict(lengths=lengths, dim=0), "dim"),
        (([cache], beams), dict(lengths=lengths, dim=[1, 1]), "one entry per tensor"),
        (([cache], beams), dict(lengths=lengths[:1], dim=1), "shape"), (([cache], beams), dict(rows=beams[:1]), "shape"),
        (([cache[:1].expand(8, -1, -1)], beams), {}, "overlap"), (([None], beams), {}, "torch tensors"),
        (([cache.clone().requires_grad_()], beams), {}, "gradients"),
        (([filled((8, 3, 4, 5, 6), torch.float32)[:, ::2, ::2, ::2, ::2]], beams), {}, "two places"),
    ]:
        with pytest.raises(ValueError, match=message):
            beam_reorder(*args, **options)


def test_reorder_interleaved_halves():
    """Two views of one buffer that share no element are two tensors."""
    import torch

    both = filled((8, 2, 6, 16), torch.bfloat16)
    check_reorder([both[:, 0], both[:, 1]], parents_of(2, 4, 3), lengths=[3, 6], dim=1)


def test_reorder_a_cache_past_32_bits():
    """Rows more than 2^31 bytes from the tensor's start."""
    import torch

    from xgraph_b200.beams import beam_reorder

    rows, width = 5, 1 << 30
    cache = torch.zeros((rows, width), dtype=torch.uint8, device="cuda")
    cache[:, -64:] = torch.arange(rows, dtype=torch.uint8, device="cuda")[:, None]
    cache[:, 12345] = torch.arange(10, 10 + rows, dtype=torch.uint8, device="cuda")
    beam_reorder(cache, torch.tensor([[4, 1, 0, 2, 3]], dtype=torch.int32, device="cuda"))
    assert cache[:, -1].tolist() == [4, 1, 0, 2, 3] and cache[:, -64].tolist() == [4, 1, 0, 2, 3]
    assert cache[:, 12345].tolist() == [14, 11, 10, 12, 13]


def test_reorder_in_a_graph():
    import torch

    from xgraph_b200.beams import beam_reorder

    cache = filled((8, 4, 64), torch.float32)
    beams = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    keep = cache.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        beam_reorder(cache, beams, stream=torch.cuda.current_stream().cuda_stream)
    parents = parents_of(2, 4, 9)
    beams.copy_(torch.from_numpy(parents))
    graph.replay()
    torch.cuda.synchronize()
    want = ref.reorder(keep.view(torch.int32).cpu().numpy(), parents)
    np.testing.assert_array_equal(cache.view(torch.int32).cpu().numpy(), want)


# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("beams", [1, 2, 4, 7, 32, 64])
@pytest.mark.parametrize("steps", [0, 1, 2, 31, 32, 33, 100, 1031])
def test_sequences(beams, steps):
    import torch

    from xgraph_b200.beams import beam_sequences

    rng = np.random.default_rng(steps * 100 + beams)
    tokens = rng.integers(0, 1 << 30, size=(steps, 3, beams)).astype(np.int32)
    parents = rng.integers(0, beams, size=(steps, 3, beams)).astype(np.int32)
    parents[rng.random(parents.shape) < 0.5 / max(steps, 1)] = -1
    parents[rng.random(parents.shape) < 0.1 / max(steps, 1)] = beams
    for lengths in (None, [0, steps, steps // 2], [-3, steps + 5, min(1, steps)]):
        given = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
        got = beam_sequences(torch.from_numpy(tokens).cuda(), torch.from_numpy(parents).cuda(), lengths=given, pad_token=-7)
        np.testing.assert_array_equal(got.cpu().numpy(), ref.sequences(tokens, parents, lengths=lengths, pad=-7))


def test_sequences_refusals():
    import torch

    from xgraph_b200.beams import beam_sequences

    trace = torch.zeros((6, 2, 4), dtype=torch.int32, device="cuda")
    for args, options, message in [
        ((trace.long(), trace), {}, "int32"), ((trace, trace[:5]), {}, "same shape"), ((trace[0], trace[0]), {}, "3-D"),
        ((trace, trace.transpose(1, 2).contiguous().transpose(1, 2)), {}, "unit stride"),
        ((trace, trace), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), "shape"),
        ((trace, trace), dict(pad_token=1 << 31), "int32"),
        ((torch.zeros((2, 2, 65), dtype=torch.int32, device="cuda"),) * 2, {}, "1 to 64 beams"),
    ]:
        with pytest.raises(ValueError, match=message):
            beam_sequences(*args, **options)
    assert beam_sequences(trace[:, :0], trace[:, :0]).shape == (0, 4, 6)


def test_sequences_longer_than_a_window_and_strided():
    import torch

    from xgraph_b200.beams import beam_sequences

    rng = np.random.default_rng(3)
    for steps, beams in ((5000, 64), (60000, 1)):
        tokens = rng.integers(0, 1 << 30, size=(steps, 5, beams)).astype(np.int32)
        parents = rng.integers(0, beams, size=(steps, 5, beams)).astype(np.int32)
        device_tokens, device_parents = torch.from_numpy(tokens).cuda(), torch.from_numpy(parents).cuda()
        got = beam_sequences(device_tokens[:, 1:4], device_parents[:, 1:4])
        np.testing.assert_array_equal(got.cpu().numpy(), ref.sequences(tokens[:, 1:4], parents[:, 1:4]))
        got = beam_sequences(device_tokens[::2], device_parents[::2])
        np.testing.assert_array_equal(got.cpu().numpy(), ref.sequences(tokens[::2], parents[::2]))
