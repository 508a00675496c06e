"""How far the selection's log-sums are from the exact ones, and what the order of two beams makes of it.

Rows of few levels (some tokens at a high one, the others at one floor) have all their terms' roundings
alike, so that they add up instead of cancelling; their exact log-sums are a formula.  A row's
log-sum may be off by MARGIN, half of what the selection calls near (kNear in csrc/beams.cu,
where the bound is derived); beams nearer than that are ordered by 64-bit sums, so the order must
be the exact one however small the distance.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")
MARGIN = 1e-6


def levels(dtype, rows, vocab, seed, *, below=(0.0, 24.0), hot=None, shift=(0.0,)):
    """Logits [rows, vocab] whose tokens `hot` (default: by row none, one, every 64th, or the first of each
    512 in 8,192) stand above one floor; the floor's and the high level's values, and how many are high."""
    import torch

    rng = np.random.default_rng(seed)
    kind = getattr(torch, dtype)
    high = torch.from_numpy(rng.choice(np.asarray(shift), rows) + rng.uniform(-2, 2, rows)).to(kind)
    floor = (high.double() - torch.from_numpy(rng.uniform(*below, rows))).to(kind)
    logits = floor.cuda()[:, None].expand(rows, vocab).contiguous()
    count = np.zeros(rows, dtype=np.int64)
    sets = [hot] if hot is not None else [np.zeros(0, int), np.array([vocab // 3]), np.arange(0, vocab, 64),
                                          np.arange(0, min(vocab, 8192), 512)]
    for k, at in enumerate(sets):
        own = torch.arange(k, rows, len(sets))
        logits[own.cuda()[:, None], torch.from_numpy(at).cuda()[None, :]] = high[own].cuda()[:, None]
        count[k:: len(sets)] = len(at)
    return logits, floor.double().numpy(), high.double().numpy(), count


def best_log(floor, high, count, vocab):
    """log-probability of a row's best token: -log(sum of exp(x - best))."""
    top = np.where(count > 0, high, floor)
    low = np.minimum(np.where(count > 0, floor - top, 0.0), 0.0)
    return -np.log(count * np.exp(np.where(count > 0, high - top, -np.inf)) + (vocab - count) * np.exp(low))


def errors(logits, best):
    """What the selection's log-sums are off by: scores that bring the best candidates next to 0, where the
    float32 result shows them."""
    import torch

    from xgraph_b200.beams import beam_select

    scores = (-best).astype(np.float32)
    got = beam_select(logits, torch.from_numpy(scores[:, None]).cuda(), candidates=1)
    return got.scores[:, 0].cpu().numpy().astype(np.float64) - (scores.astype(np.float64) + best)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1200, 300), (1200, 4097), (64, 128256), (512, 128256), (1200, 40001)])
def test_log_sums_of_few_levels(dtype, rows, vocab):
    logits, floor, high, count = levels(dtype, rows, vocab, rows + vocab, shift=(0.0, 0.0, 12.0, -40.0, 300.0))
    off = errors(logits, best_log(floor, high, count, vocab))
    assert np.abs(off).max() <= MARGIN, np.abs(off).max()


@pytest.mark.parametrize("below", [(5.0, 11.0), (10.0, 14.0)])
def test_log_sums_of_the_largest_vocabulary(below):
    """A share of a row is all of it: as many tokens as one sum can hold."""
    rows, vocab = 1200, 1 << 20
    logits, floor, high, count = levels("bfloat16", rows, vocab, 7, below=below, hot=np.arange(8) * 1024)
    off = errors(logits, best_log(floor, high, count, vocab))
    assert np.abs(off).max() <= MARGIN, np.abs(off).max()


@pytest.mark.parametrize("shift", [7e4, -7e4, 1e6])
def test_log_sums_far_from_zero(shift):
    logits, floor, high, count = levels("float32", 512, 128256, 11, shift=(shift,))
    off = errors(logits, best_log(floor, high, count, 128256))
    assert np.abs(off).max() <= MARGIN, np.abs(off).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.5, 3.0])
def test_log_sums_of_random_rows(dtype, scale):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = (torch.randn((512, 50257), generator=gen, device="cuda") * scale).to(getattr(torch, dtype))
    x = logits.double()
    best = (x.amax(1) - torch.logsumexp(x, 1)).cpu().numpy()
    off = errors(logits, best)
    assert np.abs(off).max() <= MARGIN, np.abs(off).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,below", [(512, 128256, (4.0, 10.0)), (512, 128256, (5.0, 6.0)),
                                              (1200, 1 << 20, (10.0, 11.5))])
def test_rows_unlike_each_other_are_ordered_exactly(dtype, rows, vocab, below):
    """Two beams a group whose log-sums are off in opposite directions, the one that comes out too low the
    better one by less than 6e-7."""
    import torch

    from xgraph_b200.beams import beam_select

    hot = np.arange(8) * (512 if dtype == "float32" else 1024)  # a warp's part of a step each
    if vocab < 1 << 20:
        hot = np.concatenate([hot, 65536 + hot])
    logits, floor, high, count = levels(dtype, rows, vocab, 3, below=below, hot=hot)
    best = best_log(floor, high, count, vocab)
    by_error = np.argsort(errors(logits, best))
    low, up = by_error[: rows // 2], by_error[::-1][: rows // 2]  # the farthest two, the next two, ...
    better = np.zeros(rows // 2, dtype=np.float32)
    worse = (best[low] - best[up] - 1e-9).astype(np.float32)
    over = worse.astype(np.float64) + best[up] >= best[low] - 1e-10
    worse[over] = np.nextafter(worse[over], np.float32(-np.inf))
    gap = best[low] - (worse.astype(np.float64) + best[up])
    assert (gap > 1e-10).all() and (gap < 6e-7).all()
    flip = np.arange(rows // 2) % 2 == 1  # the better beam first or second
    order = np.where(flip[:, None], np.stack([up, low], 1), np.stack([low, up], 1))
    scores = np.where(flip[:, None], np.stack([worse, better], 1), np.stack([better, worse], 1))
    logits = logits[torch.from_numpy(order.reshape(-1)).cuda()]
    got = beam_select(logits, torch.from_numpy(scores.astype(np.float32)).cuda(), candidates=2)
    np.testing.assert_array_equal(got.beams.cpu().numpy(), np.stack([flip, flip], 1).astype(np.int32))
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), np.tile(hot[:2], (rows // 2, 1)))
