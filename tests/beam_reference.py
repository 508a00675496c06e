"""Beam search's definitions in 64 bits on the host, for tests (numpy, one candidate at a time)."""

from __future__ import annotations

import numpy as np


def allowed_bits(mask_row, vocab: int) -> np.ndarray:
    bits = np.unpackbits(np.ascontiguousarray(mask_row).view(np.uint8), bitorder="little")
    return bits[:vocab] != 0


def select(logits, scores, candidates: int, *, vocab=None, mask=None, finished=None, end_token=None, renormalize=True):
    """(scores float64, beams, tokens, finished) of every group, best first; also, per group, the
    smallest distance between two of the group's leading candidates that come from different
    beams (what the order of a result can turn on)."""
    groups, beams = scores.shape
    vocab = logits.shape[1] if vocab is None else vocab
    shape = (groups, candidates)
    out = np.full(shape, -np.inf), np.full(shape, -1), np.full(shape, -1), np.zeros(shape, bool)
    gaps = np.full(groups, np.inf)
    for g in range(groups):
        found = []
        for b in range(beams):
            score = np.float64(scores[g, b])
            if not np.isfinite(score):
                continue
            if finished is not None and finished[g, b]:
                found.append((-score, b, end_token, True))
                continue
            x = logits[g * beams + b, :vocab].astype(np.float64)
            may = allowed_bits(mask[g * beams + b], vocab) if mask is not None else np.ones(vocab, bool)
            counted = x[may] if renormalize else x
            if not len(counted):
                continue
            with np.errstate(all="ignore"):
                top = counted.max()
                total = np.exp(counted - top).sum()
            if not (np.isfinite(total) and total > 0):
                continue
            tokens = np.flatnonzero(may & (x != -np.inf))
            best = tokens[np.argsort(-x[tokens], kind="stable")][: candidates + 1]
            for v in best:
                s = score + ((x[v] - top) - np.log(total))
                with np.errstate(over="ignore"):
                    kept = np.isfinite(np.float32(s))
                if kept:
                    found.append((-s, b, int(v), end_token is not None and v == end_token))
        found.sort(key=lambda c: c[:3])
        for a, b in zip(found[:candidates], found[1: candidates + 1]):
            if a[1] != b[1]:
                gaps[g] = min(gaps[g], b[0] - a[0])
        for n, (s, b, v, done) in enumerate(found[:candidates]):
            out[0][g, n], out[1][g, n], out[2][g, n], out[3][g, n] = -s, b, v, done
    return out, gaps


def reorder(tensor, beams, *, lengths=None, dim=None, rows=None):
    """A copy of `tensor` (rows first) as the reordering leaves it."""
    groups, per_group = beams.shape
    rows = np.arange(groups * per_group).reshape(beams.shape) if rows is None else rows
    out = tensor.copy()
    for g in range(groups):
        for b in range(per_group):
            if not 0 <= beams[g, b] < per_group:
                continue
            to, source = rows[g, b], rows[g, beams[g, b]]
            if not (0 <= to < len(tensor) and 0 <= source < len(tensor)):
                continue
            if lengths is None:
                out[to] = tensor[source]
            else:
                part = [slice(None)] * (tensor.ndim - 1)
                part[dim - 1] = slice(0, max(0, int(lengths[g])))
                out[(to, *part)] = tensor[(source, *part)]
    return out


def sequences(tokens, beams, *, lengths=None, pad=-1):
    steps, groups, per_group = tokens.shape
    out = np.full((groups, per_group, steps), pad, dtype=np.int64)
    for g in range(groups):
        length = steps if lengths is None else min(max(int(lengths[g]), 0), steps)
        for k in range(per_group):
            at = k
            for t in range(length - 1, -1, -1):
                out[g, k, t] = tokens[t, g, at]
                at = beams[t, g, at]
                if not 0 <= at < per_group:
                    break
    return out
