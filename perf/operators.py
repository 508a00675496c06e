"""Workloads of the beam-search operators: selection over beams and vocabulary, reordering of
per-beam state in place, and the back-trace of the written sequences.

`run` computes a case's operator with elementary torch operations, or, where `own` is true,
through xgraph_b200's entry points.  Every case is one call as a decoding loop makes it.
"""

from __future__ import annotations

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4}
# What a batch of constrained rows is made of: free text (nothing blocked), a relation label
# (a few tokens), a label's first token (half the vocabulary), and a row with no way on.
MASK_SHARES = (0.40, 0.35, 0.23, 0.02)
RELATION_TOKENS = 116  # tokens of a relation segment's mask at the 100,000-entity configuration
FINISHED = 0.2         # share of beams that have ended in a batch with ended beams


def listed():
    return [
        # one decoding step of the 16-row toy configuration, all rows constrained
        dict(name="select-toy", op="select", groups=4, beams=4, vocab=256, pad=0, dtype="f32", candidates=8,
             mask=True, finished=False, first=False, renormalize=True),
        # a single request with four beams at a large vocabulary: latency, few rows
        dict(name="select-request", op="select", groups=1, beams=4, vocab=128256, pad=0, dtype="bf16", candidates=8,
             mask=False, finished=False, first=False, renormalize=True),
        # 64 rows of the 32,000-token configuration at the first step (one live beam a request)
        dict(name="select-first", op="select", groups=8, beams=8, vocab=32000, pad=0, dtype="f32", candidates=16,
             mask=True, finished=False, first=True, renormalize=True),
        # a served batch of 256 rows without masks, some beams ended
        dict(name="select-batch", op="select", groups=32, beams=8, vocab=128256, pad=0, dtype="bf16", candidates=8,
             mask=False, finished=True, first=False, renormalize=True),
        # the same batch under the engine's masks
        dict(name="select-spans", op="select", groups=32, beams=8, vocab=128256, pad=0, dtype="bf16", candidates=16,
             mask=True, finished=False, first=False, renormalize=True),
        # wide beams at the largest vocabulary, the model's own probabilities, padded columns
        dict(name="select-wide", op="select", groups=32, beams=16, vocab=151936, pad=64, dtype="f16", candidates=32,
             mask=True, finished=True, first=False, renormalize=False),
        # token histories and small state rows of 16 slots in arbitrary order
        dict(name="reorder-toy", op="reorder", groups=4, beams=4, tensors=2, heads=1, positions=64, width=1,
             layout="phw", dtype="i32", lengths=False, rows=True),
        # the caches of one request with four beams, many layers, part of the positions written
        dict(name="reorder-request", op="reorder", groups=1, beams=4, tensors=48, heads=8, positions=1024, width=64,
             layout="hpw", dtype="bf16", lengths=True, rows=False),
        # the caches of a served batch
        dict(name="reorder-batch", op="reorder", groups=32, beams=8, tensors=8, heads=8, positions=512, width=64,
             layout="phw", dtype="bf16", lengths=True, rows=False),
        # the answers of the toy configuration's 64 steps
        dict(name="sequences-toy", op="sequences", groups=4, beams=4, steps=64, lengths=False),
        # a served batch, ragged lengths up to 1,024
        dict(name="sequences-batch", op="sequences", groups=32, beams=8, steps=1024, lengths=True),
        # wide beams and long answers
        dict(name="sequences-wide", op="sequences", groups=64, beams=32, steps=2048, lengths=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("select", "select", "reorder", "sequences"))
    if op == "select":
        vocab = _log_int(rng, 200, 151936)
        beams = _log_int(rng, 1, 32)
        most = max(1, min(256, 32 * 16 * 151936 // (vocab * beams) // 2))
        return dict(op=op, groups=_log_int(rng, 1, most), beams=beams, vocab=vocab, pad=rng.choice((0, 0, 1, 8, 64)),
                    dtype=rng.choice(("f32", "bf16", "f16")), candidates=rng.choice((beams, 2 * beams)),
                    mask=rng.random() < 0.6, finished=rng.random() < 0.4, first=rng.random() < 0.2,
                    renormalize=rng.random() < 0.7)
    if op == "reorder":
        beams, heads, width = _log_int(rng, 1, 32), rng.choice((1, 2, 5, 8)), rng.choice((1, 7, 32, 64, 128))
        positions, tensors, dtype = _log_int(rng, 1, 2048), _log_int(rng, 1, 32), rng.choice(("f32", "bf16", "i32"))
        size = tensors * beams * heads * positions * width * SIZES[dtype]
        if size > 1 << 29:
            tensors, size = 1, size // tensors
        return dict(op=op, groups=_log_int(rng, 1, max(1, min(64, (1 << 29) // size))), beams=beams, tensors=tensors,
                    heads=heads, positions=positions, width=width, layout=rng.choice(("hpw", "phw")), dtype=dtype,
                    lengths=rng.random() < 0.6, rows=rng.random() < 0.3)
    return dict(op=op, groups=_log_int(rng, 1, 64), beams=_log_int(rng, 1, 32), steps=_log_int(rng, 1, 2048),
                lengths=rng.random() < 0.6)


# ---------------------------------------------------------------------------------------
# inputs

def _parents(g, shape, beams):
    """Parent beams as a search has them: the better beams go on more often, some groups go
    on unchanged, a few places are unfilled (-1)."""
    u = torch.rand(shape, generator=g)
    parents = (beams * u**1.5).to(torch.int32).clamp_(max=beams - 1)
    same = torch.rand(shape[:-1], generator=g) < 0.15
    parents = torch.where(same[..., None], torch.arange(beams, dtype=torch.int32), parents)
    return torch.where(torch.rand(shape, generator=g) < 0.002, -1, parents).to(torch.int32)


def _prepare_select(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
    rows, cols = groups * beams, vocab + case["pad"]
    logits = torch.randn((rows, cols), generator=gen, device="cuda") * 2.0
    # a model prefers a few tokens of each row
    liked = torch.randint(vocab, (rows, 12), generator=gen, device="cuda")
    logits.scatter_add_(1, liked, torch.rand((rows, 12), generator=gen, device="cuda") * 10.0)
    scores = -20.0 * torch.rand((groups, beams), generator=gen, device="cuda").sort(1).values
    if case["first"]:
        scores[:, 1:] = -float("inf")
    mask = finished = None
    if case["mask"]:
        kind = torch.rand((rows, 1), generator=gen, device="cuda")
        a, b, c = MASK_SHARES[0], MASK_SHARES[0] + MASK_SHARES[1], 1.0 - MASK_SHARES[3]
        few = min(0.5, RELATION_TOKENS / vocab)
        share = torch.where(kind < a, 2.0, torch.where(kind < b, few, torch.where(kind < c, 0.5, -1.0)))
        words = (vocab + 31) // 32
        bits = torch.zeros((rows, words * 32), dtype=torch.bool, device="cuda")
        bits[:, :vocab] = torch.rand((rows, vocab), generator=gen, device="cuda") < share
        weights = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        mask = (bits.view(rows, words, 32) * weights).sum(-1).to(torch.int32)
    if case["finished"]:
        finished = torch.rand((groups, beams), generator=gen, device="cuda") < FINISHED
    return dict(case=case, logits=logits.to(DTYPES[case["dtype"]]), scores=scores, mask=mask, finished=finished,
                end_token=vocab // 2)


def _prepare_reorder(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    groups, beams = case["groups"], case["beams"]
    h, p, w = case["heads"], case["positions"], case["width"]
    shape = (groups * beams, *((h, p, w) if case["layout"] == "hpw" else (p, h, w)))
    if case["dtype"] == "i32":
        tensors = [torch.randint(1 << 30, shape, generator=gen, dtype=torch.int32, device="cuda")
                   for _ in range(case["tensors"])]
    else:
        tensors = [torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)
                   for _ in range(case["tensors"])]
    parents = _parents(host, (groups, beams), beams).cuda()
    lengths = rows = None
    if case["lengths"]:
        lengths = torch.randint(p // 2, p + 1, (groups,), generator=host, dtype=torch.int32).cuda()
    if case["rows"]:
        rows = torch.randperm(groups * beams, generator=host).to(torch.int32).view(groups, beams).cuda()
    return dict(case=case, tensors=tensors, parents=parents, lengths=lengths, rows=rows)


def _prepare_sequences(case, seed):
    host = torch.Generator().manual_seed(seed)
    shape = (case["steps"], case["groups"], case["beams"])
    tokens = torch.randint(128256, shape, generator=host, dtype=torch.int32).cuda()
    parents = _parents(host, shape, case["beams"]).cuda()
    lengths = None
    if case["lengths"]:
        lengths = torch.randint(case["steps"] // 16, case["steps"] + 1, (case["groups"],), generator=host,
                                dtype=torch.int32).cuda()
    return dict(case=case, tokens=tokens, parents=parents, lengths=lengths)


def prepare(case, seed):
    return {"select": _prepare_select, "reorder": _prepare_reorder, "sequences": _prepare_sequences}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------
# one pass

def run(state):
    op = state["case"]["op"]
    if op == "select":
        return _select_own(state) if own else _select_plain(state)
    if op == "reorder":
        return _reorder_own(state) if own else _reorder_plain(state)
    return _sequences_own(state) if own else _sequences_plain(state)


def _select_own(state):
    from xgraph_b200.beams import beam_select

    case = state["case"]
    got = beam_select(state["logits"], state["scores"], mask=state["mask"], finished=state["finished"],
                      candidates=case["candidates"], vocab=case["vocab"], end_token=state["end_token"],
                      renormalize=case["renormalize"])
    return got.scores, got.beams, got.tokens, got.finished


def _select_plain(state):
    """The order of two beams' candidates turns on the difference of their log-sums, so scores
    and sums are in 64 bits; within a row the order is the logits' own."""
    case, scores, finished = state["case"], state["scores"], state["finished"]
    groups, beams, vocab, wanted = case["groups"], case["beams"], case["vocab"], case["candidates"]
    rows = groups * beams
    x = state["logits"][:, :vocab].float()
    allowed = x != -float("inf")
    if state["mask"] is not None:
        bits = (state["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=x.device)) & 1
        allowed &= bits.view(rows, -1)[:, :vocab] != 0
    shown = torch.where(allowed, x, -float("inf"))
    counted = shown if case["renormalize"] else x
    top = counted.amax(1, keepdim=True)
    centre = torch.where(top.isfinite(), top, 0.0).double()
    total = (counted.double() - centre).exp().sum(1, keepdim=True)
    base = scores.view(rows, 1).double()
    alive = base.isfinite() & total.isfinite() & (total > 0)
    # a row's best: by the logit, then the lowest token (a whole-number key holds both)
    bits = (shown + 0.0).view(torch.int32).long()
    rising = torch.where(bits < 0, -(bits + (1 << 31)) - 1, bits)
    key = (rising << 20) - torch.arange(vocab, device=x.device)
    token = key.topk(min(wanted, vocab), 1).indices
    value = base + ((shown.gather(1, token).double() - centre) - total.log())
    value = torch.where(alive & allowed.gather(1, token), value, -float("inf"))
    if finished is not None:
        ended = finished.view(rows, 1)
        first = torch.arange(token.shape[1], device=x.device) == 0
        value = torch.where(ended, torch.where(first & base.isfinite(), base, -float("inf")), value)
        token = torch.where(ended, torch.where(first, state["end_token"], vocab), token)
    value = torch.where(value.float().isfinite(), value, -float("inf"))
    # the group's best: by the score, then the lowest (beam, token)
    per = token.shape[1]
    beam = torch.arange(beams, device=x.device).view(1, beams, 1).expand(groups, beams, per).reshape(groups, -1)
    flat, order = (beam * (vocab + 1) + token.view(groups, -1)).sort(1)
    ranked = value.view(groups, -1).gather(1, order).sort(dim=1, descending=True, stable=True)
    count = min(wanted, beams * per)
    best = ranked.values[:, :count]
    flat = flat.gather(1, ranked.indices[:, :count])
    filled = best > -float("inf")
    out_scores = torch.full((groups, wanted), -float("inf"), device=x.device)
    out_scores[:, :count] = best.float()
    out_beams = torch.full((groups, wanted), -1, dtype=torch.int32, device=x.device)
    out_beams[:, :count] = torch.where(filled, flat // (vocab + 1), -1).int()
    out_tokens = torch.full((groups, wanted), -1, dtype=torch.int32, device=x.device)
    out_tokens[:, :count] = torch.where(filled, flat % (vocab + 1), -1).int()
    done = out_tokens == state["end_token"]
    if finished is not None:
        done |= finished.gather(1, out_beams.clamp(min=0).long()) & (out_beams >= 0)
    return out_scores, out_beams, out_tokens, done


def _reorder_own(state):
    from xgraph_b200.beams import beam_reorder

    dim = 2 if state["case"]["layout"] == "hpw" else 1
    beam_reorder(state["tensors"], state["parents"], lengths=state["lengths"],
                 dim=dim if state["lengths"] is not None else None, rows=state["rows"])
    return state["tensors"]


def _reorder_plain(state):
    parents, lengths, rows = state["parents"], state["lengths"], state["rows"]
    groups, beams = parents.shape
    place = torch.arange(beams, device=parents.device).expand(groups, beams)
    inside = (parents >= 0) & (parents < beams)
    source = torch.where(inside, parents, place).long()
    at = torch.arange(groups * beams, device=parents.device).view(groups, beams) if rows is None else rows.long()
    source, at = at.gather(1, source).view(-1), at.view(-1)
    written = None
    if lengths is not None:
        position = torch.arange(state["case"]["positions"], device=parents.device)
        written = (position < lengths.view(groups, 1, 1)).expand(groups, beams, -1).reshape(groups * beams, -1)
        written = written[:, None, :, None] if state["case"]["layout"] == "hpw" else written[:, :, None, None]
    return [_moved(t, source, at, written) for t in state["tensors"]]


def _moved(tensor, source, at, written):
    taken = tensor[source]
    tensor[at] = taken if written is None else torch.where(written, taken, tensor[at])
    return tensor


def _sequences_own(state):
    from xgraph_b200.beams import beam_sequences

    return beam_sequences(state["tokens"], state["parents"], lengths=state["lengths"], pad_token=-1)


def _sequences_plain(state):
    """The beam of each step, by composing the steps' parent maps over doubling distances (a
    last place, beams, stands for no beam and maps to itself)."""
    tokens, parents, lengths = state["tokens"], state["parents"], state["lengths"]
    steps, groups, beams = tokens.shape
    step = torch.arange(steps, device=tokens.device).view(steps, 1, 1)
    length = torch.full((groups,), steps, device=tokens.device) if lengths is None else lengths.long()
    own_place = torch.arange(beams + 1, device=tokens.device).expand(steps, groups, beams + 1)
    maps = own_place.clone()
    linked = torch.where((parents >= 0) & (parents < beams), parents.long(), beams)
    maps[:-1, :, :beams] = linked[1:]
    maps = torch.where(step + 1 < length.view(1, groups, 1), maps, own_place)
    reach = 1
    while reach < steps:
        maps[:-reach] = maps[:-reach].gather(2, maps[reach:])
        reach *= 2
    padded = torch.cat([tokens, torch.full_like(tokens[:, :, :1], -1)], 2)
    written = padded.gather(2, maps[:, :, :beams])
    written = torch.where(step < length.view(1, groups, 1), written, -1)
    return written.permute(1, 2, 0).contiguous()


# ---------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    if case["op"] == "select":
        rows, vocab = case["groups"] * case["beams"], case["vocab"]
        live = 1.0 - FINISHED if case["finished"] else 1.0
        live *= 1.0 / case["beams"] if case["first"] else 1.0
        read = float(vocab)
        if case["mask"] and case["renormalize"]:
            read = (MASK_SHARES[0] + 0.5 * MASK_SHARES[2]) * vocab + MASK_SHARES[1] * min(vocab * 0.5, RELATION_TOKENS)
        size = live * rows * read * SIZES[case["dtype"]] + rows * 4
        size += live * rows * ((vocab + 31) // 32) * 4 if case["mask"] else 0
        return {"bytes": size + case["groups"] * case["candidates"] * 13, "flops": 4.0 * live * rows * read}
    if case["op"] == "reorder":
        host = torch.Generator().manual_seed(0)
        groups, beams = case["groups"], case["beams"]
        parents = _parents(host, (256, beams), beams)
        moved = (parents >= 0) & (parents != torch.arange(beams))
        sources = sum(len(set(p[m].tolist())) for p, m in zip(parents, moved)) / 256
        share = 0.75 if case["lengths"] else 1.0
        row = case["tensors"] * case["heads"] * case["positions"] * case["width"] * SIZES[case["dtype"]] * share
        return {"bytes": groups * (sources + float(moved.sum()) / 256) * row + groups * beams * 4, "flops": 0}
    share = 0.53 if case["lengths"] else 1.0
    entries = case["groups"] * case["beams"] * case["steps"]
    return {"bytes": entries * (8 * share + 4), "flops": 0}


# ---------------------------------------------------------------------------------------
# the definitions, in 64 bits, on the host

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(state)
    if case["op"] == "reorder":
        return _exact_reorder(state)
    return _exact_sequences(state)


def _exact_select(state):
    case = state["case"]
    beams, vocab, wanted = case["beams"], case["vocab"], case["candidates"]
    scores = state["scores"].cpu().double().numpy()
    logits = state["logits"][:, :vocab].float().cpu().numpy()
    mask = None if state["mask"] is None else state["mask"].cpu().numpy().view(np.uint8)
    ended = None if state["finished"] is None else state["finished"].cpu().numpy()
    shape = (case["groups"], wanted)
    out = np.full(shape, -np.inf), np.full(shape, -1, np.int32), np.full(shape, -1, np.int32), np.zeros(shape, bool)
    for g in range(case["groups"]):
        found = []
        for b in range(beams):
            score = scores[g, b]
            if not np.isfinite(score):
                continue
            if ended is not None and ended[g, b]:
                found.append((-score, b, state["end_token"], True))
                continue
            x = logits[g * beams + b].astype(np.float64)
            may = np.flatnonzero(x != -np.inf)
            if mask is not None:
                bits = np.unpackbits(mask[g * beams + b], bitorder="little")[:vocab]
                may = np.flatnonzero((bits != 0) & (x != -np.inf))
            over = x[may] if case["renormalize"] else x
            if not len(may) or not len(over):
                continue
            top = over.max()
            log_sum = np.log(np.exp(over - top).sum())
            y = x[may]
            if len(y) > wanted:
                edge = np.partition(y, len(y) - wanted)[len(y) - wanted]
                may, y = may[y >= edge], y[y >= edge]
            for i in np.argsort(-y, kind="stable")[:wanted]:
                found.append((-(score + ((y[i] - top) - log_sum)), b, int(may[i]), int(may[i]) == state["end_token"]))
        for n, (s, b, token, done) in enumerate(sorted(found)[:wanted]):
            out[0][g, n], out[1][g, n], out[2][g, n], out[3][g, n] = -s, b, token, done
    return out


def _exact_reorder(state):
    if sum(t.numel() for t in state["tensors"]) > 1 << 26:
        return None
    case = state["case"]
    parents = state["parents"].cpu().numpy()
    rows = np.arange(parents.size).reshape(parents.shape) if state["rows"] is None else state["rows"].cpu().numpy()
    wide = np.int64 if case["dtype"] == "i32" else np.float64
    old = [(t if case["dtype"] == "i32" else t.double()).cpu().numpy().astype(wide) for t in state["tensors"]]
    new = [t.copy() for t in old]
    for g in range(case["groups"]):
        end = case["positions"] if state["lengths"] is None else int(state["lengths"][g])
        for b in range(case["beams"]):
            if not 0 <= parents[g, b] < case["beams"]:
                continue
            to, frm = rows[g, b], rows[g, parents[g, b]]
            for o, n in zip(old, new):
                if case["layout"] == "hpw":
                    n[to, :, :end] = o[frm, :, :end]
                else:
                    n[to, :end] = o[frm, :end]
    return new


def _exact_sequences(state):
    tokens, parents = state["tokens"].cpu().numpy(), state["parents"].cpu().numpy()
    steps, groups, beams = tokens.shape
    lengths = np.full(groups, steps) if state["lengths"] is None else state["lengths"].cpu().numpy()
    out = np.full((groups, beams, steps), -1, np.int32)
    group = np.arange(groups)[:, None]
    at = np.broadcast_to(np.arange(beams), (groups, beams)).copy()
    for t in range(steps - 1, -1, -1):
        live = (t < lengths)[:, None] & (at >= 0)
        place = np.where(live, at, 0)
        out[:, :, t] = np.where(live, tokens[t][group, place], -1)
        link = parents[t][group, place]
        at = np.where(live, np.where((link >= 0) & (link < beams), link, -1), at)
    return out
