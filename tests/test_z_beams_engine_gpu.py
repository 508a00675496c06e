"""Beam search on the engine's slots: selection under the slots' masks, reordering of their
states, and a whole search against one run on the host with the oracle's states."""

from __future__ import annotations

import numpy as np
import pytest

from tests import beam_reference as ref
from tests.conftest import case_index, case_options, golden_walks, make_oracle, unpack, world

pytestmark = pytest.mark.gpu


def engine_of(case, slots, **more):
    from xgraph_b200.engine import Engine
    from xgraph_b200.kgversions import build_kg_versions
    from xgraph_b200.syntax import SpanSyntax

    _, served, _ = world(case["world"])
    index = case_index(case)
    versions = None
    if case["versions"]:
        versions = build_kg_versions(index, {k: [tuple(e) for e in v] for k, v in case["versions"].items()})
    return Engine(index, served, SpanSyntax(), slots, versions=versions, **{**case_options(case), **more}), served


def walk_case(name):
    return next(c for c in golden_walks() if c["name"] == name)


def on_gpu(values):
    import torch

    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).cuda()


def begin(engine, sequences, slots):
    engine.reset()
    engine.begin(on_gpu(slots))
    for slot, seq in zip(slots, sequences):
        engine.set_version(slot, seq["version"])
        if seq["anchor"]:
            engine.anchor(slot, seq["anchor"])
        if seq["opened"]:
            engine.open_span(slot)


@pytest.mark.parametrize("name", ["toy_ordinary", "bpe_committed", "crowd_committed"])
def test_reordered_slots_go_on_as_their_parents(name):
    """Slots in any order, groups of four: after a reorder every slot's state and mask are its
    parent's, and fed the parent's tokens it masks as the parent's walk does."""
    case = walk_case(name)
    sequences = case["sequences"][:8]
    engine, served = engine_of(case, 11)
    rng = np.random.default_rng(5)
    slots = rng.permutation(11)[:8]
    begin(engine, sequences, slots)
    steps = len(sequences[0]["tokens"])
    parents = np.array([[1, 0, 0, 3], [3, -1, 1, 9]], dtype=np.int32)
    source = np.array([1, 0, 0, 3, 7, 5, 5, 7])  # whose walk each row follows afterwards
    follows = np.arange(8)
    moves = {steps // 3, 2 * steps // 3}
    tokens = np.zeros(11, dtype=np.int32)
    from tests.conftest import golden_masks

    for step in range(steps):
        if step in moves:
            before = engine.states_host(), engine.memory_host()
            engine.fill_mask()
            masks = engine.mask_host()
            engine.reorder(on_gpu(slots).view(2, 4), on_gpu(parents))
            after = engine.states_host(), engine.memory_host()
            engine.fill_mask()
            for i in range(8):
                to, frm = slots[i], slots[source[i]]
                assert all(after[0][f][to] == before[0][f][frm] for f in before[0]), (step, i)
                assert (after[1][to] == before[1][frm]).all()
                assert (engine.mask_host()[to] == masks[frm]).all()
            for other in set(range(11)) - set(slots.tolist()):
                assert all(after[0][f][other] == before[0][f][other] for f in before[0])
            follows = follows[source]
        engine.fill_mask()
        words = engine.mask_host().view(np.uint32)
        for i, slot in enumerate(slots):
            walk = case["sequences"].index(sequences[follows[i]])
            assert unpack(words[slot], served.vocab_size) == unpack(golden_masks()[f"{name}/{walk}"][step], served.vocab_size)
        for i, slot in enumerate(slots):
            tokens[slot] = sequences[follows[i]]["tokens"][step]
        engine.advance(tokens)
    live = engine.states_host()["phase"][slots]
    assert (live != 3).all() and engine.faults() == 0


def test_reorder_moves_cursors_activity_and_stop_tables():
    """A child takes its parent's history cursor (sync goes on from there), its activity and
    its STOP table."""
    import torch

    from tests.test_stop import stop_cases, stop_world
    from xgraph_b200.engine import Engine

    case = next(c for c in stop_cases() if c["world"] == "toy")
    index, served, syntax = stop_world("toy")
    engine = Engine(index, served, syntax, 3, paths=True, committed_paths=True, stop="residual-goal")
    vocab = served.vocab_size
    walk = max(case["walks"], key=lambda w: len(w["tokens"]))
    n = len(walk["tokens"])
    engine.begin(on_gpu([0]))
    engine.set_stop(0, walk["question"])
    history = torch.zeros((3, n), dtype=torch.int32, device="cuda")
    history[0] = torch.tensor(walk["tokens"], dtype=torch.int32)
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    half = n // 2
    engine.sync(on_gpu([0]), history, zero, zero + half)
    engine.reorder(on_gpu([[2, 0]]), on_gpu([[1, 0]]))  # 2 and 0 exchanged: 0 becomes the inactive one
    history[2, half:] = history[0, half:]
    for k in range(half, n + 1):
        logits = torch.zeros((2, vocab), device="cuda")
        engine.sync_apply(on_gpu([2, 0]), history, zero, zero + k, logits)
        allowed = walk["allowed"][k] if k < n else walk["final_allowed"]
        assert torch.nonzero(~torch.isneginf(logits[0])).flatten().tolist() == allowed, k
        assert not logits[1].any()
    assert engine.faults() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_select_under_the_slots_masks(dtype, renormalize):
    """Equal to a selection under the materialized masks and to the definition, with an
    inactive slot and one in the error phase (any token); the logits are left alone."""
    import torch

    from xgraph_b200.beams import beam_select

    case = walk_case("bpe_committed")
    sequences = case["sequences"][:6]
    engine, served = engine_of(case, 9)
    slots = np.array([[4, 0, 7, 8], [2, 1, 3, 6]])
    begin(engine, sequences, slots.flatten()[[0, 1, 3, 4, 5, 7]])  # 7 and 3 stay inactive
    tokens = np.zeros(9, dtype=np.int32)
    vocab = served.vocab_size
    gen = torch.Generator(device="cuda").manual_seed(3)
    walkers = slots.flatten()[[0, 1, 3, 4, 5, 7]]
    for step in range(0, 30):
        for slot, seq in zip(walkers, sequences):
            tokens[slot] = seq["tokens"][step]
        if step == 20:
            tokens[8] = -1  # not a token: the slot is in the error phase from here on
        engine.advance(tokens)
        if step % 5:
            continue
        logits = (2 * torch.randn((8, vocab + 5), generator=gen, device="cuda")).to(getattr(torch, dtype))
        scores = -torch.rand((2, 4), generator=gen, device="cuda")
        kept = logits.clone()
        got = engine.beam_select(logits, on_gpu(slots), scores, candidates=9, renormalize=renormalize)
        assert torch.equal(logits.view(torch.uint8), kept.view(torch.uint8))
        states = engine.states_host()
        engine.fill_mask()
        mask = engine.mask_host()[slots.flatten()].copy()
        for i, slot in enumerate(slots.flatten()):
            if slot in (3, 7) or states["phase"][slot] == 3:
                mask[i] = -1
        assert (states["phase"][8] == 3) == (step >= 20)
        same = beam_select(logits, scores, mask=on_gpu(mask), vocab=vocab, candidates=9, renormalize=renormalize)
        for a, b in zip(got, same):
            assert torch.equal(a, b)
        want, _ = ref.select(logits.float().cpu().numpy(), scores.cpu().numpy(), 9, vocab=vocab, mask=mask,
                             renormalize=renormalize)
        np.testing.assert_array_equal(got.tokens.cpu().numpy(), want[2])
        np.testing.assert_array_equal(got.beams.cpu().numpy(), want[1])


@pytest.mark.parametrize("name,beams", [("bpe_committed", 4), ("toy_ordinary", 3), ("crowd_committed", 8)])
def test_a_search_equals_one_on_the_host(name, beams):
    """Sync, selection, reordering of slots and of the model's state, and the back-trace, step
    after step, against the same search with the oracle's states; the model is a table of
    logits by the last token and a per-beam state that counts what the beam has written."""
    import torch

    from xgraph_b200.beams import beam_reorder, beam_sequences

    case = walk_case(name)
    groups, steps = 3, 28
    engine, served = engine_of(case, groups * beams + 2)
    vocab = served.vocab_size
    rng = np.random.default_rng(11)
    table = (2.5 * rng.standard_normal((vocab, vocab))).astype(np.float32)
    end_token = int(rng.integers(vocab))
    slots = rng.permutation(groups * beams + 2)[: groups * beams].reshape(groups, beams).astype(np.int32)
    # the host's search
    oracle = make_oracle(case)
    states = [[oracle.opened_state(oracle.initial_state()) for _ in range(beams)] for _ in range(groups)]
    last = np.zeros((groups, beams), dtype=np.int64)
    scores = np.full((groups, beams), -np.inf, dtype=np.float32)
    scores[:, 0] = 0.0
    finished = np.zeros((groups, beams), dtype=bool)
    traces = []
    for _ in range(steps):
        mask = np.zeros((groups * beams, (vocab + 31) // 32 * 32), dtype=bool)
        for g in range(groups):
            for b in range(beams):
                if states[g][b] is None:
                    mask[g * beams + b, :vocab] = True
                else:
                    mask[g * beams + b, sorted(oracle.allowed(states[g][b]))] = True
        words = np.packbits(mask, axis=1, bitorder="little").view(np.int32)
        (value, parent, token, done), gaps = ref.select(
            table[last].reshape(groups * beams, vocab), scores, beams, mask=words, finished=finished,
            end_token=end_token)
        assert (gaps > 1e-11).all()
        traces.append((value.astype(np.float32), parent, token))
        states = [[_next(oracle, states[g], parent[g, b], token[g, b]) for b in range(beams)] for g in range(groups)]
        last, scores, finished = np.where(token < 0, last, token), value.astype(np.float32), done
    # the engine's
    engine.begin(on_gpu(slots.flatten()))
    for slot in slots.flatten():
        engine.open_span(int(slot))
    device_slots = on_gpu(slots)
    places = device_slots.flatten().long()
    logit_table = torch.from_numpy(table).cuda()
    history = torch.zeros((engine.max_sequences, steps), dtype=torch.int32, device="cuda")
    total = torch.zeros(engine.max_sequences, dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(total)
    model = torch.zeros((groups * beams, 2, steps, 8), dtype=torch.bfloat16, device="cuda")
    device_scores = torch.full((groups, beams), -float("inf"), device="cuda")
    device_scores[:, 0] = 0.0
    device_finished = torch.zeros((groups, beams), dtype=torch.bool, device="cuda")
    device_last = torch.zeros((groups, beams), dtype=torch.int64, device="cuda")
    written = torch.zeros((steps, groups, beams), dtype=torch.int32, device="cuda")
    links = torch.zeros_like(written)
    for t in range(steps):
        logits = logit_table[device_last].reshape(groups * beams, vocab)
        engine.sync(places.int(), history, zero, total)
        got = engine.beam_select(logits, device_slots, device_scores, finished=device_finished, end_token=end_token)
        value, parent, token = traces[t]
        np.testing.assert_array_equal(got.beams.cpu().numpy(), parent)
        np.testing.assert_array_equal(got.tokens.cpu().numpy(), token)
        np.testing.assert_allclose(got.scores.cpu().numpy(), value, rtol=2.0**-23, atol=2e-6 * (t + 1))
        engine.reorder(device_slots, got.beams)
        beam_reorder(model, got.beams, lengths=torch.full((groups,), t, dtype=torch.int32, device="cuda"), dim=2)
        model[:, :, t] = (got.tokens.view(-1, 1, 1) % 200).to(torch.bfloat16)
        written[t], links[t] = got.tokens, got.beams
        history[places, t] = got.tokens.flatten()
        total += 1
        device_scores, device_finished = torch.from_numpy(value).cuda(), got.finished
        device_last = torch.where(got.tokens < 0, device_last, got.tokens.long())
    texts = beam_sequences(written, links)
    np.testing.assert_array_equal(texts.cpu().numpy(),
                                  ref.sequences(np.stack([t[2] for t in traces]), np.stack([t[1] for t in traces])))
    live = torch.from_numpy(np.isfinite(traces[-1][0])).cuda()
    assert torch.equal(model[:, 0, :, 0].view(groups, beams, steps)[live], (texts % 200).to(torch.bfloat16)[live])
    assert engine.faults() == 0


def _next(oracle, states, parent, token):
    """The oracle's state after a continuation; None once a beam is empty or a finished one
    goes on with a token that its constraint does not allow (the engine's error phase)."""
    if parent < 0 or states[parent] is None or token not in oracle.allowed(states[parent]):
        return None
    return oracle.advance(states[parent], int(token))


def test_engine_refusals():
    import torch

    case = walk_case("toy_ordinary")
    engine, served = engine_of(case, 4)
    logits = torch.zeros((4, served.vocab_size), device="cuda")
    scores = torch.zeros((2, 2), device="cuda")
    slots = on_gpu([[0, 1], [2, 3]])
    engine.beam_select(logits, slots, scores)
    with pytest.raises(ValueError, match="slots"):
        engine.beam_select(logits, slots.long(), scores)
    with pytest.raises(ValueError, match="slots"):
        engine.beam_select(logits, slots.view(4), scores)
    with pytest.raises(ValueError, match="scores"):
        engine.beam_select(logits, slots, scores.double())
    with pytest.raises(ValueError, match="row per beam"):
        engine.beam_select(logits[:3], slots, scores)
    with pytest.raises(ValueError, match="same shape"):
        engine.reorder(slots, on_gpu([[0, 1]]))
    with pytest.raises(ValueError, match="max_sequences"):
        engine.reorder(on_gpu([[0, 1, 2, 3, 0]]), on_gpu([[0, 1, 2, 3, 4]]))
    with pytest.raises(ValueError, match="beams"):
        engine.reorder(slots, slots.long())
    biased, _ = engine_of(case, 4, escape_bias=-0.5)
    with pytest.raises(ValueError, match="logit policy"):
        biased.beam_select(logits, slots, scores)
