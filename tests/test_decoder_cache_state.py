"""What the decoder keeps beside its cache - attention weight, slots in use, the captured step - through every order of calls."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kuillm_b200.kuipy import _ffi
from kuillm_b200.decoder import Decoder, DecoderConfig, TreePlan
from test_decoder_tree import _decoder


@pytest.mark.gpu
def test_a_second_prompt_in_one_cache_starts_without_the_first_ones_weight(cuda):
    g = torch.Generator().manual_seed(1)
    long, short = (torch.randint(0, 1000, (2, n), generator=g).cuda() for n in (30, 9))
    dec, fresh = _decoder(64, seed=2), _decoder(64, seed=2)
    for d in (dec, fresh):
        d.alloc_cache(2, 40, track_mass=True, window=8)
    dec.prefill(long)
    dec.length = 0
    dec.prefill(short)
    fresh.prefill(short)
    assert float(fresh.mass.sum()) > 0 and torch.equal(dec.mass, fresh.mass)


def _cpu_decoder():
    return Decoder(DecoderConfig.tiny(n_layers=1, d_model=64, d_ff=64, vocab=32), device="cpu")


def test_a_captured_step_does_not_outlive_its_cache():
    dec = _cpu_decoder()
    dec.alloc_cache(2, 8)
    dec._graph, dec._tok = object(), torch.zeros(2, dtype=torch.int64)
    dec.alloc_cache(2, 8)
    assert dec._graph is None
    with pytest.raises(ValueError):
        dec.decode_graph(torch.zeros(2, dtype=torch.int64), 1)


@pytest.mark.gpu
def test_captured_generation_in_a_new_cache(cuda):
    g = torch.Generator().manual_seed(3)
    ids, dec = torch.randint(0, 1000, (2, 7), generator=g).cuda(), _decoder(64, seed=4)
    dec.alloc_cache(2, 32)
    want = dec.generate(ids, 6)
    for cap in (32, 24, 40):
        dec.alloc_cache(2, cap)
        assert torch.equal(dec.generate(ids, 6, use_graph=True), want)
        dec.length = 0
        assert torch.equal(dec.generate(ids, 6, use_graph=True), want)           # the same capture again


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_decoded_tokens_give_attention_weight_like_verified_ones(cuda, hd):
    """A token decoded step by step, eagerly or from the captured step, adds what a verified tree of one node adds."""
    g = torch.Generator().manual_seed(5)
    ids, toks = torch.randint(0, 1000, (2, 12), generator=g).cuda(), torch.randint(0, 1000, (2, 4), generator=g).cuda()
    tree, step = _decoder(hd, seed=6), _decoder(hd, seed=6)
    rows = 2 * tree.hq * tree.cfg.n_layers                             # each spreads a weight of one over what it sees
    for d in (tree, step):
        d.alloc_cache(2, 32, track_mass=True, window=4)
        d.prefill(ids)
    assert torch.equal(tree.mass, step.mass)
    for t in range(4):
        before = float(step.mass.sum())
        tree.verify(toks[:, t:t + 1], TreePlan.chain(1))
        step.decode_step(toks[:, t])
        assert abs(float(step.mass.sum()) - before - rows) < 2e-2 * rows
    # both attend in 16 bits: a score is off by about one step of its 16-bit operands (2^-8 of a few units), and so is a weight
    assert (tree.mass - step.mass).abs().max() <= 2.0 ** -4 * float(tree.mass.max())
    assert float(step.mass[:, :, 16:].abs().max()) == 0.0
    # the captured step: its warm-up leaves the weight alone, and every replay adds its tokens'
    before = step.mass.clone()
    step.capture_decode(2)
    assert torch.equal(step.mass, before)
    step.decode_graph(toks[:, 0], 3)
    assert abs(float(step.mass.sum() - before.sum()) - 3 * rows) < 2e-2 * 3 * rows
    assert float(step.mass[:, :, 15 + 4:].abs().max()) == 0.0 and float((step.mass - before).min()) >= 0.0
    step.evict(10, sinks=2, recent=3)
    assert step.kv_lens.tolist() == [10, 10] and step.next_pos.tolist() == [19, 19]
    kept = step.slot_pos[:, :, :10]
    assert bool(((kept >= 3) & (kept < 16)).any())


@pytest.mark.gpu
def test_a_step_that_may_not_fit_is_refused(cuda):
    """The cache may be filled to its last slot; a step that could pass it changes nothing, and an eviction makes room again."""
    dec = _decoder(64, seed=7)
    ids = torch.randint(0, 1000, (2, 9), generator=torch.Generator().manual_seed(8)).cuda()
    tree = TreePlan([-1, 0, 0, 1])                                      # up to three slots
    dec.alloc_cache(2, 16, track_mass=True, window=4)
    last = dec.next_token(dec.prefill(ids))
    wrong = torch.full((2, 3), 1000 - 1, dtype=torch.int64, device="cuda")
    steps = 0
    while int(dec.kv_lens.max()) + 3 <= 16 if dec.kv_lens is not None else True:      # rejected drafts take one slot a step
        _, counts, last = dec.verify(torch.cat([last[:, None], wrong], 1), tree)
        steps += 1
    assert steps >= 2
    state = [t.clone() for t in (dec.kv_lens, dec.next_pos, dec.mass, dec.slot_pos, dec.k_cache)]
    with pytest.raises(ValueError):
        dec.verify(torch.cat([last[:, None], wrong], 1), tree)
    assert all(torch.equal(a, b) for a, b in zip(state, (dec.kv_lens, dec.next_pos, dec.mass, dec.slot_pos, dec.k_cache)))
    while int(dec.kv_lens.max()) < 16:                                  # single nodes go on to the last slot
        _, _, last = dec.verify(last[:, None], TreePlan.chain(1))
    with pytest.raises(ValueError):
        dec.verify(last[:, None], TreePlan.chain(1))
    dec.evict(10, sinks=2, recent=3)
    _, counts, _ = dec.verify(torch.cat([last[:, None], wrong], 1), tree)
    assert dec.kv_lens.tolist() == (10 + counts).tolist() and _ffi.check_status(torch.device("cuda", 0)) == 0


def test_guards_hold_when_python_runs_optimised():
    code = """
import torch
from test_decoder_cache_state import _cpu_decoder
dec = _cpu_decoder()
dec.alloc_cache(1, 8)
dec.kv_lens = torch.zeros(1, dtype=torch.int64)
ids = torch.zeros(1, 1, dtype=torch.int64)
for call in (lambda: dec.prefill(ids), lambda: dec.decode_step(ids[0]), lambda: dec.capture_decode(1), lambda: dec.decode_graph(ids[0], 1)):
    try:
        call()
    except AssertionError as e:
        print("refused:", e)
"""
    tests = Path(__file__).resolve().parent
    env = {**os.environ, "PYTHONPATH": os.pathsep.join(str(p) for p in (tests, tests.parent, tests.parent / "kuillm_b200"))}
    r = subprocess.run([sys.executable, "-O", "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.stdout.count("refused:") == 4, r.stdout + r.stderr


@pytest.mark.gpu
def test_a_window_of_no_prompt_rows(cuda):
    """Without a window the prompt gives no weight, the tokens after it do."""
    dec = _decoder(64, seed=9)
    ids = torch.randint(0, 1000, (2, 9), generator=torch.Generator().manual_seed(8)).cuda()
    dec.alloc_cache(2, 16, track_mass=True, window=0)
    last = dec.next_token(dec.prefill(ids))
    assert float(dec.mass.abs().max()) == 0.0
    dec.decode_step(last)
    rows = 2 * dec.hq * dec.cfg.n_layers
    assert abs(float(dec.mass.sum()) - rows) < 2e-2 * rows
    with pytest.raises(ValueError):
        dec.alloc_cache(2, 16, track_mass=True, window=-1)


@pytest.mark.gpu
def test_right_drafts_take_fewer_steps(cuda):
    """Drafts that are the model's own continuation are accepted: a generation with them takes a fraction of the steps."""
    dec = _decoder(64, seed=5)
    ids = torch.randint(0, 1000, (1, 12), generator=torch.Generator().manual_seed(6)).cuda()
    plan, steps = TreePlan([-1, 0, 0, 1]), [0, 0]
    dec.alloc_cache(1, 64)

    def nothing(last, step):
        steps[0] += 1
        return torch.full((1, 3), 1001 - 2, dtype=torch.int64, device="cuda")
    plain = dec.generate_tree(ids, 24, plan, nothing)

    def helper(last, step):
        steps[1] += 1
        at = int(dec.next_pos[0]) - 12 if dec.kv_lens is not None else 0
        nxt = plain[0, at + 1:at + 3].tolist() + [0, 0]
        return torch.tensor([[nxt[0], 7, nxt[1]]], device="cuda")
    dec.alloc_cache(1, 64)
    helped = dec.generate_tree(ids, 24, plan, helper)
    # the same rows in the same tree positions give the same logits, so nothing but the drafts differs
    assert torch.equal(helped[0, :3], plain[0, :3])
    same = int((helped[0] == plain[0]).int().cumprod(0).sum())
    assert steps[0] >= 20 and steps[1] <= 8 + (24 - same), (steps, same)


@pytest.mark.gpu
def test_generation_with_uneven_drafts_fits_the_tokens_asked_for(cuda):
    """One sequence's drafts are right and the other's are noise, in turns: neither what the two take together nor what the faster one
    takes after its last token counts as slots in use."""
    dec = _decoder(64, seed=5)
    g = torch.Generator().manual_seed(6)
    ids, plan, new = torch.randint(0, 1000, (2, 12), generator=g).cuda(), TreePlan.chain(3), 30
    dec.alloc_cache(2, 64)
    plain = dec.generate_tree(ids, new, TreePlan.chain(1), None)
    enough = 12 + new - 1 + plan.max_depth
    for helped in (lambda b, step: b == 0, lambda b, step: b == step % 2):
        def propose(last, step):
            rows = []
            for b in range(2):
                at = int(dec.next_pos[b]) - 12 if dec.kv_lens is not None else 0
                rows.append((plain[b, at + 1:at + 3].tolist() + [0, 0])[:2] if helped(b, step) else [999, 999])
            return torch.tensor(rows, device="cuda")
        dec.alloc_cache(2, enough)
        got = dec.generate_tree(ids, new, plan, propose)
        assert got.shape == (2, new) and dec.kv_lens.tolist() == dec.next_pos.tolist() == [12 + new - 1] * 2
        assert torch.equal(got[:, :4], plain[:, :4])
