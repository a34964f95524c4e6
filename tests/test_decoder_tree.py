"""Speculative steps and the bounded cache of the decoder: trees verified in one pass against token-by-token decoding and
against the same model in fp32, and eviction against the fp32 model with the evicted positions masked out."""
import pytest
import torch

from _util import to_np
from kuillm_b200.decoder import Decoder, DecoderConfig, TreePlan
from oracle import kuiops_oracle as O


def test_tree_plan():
    t = TreePlan([-1, 0, 0, 1, 3], device="cpu")
    assert t.size == 5 and t.max_depth == 4 and t.depth.tolist() == [0, 1, 1, 2, 3]
    assert t.mask.int().tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0], [1, 1, 0, 1, 1]]
    assert TreePlan.chain(3, device="cpu").parents.tolist() == [-1, 0, 1] and TreePlan.chain(1, device="cpu").max_depth == 1
    for bad in ([], [0], [-1, -1], [-1, 1], [-1, 0, 5]):
        with pytest.raises(ValueError):
            TreePlan(bad, device="cpu")


def _decoder(hd, seed=0, **kw):
    cfg = DecoderConfig.tiny() if hd == 64 else DecoderConfig.tiny(d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, d_ff=1024)
    return Decoder(cfg, device="cuda", seed=seed, init_std=0.05)


def _twin32(dec):
    from test_decoder_gpu import _hf_twin
    return _hf_twin(dec).float()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_logits_equal_the_fp32_model_on_every_path(cuda, hd):
    dec = _decoder(hd)
    twin = _twin32(dec)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 1000, (2, 21), generator=g).cuda()
    plan = TreePlan([-1, 0, 0, 1, 1, 2, 3])
    tokens = torch.randint(0, 1000, (2, plan.size), generator=g).cuda()
    dec.alloc_cache(2, 40)
    dec.prefill(ids)
    path, counts, nxt, logits = dec.verify(tokens, plan, return_logits=True)
    for i in range(plan.size):
        chain, j = [], i
        while j >= 0:
            chain.insert(0, j)
            j = int(plan.parents[j])
        with torch.no_grad():
            want = twin(torch.cat([ids, tokens[:, chain]], 1)).logits[:, -1]
        assert O.max_rel_err(to_np(logits[:, i]), to_np(want)) <= 2e-2, i
    # the walk follows the step's own logits
    target = logits.argmax(-1).cpu()
    want = O.tree_accept(plan.parents[None].cpu().numpy(), tokens.cpu().numpy(), target.numpy())
    assert (path.cpu().numpy() == want[0]).all() and (counts.cpu().numpy() == want[1]).all() and (nxt.cpu().numpy() == want[2]).all()
    assert dec.kv_lens.tolist() == [21 + int(c) for c in counts] == dec.next_pos.tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_accepted_tokens_continue_like_decoding_step_by_step(cuda, hd):
    """Drafts that are the model's own continuation are all accepted; the cache then holds what token-by-token decoding
    leaves, and the next step's logits agree with the fp32 model."""
    dec, ref = _decoder(hd, seed=1), _decoder(hd, seed=1)
    twin = _twin32(dec)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 1000, (3, 17), generator=g).cuda()
    plan = TreePlan.chain(4)
    dec.alloc_cache(3, 40)
    ref.alloc_cache(3, 40)
    first = dec.next_token(dec.prefill(ids))
    ref.prefill(ids)
    tokens = [first]
    for _ in range(3):                                                 # what the tree kernel itself says, one node at a time
        probe = _decoder(hd, seed=1)
        probe.alloc_cache(3, 40)
        probe.prefill(ids)
        tokens.append(probe.verify(torch.stack(tokens, 1), TreePlan.chain(len(tokens)), return_logits=True)[3][:, -1].argmax(-1))
    tokens = torch.stack(tokens, 1)
    path, counts, nxt, logits = dec.verify(tokens, plan, return_logits=True)
    assert (counts == 4).all() and (path == torch.arange(4, device="cuda")).all()
    for t in range(4):
        ref.decode_step(tokens[:, t])
    for a, b in ((dec.k_cache, ref.k_cache), (dec.v_cache, ref.v_cache)):
        assert O.max_rel_err(to_np(a[:, :, :, :21]), to_np(b[:, :, :, :21])) <= 2e-2
    _, _, _, after = dec.verify(nxt[:, None], TreePlan.chain(1), return_logits=True)
    with torch.no_grad():
        want = twin(torch.cat([ids, tokens, nxt[:, None]], 1)).logits[:, -1]
    assert O.max_rel_err(to_np(after[:, 0]), to_np(want)) <= 2e-2
    with pytest.raises(AssertionError):
        dec.decode_step(nxt)


@pytest.mark.gpu
def test_evicted_cache_equals_the_model_with_those_positions_masked(cuda):
    """sinks + recent fill the budget, so every head keeps the same positions: the fp32 model with the others masked out is
    the definition.  Positions go on counting; a second eviction works on slots out of order."""
    dec = _decoder(64, seed=3)
    twin = _twin32(dec)
    g = torch.Generator().manual_seed(4)
    B, S = 2, 30
    ids = torch.randint(0, 1000, (B, S), generator=g).cuda()
    dec.alloc_cache(B, 48, track_mass=True, window=8)
    last = dec.next_token(dec.prefill(ids))
    # the window's rows each spread a weight of one per head
    per = dec.mass.sum(-1)
    assert torch.allclose(per, torch.full_like(per, 8 * dec.hq / dec.hk), rtol=2e-2)
    assert float(dec.mass[:, :, S:].abs().max()) == 0.0
    sees = torch.ones(S, S, dtype=torch.bool).tril()                    # row q of the text sees these positions
    alive, text, one = list(range(S)), ids, TreePlan.chain(1)
    for budget, sinks in ((20, 4), (16, 2)):
        n = text.shape[1]
        src = dec.evict(budget, sinks=sinks, recent=budget - sinks)
        alive = [q for q in alive if q < sinks or q >= n - (budget - sinks)]
        assert len(alive) == budget and dec.kv_lens.tolist() == [budget] * B and dec.next_pos.tolist() == [n] * B
        assert src.shape == (2 * B, dec.hk, budget)
        for row in dec.slot_pos[:, :, :budget].reshape(-1, budget).tolist():
            assert sorted(row) == alive
        for _ in range(3):
            before = dec.mass.sum()
            _, _, nxt, logits = dec.verify(last[:, None], one, return_logits=True)
            rows = B * dec.hq * dec.cfg.n_layers                        # each spreads a weight of one over what it sees
            assert abs(float(dec.mass.sum() - before) - rows) < 2e-2 * rows
            text = torch.cat([text, last[:, None]], 1)
            n = text.shape[1]
            alive = alive + [n - 1]
            sees = torch.nn.functional.pad(sees, (0, 1, 0, 1))
            sees[-1, alive] = True
            mask = torch.where(sees, 0.0, float("-inf")).cuda().expand(B, 1, n, n)
            with torch.no_grad():
                want = twin(text, attention_mask=mask).logits[:, -1]
            assert O.max_rel_err(to_np(logits[:, 0]), to_np(want)) <= 2e-2
            last = nxt


@pytest.mark.gpu
def test_generate_tree_equals_greedy_and_stays_within_its_cache(cuda):
    """Drafts from the greedy continuation and drafts that are noise give the same tokens; with a budget the generation runs
    past the capacity."""
    dec = _decoder(64, seed=5)
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(0, 1000, (2, 12), generator=g).cuda()
    plan = TreePlan([-1, 0, 0, 1])
    noise = lambda last, step: torch.randint(0, 1000, (2, 3), generator=g).cuda()               # noqa: E731
    dec.alloc_cache(2, 64)
    plain = dec.generate_tree(ids, 20, TreePlan.chain(1), None)
    dec.alloc_cache(2, 64)
    drafted = dec.generate_tree(ids, 20, plan, noise)

    def helper(last, step):                                              # the continuation at each sequence's own position
        rows = []
        for b in range(2):
            at = int(dec.next_pos[b]) - 12 if dec.kv_lens is not None else 0
            nxt = plain[b, at + 1:at + 3].tolist() + [0, 0]
            rows.append([nxt[0], 7, nxt[1]])
        return torch.tensor(rows).cuda()
    dec.alloc_cache(2, 64)
    helped = dec.generate_tree(ids, 20, plan, helper)
    assert drafted.shape == helped.shape == plain.shape == (2, 20)
    # greedy tokens agree until, at the earliest, two logits lie within rounding of each other
    for other in (drafted, helped):
        for b in range(2):
            same = int((other[b] == plain[b]).int().cumprod(0).sum())
            if same < 20:
                twin = _twin32(dec)
                with torch.no_grad():
                    top = twin(torch.cat([ids[b:b + 1], plain[b:b + 1, :same]], 1)).logits[0, -1].topk(2).values
                assert float(top[0] - top[1]) <= 2 * 2e-2 * float(top[0].abs().max())
    assert int(dec.next_pos.min()) >= 12 + 19
    dec.alloc_cache(2, 24, track_mass=True, window=8)
    long = dec.generate_tree(ids, 60, plan, noise, budget=16, sinks=2, recent=6)
    assert long.shape == (2, 60) and int(dec.kv_lens.max()) <= 24 and int(dec.next_pos.min()) >= 12 + 59
    with pytest.raises(ValueError):
        dec.alloc_cache(2, 24)
        dec.generate_tree(ids, 60, plan, noise)


@pytest.mark.gpu
def test_paths_that_take_slots_for_positions_are_refused_after_a_tree_step(cuda):
    dec = _decoder(64, seed=8)
    ids = torch.randint(0, 1000, (1, 5), generator=torch.Generator().manual_seed(1)).cuda()
    dec.alloc_cache(1, 16)
    one = TreePlan.chain(1)
    dec.verify(ids[:, :1], one)                                          # a cache may start with a tree step, without a prompt
    for call in (lambda: dec.prefill(ids), lambda: dec.decode_step(ids[:, 0]), lambda: dec.capture_decode(1), lambda: dec.decode_graph(ids[:, 0], 1)):
        with pytest.raises(AssertionError):
            call()
    dec.alloc_cache(1, 16)
    dec.prefill(ids)
    dec.decode_step(ids[:, 0])


@pytest.mark.gpu
def test_a_tree_step_without_a_prompt_equals_a_prompt(cuda):
    dec = _decoder(64, seed=9)
    ids = torch.randint(0, 1000, (2, 5), generator=torch.Generator().manual_seed(2)).cuda()
    dec.alloc_cache(2, 16)
    _, _, _, logits = dec.verify(ids, TreePlan.chain(5), return_logits=True)
    with torch.no_grad():
        want = _twin32(dec)(ids).logits
    assert O.max_rel_err(to_np(logits), to_np(want)) <= 2e-2
