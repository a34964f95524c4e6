"""What the decoder keeps beside its cache - attention weight, slots in use, the captured step - through every order of calls."""
import pytest
import torch

from kuillm_b200.decoder import Decoder, DecoderConfig
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
