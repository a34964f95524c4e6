"""What the decoder keeps beside its cache - attention weight, slots in use, the captured step - through every order of calls."""
import pytest
import torch

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
