"""Q8Decoder's trees of drafted tokens: what step_tree keeps and what accept_path refuses."""
import pytest
import torch

from talechime_b200.decoder import Q8Decoder, synthetic_weights
from test_decoder_kv_gpu import FLIP_REL_L2, PROMPT, _cfg, _greedy, _rel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = _cfg(max_pos=256)
    return cfg, synthetic_weights(cfg, seed=5)


def test_step_tree_keeps_the_longer_of_two_equal_branches(cuda_device, model):
    cfg, w = model
    plain, dec = (Q8Decoder(cfg, w, device=cuda_device) for _ in range(2))
    for d in (plain, dec):
        d.prefill(PROMPT)
    first = int(plain.token.item())
    want = _greedy(plain, 5)
    got = dec.step_tree([first, want[0], want[0], want[1], want[2]], [-1, 0, 0, 2, 3])
    assert got == want[:4]
    assert int(dec.pos.item()) == len(PROMPT) + 4
    assert got + _greedy(dec, 1) == want
    n = len(PROMPT) + 4
    for li in range(cfg.layers):
        assert _rel(dec.k_cache[li][:, :n], plain.k_cache[li][:, :n]) <= FLIP_REL_L2
