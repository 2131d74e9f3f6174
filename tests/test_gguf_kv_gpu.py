"""Q8Decoder.from_gguf reaches what a decoder made from its weights does: tracked attention and eviction,
block-sparse attention, batches, trees."""
import pytest
import torch

from talechime_b200 import Q8LinError
from talechime_b200.decoder import Q8Decoder, synthetic_weights
from tests.test_decoder_kv_gpu import PROMPT, _cfg
from tests.test_gguf_gpu import _write_decoder

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def file(tmp_path_factory):
    import numpy as np

    cfg = _cfg(max_t=48, max_pos=200)
    w = synthetic_weights(cfg, seed=9)
    factors = np.random.default_rng(3).uniform(1.0, 2.0, cfg.head_dim // 2).astype(np.float32)
    return cfg, w, factors, _write_decoder(tmp_path_factory.mktemp("gguf") / "kv.gguf", cfg, w, factors)


def test_eviction_of_a_decoder_from_a_file(cuda_device, file):
    cfg, w, factors, path = file
    dec = Q8Decoder.from_gguf(path, device=cuda_device, max_t=48, max_pos=200, track_weights=True, blocks=(16, 2))
    ref = Q8Decoder(cfg, w, device=cuda_device, rope_factors=factors, track_weights=True, blocks=(16, 2))
    assert dec.cfg == cfg and dec.cos.shape == (200, 64)
    for d in (dec, ref):
        d.prefill(PROMPT * 4, mode="tracked")
        assert d.evict(20, sink=2, recent=4) == 12
        for mode in ("tracked", "blocks"):
            d.step(mode)
        d.step_tree([int(d.token.item()), 3], [-1, 0])
    assert torch.equal(dec.logits, ref.logits) and torch.equal(dec.tree_logits, ref.tree_logits)
    assert all(torch.equal(a, b) for a, b in zip(dec.kv_weight, ref.kv_weight))
    assert all(torch.equal(a, b) for a, b in zip(dec.block_keys, ref.block_keys))


def test_batch_of_a_decoder_from_a_file(cuda_device, file):
    cfg, w, factors, path = file
    dec = Q8Decoder.from_gguf(path, device=cuda_device, max_t=48, batch=2, track_weights=True)
    dec.prefill([PROMPT, PROMPT[::-1]], mode="tracked")
    assert dec.kv_weight[0].shape == (2, cfg.kv_heads, 48)
    with pytest.raises(Q8LinError):
        dec.evict(4)  # tables for max_t positions alone
    assert Q8Decoder.from_gguf(path, device=cuda_device, max_t=48).kv_weight is None
