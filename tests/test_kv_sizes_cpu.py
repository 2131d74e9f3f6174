"""Sizes that the KV-cache operators refuse before anything reaches a device (no GPU)."""
import pytest
import torch

from talechime_b200 import Q8LinError, _lib, attention
from talechime_b200.decoder import DecoderConfig, Q8Decoder

K = torch.zeros((1, 2, 64, 128))
POS = torch.zeros(1, dtype=torch.int32)
W = torch.zeros((1, 2, 64))


def _status(fn) -> int:
    with pytest.raises(Q8LinError) as e:
        fn()
    return e.value.status


@pytest.mark.parametrize("big", [2 ** 31, 2 ** 32, 2 ** 32 + 64, -2 ** 31 - 1])
def test_numbers_beyond_32_bits_are_refused(big):
    """They would be cut: 2^32 + 64 rows of a block to 64, for keys that hold one block."""
    q = torch.zeros((1, 1, 4, 128))
    for fn in (lambda: attention.block_keys(K, POS, big, 16), lambda: attention.block_keys(K, POS, 4, big),
               lambda: attention.attention_blocks(q, K, K, K, POS, big, 2),
               lambda: attention.attention_blocks(q, K, K, K, POS, 16, big),
               lambda: attention.kv_evict(W, K, K, POS, big), lambda: attention.kv_evict(W, K, K, POS, 8, sink=big),
               lambda: attention.kv_evict(W, K, K, POS, 8, recent=big)):
        assert _status(fn) == _lib.ERR_SHAPE
    assert _status(lambda: attention.block_keys(K, POS, 4, 16)) == _lib.ERR_DEVICE  # the CPU is what is left to refuse


@pytest.mark.parametrize("blocks,max_t", [((0, 4), 640), ((-16, 4), 640), ((24, 4), 640), ((256, 4), 640), ((64, 0), 640),
                                          ((64, 16385), 640), ((16, 4), 16 * 16384 + 1)])
def test_decoder_refuses_block_sizes_before_it_is_made(blocks, max_t):
    cfg = DecoderConfig(hidden=256, layers=1, heads=4, kv_heads=2, inter=512, vocab=100, max_t=max_t)
    assert _status(lambda: Q8Decoder(cfg, {}, blocks=blocks)) == _lib.ERR_SHAPE
