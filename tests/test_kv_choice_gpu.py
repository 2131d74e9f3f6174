"""The choice of blocks in its three forms (a CTA a token, a cluster of CTAs a token, eight tokens a CTA) and
lists longer than the attention kernel holds in shared memory, against the float64 definition."""
import math

import pytest
import torch

from talechime_b200 import attention
from test_kv_attention_gpu import _blocks_ref, _caches, _close, _gen, _i32

pytestmark = pytest.mark.gpu


def _form(batch, t, hkv, blocks):
    """CTAs a token, or "eight" tokens a CTA, by the rule of launch_kv_pick."""
    rows = batch * t * hkv
    if t >= 8 and rows // 8 >= 74 and blocks * 64 <= 128 * 1024:
        return "eight"
    ranks = 1
    while ranks < 8 and rows * ranks * 2 <= 296 and blocks >= 128 * ranks:
        ranks *= 2
    return ranks


CASES = [
    # B, t, hq, hkv, pos, max_t, block, topk, form
    (1, 1, 4, 2, [16 * 129 + 3], 16 * 130, 16, 7, 2),
    (2, 1, 8, 1, [64 * 299, 64 * 130 + 63], 64 * 300, 64, 16, 4),
    (1, 3, 4, 2, [16 * 1099 + 5], 16 * 1100, 16, 33, 8),
    (1, 1, 2, 1, [16 * 1100 - 1], 16 * 1100, 16, 1, 8),
    (1, 2, 4, 4, [40], 16 * 600, 16, 5, 8),            # a cluster of eight for three blocks
    (1, 1, 4, 2, [16 * 130 - 16], 16 * 130, 16, 200, 2),  # topk beyond the blocks
    (2, 75, 8, 4, [3, 350], 400, 16, 6, "eight"),      # a last list of three tokens; rows past the cache
    (1, 150, 8, 4, [0], 200, 16, 3, "eight"),          # fewer blocks than topk in front
    (3, 100, 2, 2, [1000, -1, 16 * 70 + 1], 1300, 16, 40, "eight"),
    (1, 1, 2, 1, [16 * 699 + 2], 16 * 700, 16, 600, 8),   # lists beyond 512: parts of one
    (1, 40, 8, 8, [16 * 690], 16 * 700, 16, 600, 1),      # whole ones
]


@pytest.mark.parametrize("B,t,hq,hkv,pos,max_t,block,topk,form", CASES)
def test_choice_matches_its_definition(cuda_device, B, t, hq, hkv, pos, max_t, block, topk, form):
    blocks = -(-max_t // block)
    assert _form(B, t, hkv, blocks) == form
    dev = cuda_device
    g = _gen(t + topk, dev)
    k, v = _caches(g, B, hkv, max_t, dev, fill=[p + t if p >= 0 else 0 for p in pos])
    q = torch.randn((B, t, hq, 128), generator=g, device=dev)
    keys = attention.block_keys(k, _i32([0 if p >= 0 else -1 for p in pos], dev), max_t, block)
    # equal blocks, near and far apart, and blocks whose key is not a number
    for c in range(2, blocks - 1, 9):
        keys[:, :, c] = keys[:, :, c // 2]
    keys[:, :, 5::37] = math.nan
    ref, iref = _blocks_ref(q, k, v, keys, pos, block, topk)
    out, index = attention.attention_blocks(q, k, v, keys, _i32(pos, dev), block, topk)
    assert torch.equal(index.cpu(), iref)
    _close(out, ref)
