"""How the attention kernels over the KV caches share their work out: whole units in turn, an even split
in which a CTA holds the end of one unit and the start of the next, CTAs of a unit's own.  Each case says
which it means, by the rule of csrc/kv_core.cuh told over here, and is held to the float64
definitions and the bound of tests/test_kv_attention_gpu.py."""
import numpy as np
import pytest
import torch

from talechime_b200 import attention
from test_kv_attention_gpu import _blocks_ref, _caches, _close, _gen, _i32, _random_tree, _tables, _tree_ref, _weights_ref

pytestmark = pytest.mark.gpu

GRID = 148


def _rule(chunks, least, cost):
    """"whole", "own" or "even" for units of so many chunks; least: chunks a CTA takes at least, cost:
    chunks that take as long as starting on a unit."""
    units = len(chunks)
    if units >= 2 * GRID:
        return "whole"
    quota = max(-(-sum(chunks) // GRID), least)
    if units < GRID:
        q = max(min(-(-max(chunks) // (GRID // units)), -(-sum(chunks) // (GRID - units))), least)
        if q <= quota + cost:
            return "own"
    return "even"


def _causal_chunks(B, t, group, hkv, pos, max_t):
    """Chunks of every unit of causal or tree rows, and the rule's two costs."""
    rows = t * group
    per = 8 if rows <= 8 else 16 if rows <= 16 else 128
    out = []
    for p in pos:
        for _ in range(hkv):
            for r0 in range(0, rows, per):
                last = (min(r0 + per, rows) - 1) // group
                keys = min(p + last + 1, max_t) if 0 <= p < max_t else 0
                out.append(-(-keys // (64 if per == 128 else 16)))
    return out, (2, 4) if per == 128 else (8, 8)


FORTY = [100, 0, -1, 60, 139, 150, 199, 3, 128, 64] * 4

SHARES = [
    # B, t, hq, hkv, pos, max_t, share
    (40, 60, 16, 2, FORTY, 200, "whole"),                        # 320 units of 128 rows, some past the cache, some without keys
    (20, 60, 16, 2, FORTY[:20], 200, "even"),                    # 160 units of 128 rows
    (25, 20, 16, 4, [1900 - 3 * b for b in range(25)], 1950, "even"),  # 100 units of 80 rows over long histories
    (12, 33, 16, 2, [900 - 70 * b for b in range(12)], 960, "own"),    # 72 units of 128, 128 and 8 rows
    (20, 1, 16, 8, [40 * b for b in range(20)], 800, "even"),    # 160 units of 8 rows
    (20, 1, 96, 8, [40 * b for b in range(20)], 800, "even"),    # 160 units of 16
    (25, 1, 16, 4, [1600 - 5 * b for b in range(25)], 1610, "even"),   # 100 units of 8 over long histories
    (40, 1, 96, 8, [10 * b for b in range(40)], 400, "whole"),   # 320 units of 16
]


@pytest.mark.parametrize("B,t,hq,hkv,pos,max_t,share", SHARES)
def test_weights_in_every_share(cuda_device, B, t, hq, hkv, pos, max_t, share):
    chunks, costs = _causal_chunks(B, t, hq // hkv, hkv, pos, max_t)
    assert _rule(chunks, *costs) == share
    dev = cuda_device
    g = _gen(B + t, dev)
    k, v = _caches(g, B, hkv, max_t, dev, fill=[p + t if p >= 0 else 0 for p in pos])
    q = torch.randn((B, t, hq, 128), generator=g, device=dev) * 1.5
    weight = torch.zeros((B, hkv, max_t), device=dev)
    ref, wref = _weights_ref(q, k, v, pos, weight)
    out = attention.attention_weights(q, k, v, _i32(pos, dev), weight)
    _close(out, ref)
    _close(weight, wref, "weight")


@pytest.mark.parametrize("B,n,hq,hkv,pos,max_t,share", SHARES[:4] + [
    (20, 2, 64, 8, [40 * b for b in range(20)], 800, "even"),    # 160 units of 16 rows
    (20, 1, 16, 8, [40 * b for b in range(20)], 800, "even"),
])
def test_trees_in_every_share(cuda_device, B, n, hq, hkv, pos, max_t, share):
    rows = n * (hq // hkv)
    assert rows <= 16 or B * hkv * -(-rows // 16) * max_t > 10 * GRID * 16  # else the 16-row kernel has it
    chunks, costs = _causal_chunks(B, n, hq // hkv, hkv, pos, max_t)
    assert _rule(chunks, *costs) == share
    dev = cuda_device
    g = _gen(B + n, dev)
    rng = np.random.default_rng(n)
    k, v = _caches(g, B, hkv, max_t, dev, fill=pos)
    qkv = torch.randn((B, n, (hq + 2 * hkv) * 128), generator=g, device=dev)
    parents = _i32([_random_tree(rng, n, 6) for _ in range(B)], dev)
    cos, sin = _tables(max_t, dev)
    ref, kr, vr = _tree_ref(qkv, parents, pos, cos, sin, k, v, hq)
    out = attention.rope_attention_tree(qkv, parents, _i32(pos, dev), cos, sin, k, v)
    _close(out, ref)
    assert torch.equal(torch.nan_to_num(k, 7.0), torch.nan_to_num(kr, 7.0))
    assert torch.equal(torch.nan_to_num(v, 7.0), torch.nan_to_num(vr, 7.0))


@pytest.mark.parametrize("B,t,hq,hkv,pos,max_t,block,topk,share", [
    (1, 20, 16, 8, [400], 500, 16, 6, "even"),        # 160 units of 2 rows
    (2, 10, 96, 8, [700, 300], 800, 32, 4, "even"),   # 160 units of 12
    (1, 9, 16, 8, [400], 500, 16, 6, "own"),
])
def test_blocks_in_every_share(cuda_device, B, t, hq, hkv, pos, max_t, block, topk, share):
    at = [p + i for p in pos for i in range(t) for _ in range(hkv)]
    assert _rule([min(topk, x // block) * (block // 16) + x % block // 16 + 1 for x in at], 8, 8) == share
    dev = cuda_device
    g = _gen(t + block, dev)
    k, v = _caches(g, B, hkv, max_t, dev, fill=[p + t for p in pos])
    q = torch.randn((B, t, hq, 128), generator=g, device=dev) * 1.5
    keys = attention.block_keys(k, _i32([0] * B, dev), max_t, block)
    ref, iref = _blocks_ref(q, k, v, keys, pos, block, topk)
    out, index = attention.attention_blocks(q, k, v, keys, _i32(pos, dev), block, topk)
    assert torch.equal(index.cpu(), iref)
    _close(out, ref)
