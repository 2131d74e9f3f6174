"""Waits that run out in the tensor-core attention kernels: with a limit of 0 a wait that is not over at once
gives up.  Whatever was given up on is NaN, whatever is not NaN is right, the fault word says so, and
the next call with the usual limit is right."""
import ctypes

import pytest
import torch

from talechime_b200 import _lib, attention
from test_kv_attention_gpu import _caches, _close, _gen, _i32, _tables, _tree_ref, _weights_ref

pytestmark = pytest.mark.gpu

SHAPES = [
    # B, t, hq, hkv, pos, max_t
    (2, 40, 16, 2, [600, 300], 700),                            # CTAs of a unit's own, parts merged
    (20, 60, 16, 2, [100, 0, 60, 139, 3] * 4, 200),             # an even split
    (40, 60, 16, 2, [100, 0, -1, 139, 199] * 8, 200),           # whole units in turn
]


class _NoWaiting:
    def __enter__(self):
        self.lib, flags = _lib.lib(), ctypes.c_uint32(0)
        _lib.check(self.lib.q8lin_fault_status(0, ctypes.byref(flags), 1))
        self.old = self.lib.q8lin_wait_limit_ns()
        assert self.lib.q8lin_set_wait_limit_ns(0) == 0
        return self

    def __exit__(self, *_):
        torch.cuda.synchronize()
        self.lib.q8lin_set_wait_limit_ns(self.old)

    def flags(self) -> int:
        flags = ctypes.c_uint32(0)
        _lib.check(self.lib.q8lin_fault_status(0, ctypes.byref(flags), 1))
        return flags.value


def _right_or_nan(got, ref, what):
    _close(torch.where(torch.isnan(got), ref.to(got.dtype), got), ref, what)


@pytest.mark.parametrize("B,t,hq,hkv,pos,max_t", SHAPES)
def test_weights_given_up_on_are_nan(cuda_device, B, t, hq, hkv, pos, max_t):
    dev = cuda_device
    g = _gen(121, dev)
    k, v = _caches(g, B, hkv, max_t, dev)
    q = torch.randn((B, t, hq, 128), generator=g, device=dev)
    zero = torch.zeros((B, hkv, max_t), device=dev)
    ref, wref = _weights_ref(q, k, v, pos, zero)
    for _ in range(5):
        w = zero.clone()
        with _NoWaiting() as limit:
            out = attention.attention_weights(q, k, v, _i32(pos, dev), w)
        gave_up = limit.flags()
        assert gave_up in (0, 32) and (gave_up or not (torch.isnan(out).any() or torch.isnan(w).any()))
        _right_or_nan(out, ref, "out")
        _right_or_nan(w, wref, "weight")
    w = zero.clone()
    _close(attention.attention_weights(q, k, v, _i32(pos, dev), w), ref)
    _close(w, wref, "weight")


@pytest.mark.parametrize("B,n,hq,hkv,pos,max_t", SHAPES)
def test_trees_given_up_on_are_nan(cuda_device, B, n, hq, hkv, pos, max_t):
    dev = cuda_device
    g = _gen(122, dev)
    k, v = _caches(g, B, hkv, max_t, dev)
    qkv = torch.randn((B, n, (hq + 2 * hkv) * 128), generator=g, device=dev)
    parents = _i32([[(i - 1) // 2 if i else -1 for i in range(n)]] * B, dev)
    cos, sin = _tables(max_t, dev)
    ref, _, _ = _tree_ref(qkv, parents, pos, cos, sin, k, v, hq)
    for _ in range(5):
        with _NoWaiting() as limit:
            out = attention.rope_attention_tree(qkv, parents, _i32(pos, dev), cos, sin, k, v)
        gave_up = limit.flags()
        assert gave_up in (0, 32) and (gave_up or not torch.isnan(out).any())
        _right_or_nan(out, ref, "out")
    _close(attention.rope_attention_tree(qkv, parents, _i32(pos, dev), cos, sin, k, v), ref)
