"""Argument checks of the KV-cache attention entry points (no GPU)."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p
GOOD, ODD = P(4096), P(4100)


@pytest.fixture(scope="module")
def lib():
    from talechime_b200 import _lib, build

    build.build()
    return _lib.lib()


def _tree(lib, ptr=GOOD, batch=1, n=4, hq=4, hkv=2, d=128, max_t=16, ws=GOOD, size=1 << 30):
    return lib.q8lin_rope_attention_tree(ptr, ptr, ptr, ptr, ptr, ptr, ptr, batch, n, hq, hkv, d, max_t, ws, size, ptr,
                                         None)


def _weights(lib, ptr=GOOD, batch=1, n=4, hq=4, hkv=2, d=128, max_t=16, ws=GOOD, size=1 << 30):
    return lib.q8lin_attention_weights(ptr, ptr, ptr, ptr, batch, n, hq, hkv, d, max_t, ptr, ws, size, ptr, None)


def _blocks(lib, ptr=GOOD, batch=1, n=4, hq=4, hkv=2, d=128, max_t=16, ws=GOOD, size=1 << 30, block=16, topk=2):
    return lib.q8lin_attention_blocks(ptr, ptr, ptr, ptr, ptr, batch, n, hq, hkv, d, max_t, block, topk, ws, size, ptr,
                                      ptr, None)


@pytest.mark.parametrize("fn", [_tree, _weights, _blocks], ids=["tree", "weights", "blocks"])
def test_attention_entry_points_check_arguments_before_touching_cuda(lib, fn):
    assert fn(lib, d=64) == 2
    assert fn(lib, hq=3) == 2
    assert fn(lib, hkv=0) == 2
    assert fn(lib, batch=0) == 2
    assert fn(lib, batch=40000) == 2
    assert fn(lib, n=-1) == 2
    assert fn(lib, n=17) == 2 and b"context limit" in lib.q8lin_last_error()
    assert fn(lib, max_t=0) == 2
    assert fn(lib, ptr=None) == 1
    assert fn(lib, ws=None) == 1
    assert fn(lib, ptr=ODD) == 3
    assert fn(lib, ws=ODD) == 3
    assert fn(lib, size=16) == 8 and b"workspace" in lib.q8lin_last_error()


def test_sizes_of_their_own(lib):
    assert _tree(lib, n=0) == 2
    assert _tree(lib, n=257, max_t=1000) == 2
    assert _weights(lib, n=0) == 0 and _blocks(lib, n=0) == 0  # nothing to do
    for block in (0, 8, 24, 256):
        assert _blocks(lib, block=block) == 2
    assert _blocks(lib, topk=0) == 2
    assert _blocks(lib, block=16, max_t=16 * 16384 + 1) == 2


def test_evict_and_move_check_arguments(lib):
    ev = lambda keep=8, sink=2, recent=2, d=128, max_t=16, w=GOOD, k=GOOD, v=GOOD, idx=GOOD: lib.q8lin_kv_evict(
        w, GOOD, 1, 2, d, max_t, keep, sink, recent, k, v, idx, None, None)
    assert ev(keep=17) == 2 and ev(keep=-1) == 2 and ev(sink=-1) == 2 and ev(recent=-1) == 2
    assert ev(keep=3) == 2 and ev(d=64) == 2 and ev(max_t=0) == 2
    assert ev(w=None) == 1 and ev(idx=None) == 1 and ev(v=None) == 1
    assert ev(k=ODD) == 3
    mv = lambda count=4, heads=1, d=128, k=GOOD, idx=GOOD: lib.q8lin_kv_move_rows(k, GOOD, idx, None, 1, 2, heads, d, 16,
                                                                                count, None)
    assert mv(heads=3) == 2 and mv(count=17) == 2 and mv(count=-1) == 2 and mv(d=64) == 2
    assert mv(k=None) == 1 and mv(idx=None) == 1 and mv(k=ODD) == 3
    assert mv(count=0) == 0
    bk = lambda t=4, block=16, k=GOOD: lib.q8lin_kv_block_keys(k, GOOD, 1, t, 2, 128, 16, block, GOOD, None)
    assert bk(block=20) == 2 and bk(t=17) == 2 and bk(t=-1) == 2 and bk(k=None) == 1 and bk(t=0) == 0


def test_workspace_sizes(lib):
    for f, extra in ((lib.q8lin_attention_tree_workspace_size, ()), (lib.q8lin_attention_blocks_workspace_size, ()),
                     (lib.q8lin_attention_weights_workspace_size, (64,))):
        assert f(0, 4, 4, 2, *extra) == 0 and f(1, 0, 4, 2, *extra) == 0 and f(1, 4, 3, 2, *extra) == 0
        assert f(1, 4, 4, 2, *extra) > 0
    assert lib.q8lin_attention_tree_workspace_size(1, 257, 4, 2) == 0


def test_python_surface_refuses_the_cpu():
    from talechime_b200 import Q8LinError, _lib, attention

    k = torch.zeros((1, 2, 16, 128))
    with pytest.raises(Q8LinError) as e:
        attention.attention_weights(torch.zeros((1, 1, 4, 128)), k, k, torch.zeros(1, dtype=torch.int32),
                                    torch.zeros((1, 2, 16)))
    assert e.value.status == _lib.ERR_DEVICE
