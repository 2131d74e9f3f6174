"""Attention over the decoder's f32 KV caches beyond one causal prompt or one token.

Caches are ``[batch, kv_heads, max_t, 128]`` (``[kv_heads, max_t, 128]`` for one sequence, as
``Q8Decoder`` holds them); ``pos`` int32 ``[batch]`` on the device is the number of rows each
sequence had before the call.

* ``rope_attention_tree`` -- RoPE, append and attention of a tree of drafted tokens;
* ``attention_weights``   -- causal attention that also accumulates every key's softmax weight;
* ``kv_evict``            -- keep a cache's heaviest rows by that accumulator, in place;
* ``kv_move_rows``        -- move chosen rows together in place (a tree's accepted path);
* ``block_keys`` / ``attention_blocks`` -- attention over the blocks of keys that a score
  against the blocks' mean keys selects.

What a row does not see may hold anything; queries and visible keys and values are finite (their
sizes: include/q8lin.h).  Outputs overlap no input.

All arithmetic runs in libq8lin.so on the current stream of the tensors' device; this module
checks arguments, allocates outputs and scratch (from torch's caching allocator, so a captured
graph keeps its own) and passes pointers.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import Q8LinError, check

HEAD_DIM = 128


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> None:
    if t.dtype is dtype and t.device == device and t.is_contiguous():
        return
    if t.dtype != dtype:
        raise Q8LinError(_lib.ERR_INVALID_ARGUMENT, f"{name} dtype {t.dtype} is not {dtype}")
    if not t.is_contiguous():
        raise Q8LinError(_lib.ERR_INVALID_ARGUMENT, f"{name} is not contiguous")
    if t.device != device:
        raise Q8LinError(_lib.ERR_DEVICE, f"{name} on {t.device}, expected {device}")


def _shape(t: torch.Tensor, name: str, *shape: int) -> None:
    if t.shape != shape:
        raise Q8LinError(_lib.ERR_SHAPE, f"{name} is {tuple(t.shape)}, expected {shape}")


def _int32(**sizes: int) -> None:
    """The numbers that the C entry points take as they are fit (ctypes would cut them)."""
    for name, n in sizes.items():
        if not -2 ** 31 <= n < 2 ** 31:
            raise Q8LinError(_lib.ERR_SHAPE, f"{name} {n} does not fit 32 bits")


def _caches(k_cache: torch.Tensor, v_cache: Optional[torch.Tensor]) -> tuple[int, int, int, torch.device]:
    """(batch, kv heads, max_t, device) of a pair of caches."""
    dev = k_cache.device
    if dev.type != "cuda":
        raise Q8LinError(_lib.ERR_DEVICE, "the caches live on a CUDA device; there is no CPU path")
    shape = k_cache.shape
    if len(shape) == 3:
        batch, (hkv, max_t, d) = 1, shape
    elif len(shape) == 4:
        batch, hkv, max_t, d = shape
    else:
        raise Q8LinError(_lib.ERR_SHAPE, f"cache must be [batch, kv_heads, max_t, {HEAD_DIM}], got {tuple(shape)}")
    if d != HEAD_DIM or hkv == 0 or max_t == 0 or batch == 0:
        raise Q8LinError(_lib.ERR_SHAPE, f"cache must be [batch, kv_heads, max_t, {HEAD_DIM}], got {tuple(shape)}")
    _need(k_cache, "k_cache", torch.float32, dev)
    if v_cache is not None:
        _need(v_cache, "v_cache", torch.float32, dev)
        if v_cache.shape != shape:
            raise Q8LinError(_lib.ERR_SHAPE, f"v_cache is {tuple(v_cache.shape)}, k_cache {tuple(shape)}")
    return batch, hkv, max_t, dev


def _queries(q: torch.Tensor, batch: int, hkv: int, dev: torch.device) -> tuple[int, int]:
    """(rows per sequence, query heads) of q [batch, t, heads, 128]."""
    _need(q, "q", torch.float32, dev)
    if q.dim() != 4 or q.shape[0] != batch or q.shape[3] != HEAD_DIM or q.shape[2] == 0 or q.shape[2] % hkv:
        raise Q8LinError(_lib.ERR_SHAPE, f"q must be [{batch}, t, heads, {HEAD_DIM}] with heads a multiple of {hkv}, "
                                         f"got {tuple(q.shape)}")
    return q.shape[1], q.shape[2]


def _out(out: Optional[torch.Tensor], dev: torch.device, *shape: int) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.float32, device=dev)
    _need(out, "out", torch.float32, dev)
    _shape(out, "out", *shape)
    return out


def _scratch(workspace: Optional[torch.Tensor], size: int, dev: torch.device) -> torch.Tensor:
    if workspace is None:
        return torch.empty(size, dtype=torch.uint8, device=dev)
    _need(workspace, "workspace", torch.uint8, dev)
    return workspace


def _call(fn, dev: torch.device, *args) -> None:
    # the raw handle of the current stream: torch.cuda.current_stream builds an object for it, a
    # fifth of a small call's time
    index = dev.index
    if torch.cuda.current_device() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status != _lib.OK:
        check(status)


def rope_attention_tree(qkv: torch.Tensor, parents: torch.Tensor, pos: torch.Tensor, cos: torch.Tensor,
                        sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        out: Optional[torch.Tensor] = None,
                        workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens per sequence (q8lin_rope_attention_tree).

    ``qkv`` [batch, n, (heads + 2 kv_heads) * 128] as the fused projection leaves it; ``parents``
    int32 [batch, n]: node i's parent (a node before it) or -1 for the history.  Node i takes
    cache row pos + i and the RoPE position pos + depth, and sees the history, its ancestors
    and itself.  A node with any other parent, all nodes below it, and nodes past max_t are no
    rows: output 0, nothing appended.  ``cos`` / ``sin`` [>= max_t, 64].  Returns out
    [batch, n, heads, 128]; ``k_cache`` / ``v_cache`` hold the appended rows."""
    batch, hkv, max_t, dev = _caches(k_cache, v_cache)
    _need(qkv, "qkv", torch.float32, dev)
    if qkv.dim() != 3 or qkv.shape[0] != batch or qkv.shape[2] % HEAD_DIM:
        raise Q8LinError(_lib.ERR_SHAPE, f"qkv must be [{batch}, n, (heads + 2 kv_heads) * {HEAD_DIM}], "
                                         f"got {tuple(qkv.shape)}")
    n, hq = qkv.shape[1], qkv.shape[2] // HEAD_DIM - 2 * hkv
    if hq <= 0 or hq % hkv:
        raise Q8LinError(_lib.ERR_SHAPE, f"{hq} query heads over {hkv} kv heads")
    _need(parents, "parents", torch.int32, dev)
    _shape(parents, "parents", batch, n)
    _need(pos, "pos", torch.int32, dev)
    _shape(pos, "pos", batch)
    for name, t in (("cos", cos), ("sin", sin)):
        _need(t, name, torch.float32, dev)
        if t.dim() != 2 or t.shape[0] < max_t or t.shape[1] != HEAD_DIM // 2:
            raise Q8LinError(_lib.ERR_SHAPE, f"{name} must be [>= {max_t}, {HEAD_DIM // 2}], got {tuple(t.shape)}")
    out = _out(out, dev, batch, n, hq, HEAD_DIM)
    L = _lib.lib()
    ws = _scratch(workspace, L.q8lin_attention_tree_workspace_size(batch, n, hq, hkv), dev)
    _call(L.q8lin_rope_attention_tree, dev, qkv.data_ptr(), parents.data_ptr(), pos.data_ptr(), cos.data_ptr(),
          sin.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), batch, n, hq, hkv, HEAD_DIM, max_t, ws.data_ptr(),
          ws.numel(), out.data_ptr())
    return out


def attention_weights(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
                      weight: torch.Tensor, out: Optional[torch.Tensor] = None,
                      workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of rows pos .. pos + t - 1 (q [batch, t, heads, 128], rotated; their keys
    and values already in the caches) that adds every key's softmax weight, summed over the rows
    and the heads of the group, to ``weight`` [batch, kv_heads, max_t] (q8lin_attention_weights).
    Returns out [batch, t, heads, 128]."""
    batch, hkv, max_t, dev = _caches(k_cache, v_cache)
    t, hq = _queries(q, batch, hkv, dev)
    _need(pos, "pos", torch.int32, dev)
    _shape(pos, "pos", batch)
    _weight(weight, "weight", batch, hkv, max_t, dev)
    out = _out(out, dev, batch, t, hq, HEAD_DIM)
    L = _lib.lib()
    ws = _scratch(workspace, L.q8lin_attention_weights_workspace_size(batch, t, hq, hkv, max_t), dev)
    _call(L.q8lin_attention_weights, dev, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), pos.data_ptr(), batch, t,
          hq, hkv, HEAD_DIM, max_t, weight.data_ptr(), ws.data_ptr(), ws.numel(), out.data_ptr())
    return out


def _weight(w: torch.Tensor, name: str, batch: int, hkv: int, max_t: int, dev: torch.device) -> None:
    _need(w, name, torch.float32, dev)
    if w.shape != (batch, hkv, max_t) and not (batch == 1 and w.shape == (hkv, max_t)):
        raise Q8LinError(_lib.ERR_SHAPE, f"{name} is {tuple(w.shape)}, expected {(batch, hkv, max_t)}")


def kv_evict(weight: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, length: torch.Tensor, keep: int,
             sink: int = 0, recent: int = 0, weight_out: Optional[torch.Tensor] = None,
             index: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keep min(length, keep) rows of every head of the caches, in place and in order: rows
    [0, sink), the last ``recent`` of the ``length`` [batch] (int32, device) rows, and the
    heaviest of the others by ``weight`` [batch, kv_heads, max_t] (equal weights: the lower row;
    NaN: lowest).  Rows behind the kept ones stay as they were.  ``weight_out`` (may be
    ``weight``) gets the kept rows' weights and 0 behind them.  Returns the kept rows' former
    places, int32 [batch, kv_heads, keep], -1 behind the last (q8lin_kv_evict)."""
    _int32(keep=keep, sink=sink, recent=recent)
    batch, hkv, max_t, dev = _caches(k_cache, v_cache)
    _weight(weight, "weight", batch, hkv, max_t, dev)
    _need(length, "length", torch.int32, dev)
    _shape(length, "length", batch)
    if weight_out is not None:
        _weight(weight_out, "weight_out", batch, hkv, max_t, dev)
    if not 0 <= keep <= max_t:
        raise Q8LinError(_lib.ERR_SHAPE, f"keep {keep} is not in [0, {max_t}]")
    if index is None:
        index = torch.empty((batch, hkv, keep), dtype=torch.int32, device=dev)
    else:
        _need(index, "index", torch.int32, dev)
        _shape(index, "index", batch, hkv, keep)
    _call(_lib.lib().q8lin_kv_evict, dev, weight.data_ptr(), length.data_ptr(), batch, hkv, HEAD_DIM, max_t, keep, sink,
          recent, k_cache.data_ptr(), v_cache.data_ptr(), index.data_ptr(),
          None if weight_out is None else weight_out.data_ptr())
    return index


def kv_move_rows(k_cache: torch.Tensor, v_cache: torch.Tensor, index: torch.Tensor,
                 base: Optional[torch.Tensor] = None) -> None:
    """Cache row base + i <- row base + index[i] in place, for ascending int32 indices with
    index[i] >= i: ``index`` [batch, count] (every head alike) or [batch, kv_heads, count];
    ``base`` int32 [batch] on the device (None: 0).  Other indices move nothing
    (q8lin_kv_move_rows)."""
    batch, hkv, max_t, dev = _caches(k_cache, v_cache)
    _need(index, "index", torch.int32, dev)
    if index.dim() not in (2, 3) or index.shape[0] != batch or (index.dim() == 3 and index.shape[1] != hkv):
        raise Q8LinError(_lib.ERR_SHAPE, f"index must be [{batch}, count] or [{batch}, {hkv}, count], "
                                         f"got {tuple(index.shape)}")
    if base is not None:
        _need(base, "base", torch.int32, dev)
        _shape(base, "base", batch)
    _call(_lib.lib().q8lin_kv_move_rows, dev, k_cache.data_ptr(), v_cache.data_ptr(), index.data_ptr(),
          None if base is None else base.data_ptr(), batch, hkv, 1 if index.dim() == 2 else hkv, HEAD_DIM, max_t,
          index.shape[-1])


def block_keys(k_cache: torch.Tensor, pos: torch.Tensor, t: int, block: int,
               keys: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Write the mean key of every block of ``block`` rows that rows pos .. pos + t - 1 complete
    into ``keys`` [batch, kv_heads, ceil(max_t / block), 128]; other blocks stay as they were (0
    in a new tensor).  Returns keys (q8lin_kv_block_keys)."""
    _int32(t=t, block=block)
    batch, hkv, max_t, dev = _caches(k_cache, None)
    _need(pos, "pos", torch.int32, dev)
    _shape(pos, "pos", batch)
    if block <= 0:
        raise Q8LinError(_lib.ERR_SHAPE, f"block {block} is not positive")
    shape = (batch, hkv, -(-max_t // block), HEAD_DIM)
    if keys is None:
        keys = torch.zeros(shape, dtype=torch.float32, device=dev)
    else:
        _need(keys, "keys", torch.float32, dev)
        _shape(keys, "keys", *shape)
    _call(_lib.lib().q8lin_kv_block_keys, dev, k_cache.data_ptr(), pos.data_ptr(), batch, t, hkv, HEAD_DIM, max_t, block,
          keys.data_ptr())
    return keys


def attention_blocks(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, keys: torch.Tensor,
                     pos: torch.Tensor, block: int, topk: int, out: Optional[torch.Tensor] = None,
                     index: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of rows pos .. pos + t - 1 (as ``attention_weights``) over chosen blocks: each
    row's own block up to itself and, per kv head, the ``topk`` blocks before it whose mean key
    (``keys``, see ``block_keys``) scores highest against the sum of the group's queries (f64;
    equal scores: the lower block; NaN: lowest).  Returns out [batch, t, heads, 128] and the
    chosen blocks, int32 [batch, t, kv_heads, topk], ascending, -1 behind the last
    (q8lin_attention_blocks)."""
    _int32(block=block, topk=topk)
    batch, hkv, max_t, dev = _caches(k_cache, v_cache)
    t, hq = _queries(q, batch, hkv, dev)
    _need(pos, "pos", torch.int32, dev)
    _shape(pos, "pos", batch)
    if block <= 0 or topk <= 0:
        raise Q8LinError(_lib.ERR_SHAPE, f"block {block} and topk {topk} must be positive")
    _need(keys, "keys", torch.float32, dev)
    _shape(keys, "keys", batch, hkv, -(-max_t // block), HEAD_DIM)
    out = _out(out, dev, batch, t, hq, HEAD_DIM)
    if index is None:
        index = torch.empty((batch, t, hkv, topk), dtype=torch.int32, device=dev)
    else:
        _need(index, "index", torch.int32, dev)
        _shape(index, "index", batch, t, hkv, topk)
    L = _lib.lib()
    ws = _scratch(workspace, L.q8lin_attention_blocks_workspace_size(batch, t, hq, hkv), dev)
    _call(L.q8lin_attention_blocks, dev, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), keys.data_ptr(),
          pos.data_ptr(), batch, t, hq, hkv, HEAD_DIM, max_t, block, topk, ws.data_ptr(), ws.numel(), index.data_ptr(),
          out.data_ptr())
    return out, index
