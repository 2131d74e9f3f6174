"""How the tensor-core kernels of the KV-cache attention are called: replayed from graphs as positions grow,
on two streams at once, again and again, on workspaces of the caller that hold anything."""
import pytest
import torch

from talechime_b200 import _lib, attention
from test_kv_attention_gpu import D, _caches, _gen, _i32, _tables

pytestmark = pytest.mark.gpu

SHAPES = [
    # B, n (tree), t (prompt), hq, hkv, pos, pos of the replays, max_t
    (2, 40, 130, 16, 2, [300, 17], ([400, 9], [130, 1290]), 1500),   # trees over a large cache by the tensor cores, several parts a unit
    (40, 60, 60, 16, 2, [100, 0, 60, 139, 3] * 8, ([20, 90, 130, 1, 64] * 8, [139, 80, 0, 77, 100] * 8), 200),  # whole units in turn
    (20, 60, 60, 16, 2, [100, 0, 60, 139, 3] * 4, ([20, 90, 130, 1, 64] * 4, [139, 80, 0, 77, 100] * 4), 200),  # an even split
]


def _case(dev, shape, seed):
    B, n, t, hq, hkv, pos, _, max_t = shape
    g = _gen(seed, dev)
    k, v = _caches(g, B, hkv, max_t, dev)
    cos, sin = _tables(max_t, dev)
    parents = torch.clamp(torch.arange(n, device=dev) - 1 - torch.randint(0, 5, (B, n), generator=g, device=dev), min=-1)
    return dict(k=k, v=v, cos=cos, sin=sin, qkv=torch.randn((B, n, (hq + 2 * hkv) * D), generator=g, device=dev),
                q=torch.randn((B, t, hq, D), generator=g, device=dev), parents=parents.to(torch.int32), pos=_i32(pos, dev),
                w=torch.zeros((B, hkv, max_t), device=dev))


def _run(c, **kw):
    a = attention.rope_attention_tree(c["qkv"], c["parents"], c["pos"], c["cos"], c["sin"], c["k"], c["v"], **kw.get("tree", {}))
    b = attention.attention_weights(c["q"], c["k"], c["v"], c["pos"], c["w"], **kw.get("weights", {}))
    return a, b


def _same(c, outs, f, want):
    return all(torch.equal(x, y) for x, y in zip(outs, want)) and all(torch.equal(c[n], f[n]) for n in ("k", "v", "w"))


@pytest.mark.parametrize("shape", SHAPES, ids=["parts", "whole", "even"])
def test_graphs_replay_as_positions_grow(cuda_device, shape):
    """Two graphs of the same shape, each with its own workspaces, replayed behind one another at other
    positions and inputs: as the eager calls."""
    dev = cuda_device
    _run(_case(dev, shape, 1))  # kernel attributes before the captures
    graphs = []
    for seed in (2, 3):
        c = _case(dev, shape, seed)
        s, graph = torch.cuda.Stream(dev), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            outs = _run(c)
        graphs.append((graph, c, outs))
    for i, pos in enumerate(shape[6]):
        fresh = [_case(dev, shape, 10 + 2 * i + j) for j in range(2)]
        for (_, c, _), f in zip(graphs, fresh):
            f["pos"].copy_(_i32(pos, dev))
            for name in c:
                c[name].copy_(f[name])
        torch.cuda.synchronize()
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, c, outs), f in zip(graphs, fresh):
            assert _same(c, outs, f, _run(f))
    del graphs


@pytest.mark.parametrize("shape", SHAPES, ids=["parts", "whole", "even"])
def test_two_streams_at_once(cuda_device, shape):
    """Two calls in flight, which share the SMs' tensor memory: each as alone, three times over."""
    dev = cuda_device
    alone = [_case(dev, shape, s) for s in (21, 22)]
    want = [_run(c) for c in alone]
    streams = [torch.cuda.Stream(dev) for _ in alone]
    for _ in range(3):
        cases = [_case(dev, shape, s) for s in (21, 22)]
        torch.cuda.synchronize()
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(_run(c))
        torch.cuda.synchronize()
        for c, o, f, w in zip(cases, got, alone, want):
            assert _same(c, o, f, w)


@pytest.mark.parametrize("shape", SHAPES, ids=["parts", "whole", "even"])
def test_any_workspace_gives_the_same_bits(cuda_device, shape):
    """Workspaces filled with ones, NaN patterns and what the call before left: the same bits as torch's own."""
    dev, L = cuda_device, _lib.lib()
    B, n, t, hq, hkv, _, _, max_t = shape
    first = _case(dev, shape, 31)
    want = _run(first)
    wt = torch.empty(L.q8lin_attention_tree_workspace_size(B, n, hq, hkv), dtype=torch.uint8, device=dev)
    ww = torch.empty(L.q8lin_attention_weights_workspace_size(B, t, hq, hkv, max_t), dtype=torch.uint8, device=dev)
    for fill in (0xab, 0xff, 0x7f, None):
        if fill is not None:
            wt.fill_(fill)
            ww.fill_(fill)
        c = _case(dev, shape, 31)
        assert _same(c, _run(c, tree={"workspace": wt}, weights={"workspace": ww}), first, want)
