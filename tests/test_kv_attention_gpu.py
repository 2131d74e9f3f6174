"""Tree attention, attention with accumulated weights, eviction, row moves and block-sparse
attention over the f32 KV caches (csrc/kv_attention.cu, csrc/kv_cache.cu) against their
definitions in 64 bits.

Tolerance of the attention outputs.  A score is a sum of 128 products; each product is off by
at most 2^-20 of itself (tf32 pairs) and the f32 sum by at most 128 * 2^-24 = 2^-17 of the sum
of the products' sizes, which for unit normal q and k is about 128 * 0.64 / sqrt(128) = 7.2 after
scaling: under 6.2e-5 if every error pointed the same way, about 1/sqrt(128) of that, 5e-6, as
they fall.  exp2 and the weighted sums add a few 2^-23.  So outputs are held to a relative L2
error of 1e-5 (the bar of the library's f32 outputs) and a largest error of 6.2e-5 * 2 of the
largest value; weights (sums of probabilities) likewise.
"""
import math

import numpy as np
import pytest
import torch

from talechime_b200 import Q8LinError, _lib, attention

pytestmark = pytest.mark.gpu

D = 128
SCALE = float(np.float32(1.0 / math.sqrt(D)))
REL_L2 = 1e-5
MAX_FRAC = 1.3e-4


def _close(got, ref, what="out"):
    got, ref = got.double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all(), what
    err = (got - ref).norm() / max(float(ref.norm()), 1e-30)
    assert err <= REL_L2, f"{what}: relative L2 {err:.2e}"
    top = float(ref.abs().max()) if ref.numel() else 0.0
    assert float((got - ref).abs().max()) <= MAX_FRAC * top + 1e-30, what


def _caches(rng, B, hkv, max_t, dev, fill=None):
    k = torch.randn((B, hkv, max_t, D), generator=rng, device=dev)
    v = torch.randn((B, hkv, max_t, D), generator=rng, device=dev)
    if fill is not None:  # rows past a sequence's length
        for b, n in enumerate(fill):
            k[b, :, max(n, 0):] = math.nan
            v[b, :, max(n, 0):] = math.nan
    return k, v


def _gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _tables(rows, dev):
    freq = (10000.0 ** (-2.0 * np.arange(64) / D)).astype(np.float32)
    ang = (np.arange(rows, dtype=np.float32)[:, None] * freq).astype(np.float32)
    return torch.from_numpy(np.cos(ang)).to(dev), torch.from_numpy(np.sin(ang)).to(dev)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _softmax_rows(q, k, v, seen):
    """f64 attention of one head, rows that see nothing 0.  q [R, D], k / v [L, D], seen [R, L]."""
    s = (q.double() @ torch.nan_to_num(k.double()).T) * SCALE
    s = s.masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1))
    return p @ torch.nan_to_num(v.double()), p


def _rotate(x, c, s):
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat([lo * c + hi * (-s), hi * c + lo * s], -1)


# ---- trees -------------------------------------------------------------------------------

def _paths(parents, pos, max_t):
    """Node -> its path from the root, or None for what is no row."""
    out = []
    for i, p in enumerate(parents):
        if p == -1:
            path = [i]
        elif 0 <= p < i and out[p] is not None:
            path = out[p] + [i]
        else:
            path = None
        out.append(path if pos >= 0 and pos + i < max_t else None)
    return out


def _tree_ref(qkv, parents, pos, cos, sin, k, v, hq):
    B, n = parents.shape
    hkv, max_t = k.shape[1], k.shape[2]
    k, v = k.clone(), v.clone()
    out = torch.zeros((B, n, hq, D), dtype=torch.float64, device=k.device)
    for b in range(B):
        p0 = int(pos[b])
        paths = _paths(parents[b].tolist(), p0, max_t)
        x = qkv[b].view(n, hq + 2 * hkv, D)
        rows = [i for i in range(n) if paths[i] is not None]
        if not rows:
            continue
        at = torch.tensor([p0 + len(paths[i]) - 1 for i in rows], device=k.device)
        rot = _rotate(x[rows][:, :hq + hkv], cos[at][:, None], sin[at][:, None])
        where = torch.tensor([p0 + i for i in rows], device=k.device)
        k[b][:, where] = rot[:, hq:].transpose(0, 1)
        v[b][:, where] = x[rows][:, hq + hkv:].transpose(0, 1)
        L = min(p0 + n, max_t)
        seen = torch.zeros((len(rows), L), dtype=torch.bool, device=k.device)
        seen[:, :p0] = True
        for r, i in enumerate(rows):
            seen[r, [p0 + a for a in paths[i]]] = True
        for h in range(hq):
            o, _ = _softmax_rows(rot[:, h], k[b, h // (hq // hkv), :L], v[b, h // (hq // hkv), :L], seen)
            out[b, rows, h] = o
    return out, k, v


def _random_tree(rng, n, width):
    return [int(rng.integers(max(-1, i - width), i)) if i else -1 for i in range(n)]


TREES = [
    # B, n, hq, hkv, pos, max_t, kind
    (1, 1, 2, 2, [0], 1, "random"),               # one token, an empty history, a cache of one row
    (1, 1, 16, 2, [77], 100, "random"),           # the single-token form
    (2, 5, 16, 2, [0, 3], 16, "random"),          # fewer keys than a chunk
    (1, 8, 16, 2, [200], 640, "random"),
    (3, 33, 16, 2, [100, 31, 250], 300, "random"),  # ragged, odd sizes
    (1, 16, 16, 16, [500], 517, "random"),        # no grouping, the cache one row short of full
    (2, 7, 12, 4, [64, 16], 80, "random"),        # a group of 3: rows of a unit cross tokens
    (1, 3, 40, 1, [130], 140, "random"),          # a group of 40: a token's heads cross units
    (1, 256, 4, 2, [300], 600, "chain"),          # the longest path
    (1, 256, 8, 8, [10], 300, "star"),            # all siblings
    (8, 64, 16, 2, [900, 800, 1, 0, 64, 63, 65, 900], 1000, "random"),  # many units
    (4, 20, 8, 8, [90, 85, 100, -1], 100, "random"),  # nodes past the cache; no sequence
    (20, 16, 16, 2, [50, 0, -1, 54, 60, 69, 70, 3, 16, 15] * 2, 70, "random"),  # 320 units of 16 rows in a small cache
    (20, 2, 16, 16, [50, 0, -1, 54, 60, 69, 70, 3, 16, 15] * 2, 70, "random"),  # 320 units of 8
]


@pytest.mark.parametrize("B,n,hq,hkv,pos,max_t,kind", TREES)
def test_tree_matches_its_definition(cuda_device, B, n, hq, hkv, pos, max_t, kind):
    """Outputs against float64; appended rows bit-exact (each product rounded, then added);
    every other cache row, NaN behind the histories, as it was."""
    dev = cuda_device
    g = _gen(B * 100 + n, dev)
    rng = np.random.default_rng(n)
    k, v = _caches(g, B, hkv, max_t, dev, fill=pos)
    qkv = torch.randn((B, n, (hq + 2 * hkv) * D), generator=g, device=dev)
    tree = {"random": lambda: _random_tree(rng, n, 6), "chain": lambda: list(range(-1, n - 1)),
            "star": lambda: [-1] * n}[kind]
    parents = _i32([tree() for _ in range(B)], dev)
    cos, sin = _tables(max_t, dev)
    ref, kr, vr = _tree_ref(qkv, parents, pos, cos, sin, k, v, hq)
    out = attention.rope_attention_tree(qkv, parents, _i32(pos, dev), cos, sin, k, v)
    _close(out, ref)
    assert torch.equal(torch.nan_to_num(k, 7.0), torch.nan_to_num(kr, 7.0))
    assert torch.equal(torch.nan_to_num(v, 7.0), torch.nan_to_num(vr, 7.0))


ROOMY = 24000  # rows of a cache in which more than 16 rows a kv head take the tcgen05 kernel whatever their number


@pytest.mark.parametrize("B,n,hq,hkv,pos,max_t,kind", [(*c[:5], ROOMY, c[6]) for c in TREES if c[1] * c[2] // c[3] > 16] + [
    (1, 3, 16, 2, [40], ROOMY, "random"),
    (2, 20, 8, 1, [ROOMY - 10, ROOMY - 20], ROOMY, "chain"),  # nodes past the cache; exactly full
])
def test_tree_in_a_roomy_cache(cuda_device, B, n, hq, hkv, pos, max_t, kind):
    test_tree_matches_its_definition(cuda_device, B, n, hq, hkv, pos, max_t, kind)


def test_tree_nodes_without_a_path_are_no_rows(cuda_device):
    """A parent that is the node itself, behind it or below -1, and everything under such a
    node: output 0, no cache row, seen by nobody; the other nodes as without them."""
    dev, n, hq, hkv, max_t = cuda_device, 9, 4, 2, 40
    g = _gen(5, dev)
    parents = _i32([[-1, 0, 2, 2, 1, 7, -2, 4, 5], [-1, -5, 100, 0, 3, 1, 4, 6, 7]], dev)
    pos = [20, 11]
    k, v = _caches(g, 2, hkv, max_t, dev, fill=pos)
    qkv = torch.randn((2, n, (hq + 2 * hkv) * D), generator=g, device=dev)
    cos, sin = _tables(max_t, dev)
    ref, kr, vr = _tree_ref(qkv, parents, pos, cos, sin, k, v, hq)
    out = attention.rope_attention_tree(qkv, parents, _i32(pos, dev), cos, sin, k, v)
    _close(out, ref)
    for b, dead in enumerate(([2, 3, 5, 6, 8], [1, 2, 5])):
        assert torch.count_nonzero(out[b, dead]) == 0
    assert torch.equal(torch.nan_to_num(k, 7.0), torch.nan_to_num(kr, 7.0))
    assert torch.equal(torch.nan_to_num(v, 7.0), torch.nan_to_num(vr, 7.0))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n,hq,hkv,max_t", [(12, 4, 2, 100), (40, 16, 2, 100), (40, 16, 2, ROOMY)])
def test_tree_siblings_do_not_meet(cuda_device, bad, n, hq, hkv, max_t):
    """A node whose value row is not finite spoils itself and what is below it, nothing else."""
    dev = cuda_device
    g = _gen(6, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    qkv = torch.randn((1, n, (hq + 2 * hkv) * D), generator=g, device=dev)
    parents = [-1, 0, 0, 1, 1, 2, 2] + [1 + (i % 2) for i in range(7, n)]
    cos, sin = _tables(max_t, dev)
    clean = attention.rope_attention_tree(qkv, _i32([parents], dev), _i32([50], dev), cos, sin, k.clone(), v.clone())
    qkv.view(1, n, -1, D)[0, 2, hq + hkv:, 5] = bad  # node 2's value row
    out = attention.rope_attention_tree(qkv, _i32([parents], dev), _i32([50], dev), cos, sin, k, v)
    paths = _paths(parents, 50, max_t)
    spoiled = [i for i in range(n) if 2 in paths[i]]
    free = [i for i in range(n) if 2 not in paths[i]]
    assert not torch.isfinite(out[0, spoiled][..., 5]).any()
    _close(out[0, free], clean[0, free].double())


def test_tree_equals_steps_along_its_paths(cuda_device):
    """A path of the tree gives what the same tokens give one after another."""
    dev, hq, hkv, max_t, p0 = cuda_device, 8, 2, 64, 21
    g = _gen(7, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    parents = [-1, 0, 0, 2, 1, 3]
    qkv = torch.randn((1, 6, (hq + 2 * hkv) * D), generator=g, device=dev)
    cos, sin = _tables(max_t, dev)
    k2, v2 = k.clone(), v.clone()
    out = attention.rope_attention_tree(qkv, _i32([parents], dev), _i32([p0], dev), cos, sin, k, v)
    path = [0, 2, 3, 5]
    for d, i in enumerate(path):
        one = attention.rope_attention_tree(qkv[:, i:i + 1].contiguous(), _i32([[-1]], dev), _i32([p0 + d], dev), cos,
                                            sin, k2, v2)
        _close(out[0, i], one[0, 0].double())
    attention.kv_move_rows(k, v, _i32([path], dev), base=_i32([p0], dev))
    n = p0 + len(path)
    assert torch.equal(k[:, :, :n], k2[:, :, :n]) and torch.equal(v[:, :, :n], v2[:, :, :n])


# ---- accumulated weights -------------------------------------------------------------------

def _weights_ref(q, k, v, pos, weight):
    B, t, hq, _ = q.shape
    hkv, max_t = k.shape[1], k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    w = weight.double().clone()
    for b in range(B):
        p0 = int(pos[b])
        rows = [i for i in range(t) if p0 >= 0 and p0 + i < max_t]
        if not rows:
            continue
        L = min(p0 + t, max_t)
        seen = torch.arange(L, device=q.device) <= (p0 + torch.tensor(rows, device=q.device))[:, None]
        for h in range(hq):
            kh = h // (hq // hkv)
            out[b, rows, h], p = _softmax_rows(q[b, rows, h], k[b, kh, :L], v[b, kh, :L], seen)
            w[b, kh, :L] += p.sum(0)
    return out, w


WEIGHTS = [
    # B, t, hq, hkv, pos, max_t
    (1, 1, 2, 2, [0], 1),                 # one key
    (1, 1, 16, 2, [500], 640),            # the decode form
    (3, 1, 16, 16, [15, 16, 17], 40),     # around a chunk's end
    (2, 1, 32, 1, [99, 40], 130),         # a group of 32: more rows than a unit holds
    (2, 2, 16, 2, [1030, 5], 1100),       # two tokens whose scores are stored, two key ranges
    (1, 16, 4, 4, [0], 16),
    (2, 3, 12, 4, [50, 0], 60),           # a group of 3
    (1, 100, 16, 2, [0], 100),            # a prompt; the cache exactly full
    (2, 65, 8, 8, [37, 0], 120),          # a later chunk, ragged
    (1, 130, 16, 2, [300], 512),
    (2, 40, 4, 2, [90, -1], 100),         # rows past the cache; no sequence
    (40, 1, 16, 16, list(range(0, 400, 10)), 500),  # more units than a split serves
]


@pytest.mark.parametrize("B,t,hq,hkv,pos,max_t", WEIGHTS)
def test_weights_match_their_definition(cuda_device, B, t, hq, hkv, pos, max_t):
    dev = cuda_device
    g = _gen(t * 10 + B, dev)
    k, v = _caches(g, B, hkv, max_t, dev, fill=[p + t if p >= 0 else 0 for p in pos])
    q = torch.randn((B, t, hq, D), generator=g, device=dev) * 1.5
    weight = torch.rand((B, hkv, max_t), generator=g, device=dev) * 0.01
    ref, wref = _weights_ref(q, k, v, pos, weight)
    before = weight.clone()
    out = attention.attention_weights(q, k, v, _i32(pos, dev), weight)
    _close(out, ref)
    _close(weight - before, wref - before.double(), "weight")
    for b, p in enumerate(pos):  # keys behind the last row keep their weight
        end = min(p + t, max_t) if p >= 0 else 0
        assert torch.equal(weight[b, :, end:], before[b, :, end:])


def test_weights_of_rows_past_the_cache_do_not_count(cuda_device):
    """Queries of rows past max_t may hold anything: no NaN of theirs reaches a weight."""
    dev = cuda_device
    g = _gen(9, dev)
    for t, hq, hkv in ((2, 4, 2), (20, 16, 2)):
        k, v = _caches(g, 1, hkv, 32, dev)
        q = torch.randn((1, t, hq, D), generator=g, device=dev)
        q[:, 1:] = math.nan
        w = torch.zeros((1, hkv, 32), device=dev)
        out = attention.attention_weights(q, k, v, _i32([31], dev), w)
        assert torch.isfinite(out[:, :1]).all() and torch.count_nonzero(out[:, 1:]) == 0
        torch.testing.assert_close(w.sum(-1), torch.full((1, hkv), float(hq // hkv), device=dev), rtol=1e-5, atol=0)


@pytest.mark.parametrize("t", [3, 50])
def test_weights_masked_values_that_are_not_finite(cuda_device, t):
    """A later row's key and value that are not finite do not reach the rows before it."""
    dev, hq, hkv, max_t, p0 = cuda_device, 4, 2, 100, 20
    g = _gen(10, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    q = torch.randn((1, t, hq, D), generator=g, device=dev)
    ref, _ = _weights_ref(q, k, v, [p0], torch.zeros((1, hkv, max_t), device=dev))
    k[0, :, p0 + t - 1, 3] = math.nan
    v[0, :, p0 + t - 1, 7] = math.inf
    out = attention.attention_weights(q, k, v, _i32([p0], dev), torch.zeros((1, hkv, max_t), device=dev))
    _close(out[:, :t - 1], ref[:, :t - 1])


def test_weights_large_and_small_numbers(cuda_device):
    """Queries and keys of very different sizes whose scores are ordinary, and a score range
    that leaves all but one key without weight."""
    dev, hq, hkv, L = cuda_device, 4, 2, 70
    g = _gen(11, dev)
    k, v = _caches(g, 1, hkv, L, dev)
    q = torch.randn((1, 1, hq, D), generator=g, device=dev)
    for qs, ks, vs in ((1e-18, 1e18, 1e30), (1e12, 1e-12, 1e-30), (30.0, 3.0, 1.0)):
        q1, k1, v1 = q * qs, k * ks, v * vs
        ref, wref = _weights_ref(q1, k1, v1, [L - 1], torch.zeros((1, hkv, L), device=dev))
        w = torch.zeros((1, hkv, L), device=dev)
        out = attention.attention_weights(q1, k1, v1, _i32([L - 1], dev), w)
        # (30, 3): scores up to 90 times larger, so their error is too
        tol = 90 * REL_L2 if qs == 30.0 else REL_L2
        assert float((out.double() - ref).norm() / ref.norm()) <= tol
        assert float((w.double() - wref).norm() / wref.norm()) <= tol


@pytest.mark.parametrize("t", [1, 40])
def test_weights_values_of_very_different_sizes(cuda_device, t):
    """Keys and values whose sizes differ by 2^40 from one stretch of the cache to the next: each
    output against float64 within the error its largest value allows, which rows that see only
    the small values show at their own size."""
    dev, hq, hkv, max_t, p0 = cuda_device, 16, 2, 400, 200
    g = _gen(12, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    size = torch.ones(max_t, device=dev)
    size[:64], size[64:72], size[100:130], size[215:] = 2.0 ** -20, 2.0 ** 20, 2.0 ** -10, 2.0 ** 25
    v *= size[:, None]
    k *= size.clamp(max=1.0)[:, None]
    q = torch.randn((1, t, hq, D), generator=g, device=dev)
    k[0, :, 64:72] = -100 * q[0, 0].view(hkv, 8, D).sum(1, keepdim=True)  # unseen in effect by token 0
    ref, wref = _weights_ref(q, k, v, [p0], torch.zeros((1, hkv, max_t), device=dev))
    w = torch.zeros((1, hkv, max_t), device=dev)
    out = attention.attention_weights(q, k, v, _i32([p0], dev), w)
    for i in range(t):
        err, top = float((out[0, i].double() - ref[0, i]).norm()), float(ref[0, i].norm())
        assert err <= 10 * REL_L2 * top, (i, err / top)  # scores up to 100 * |q|^2: their f32 rounding
    assert float((w.double() - wref).norm() / wref.norm()) <= 10 * REL_L2


@pytest.mark.parametrize("n,hq,hkv,max_t", [(12, 4, 2, 200), (40, 16, 2, 200), (40, 16, 2, ROOMY)])
def test_tree_finite_part_of_a_value_row_counts(cuda_device, n, hq, hkv, max_t):
    """A history value with one infinite dimension spoils that dimension of the rows that see it
    and counts as it is in the others."""
    dev, p0 = cuda_device, 100
    g = _gen(14, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    v[0, :, 97, 9] = math.inf  # in the last tile, before the tree
    v[0, :, 97, 10:] *= 50.0
    v[0, :, 20, 9] = -math.inf  # in a tile without a mask
    qkv = torch.randn((1, n, (hq + 2 * hkv) * D), generator=g, device=dev)
    parents = _i32([[-1] + [i // 2 for i in range(n - 1)]], dev)
    cos, sin = _tables(max_t, dev)
    clean = v.clone()
    clean[0, :, 97, 9] = clean[0, :, 20, 9] = 0.0
    ref, _, _ = _tree_ref(qkv, parents, [p0], cos, sin, k, clean, hq)
    out = attention.rope_attention_tree(qkv, parents, _i32([p0], dev), cos, sin, k, v)
    assert not torch.isfinite(out[..., 9]).any()
    rest = [d for d in range(D) if d != 9]
    _close(out[..., rest], ref[..., rest])


# ---- eviction ------------------------------------------------------------------------------

def _evict_ref(w, length, keep, sink, recent):
    """Kept rows, ascending."""
    if length <= keep:
        return list(range(length))
    mid = range(sink, length - recent)
    key = lambda i: (-math.inf if math.isnan(w[i]) else w[i] + 0.0, 0 if math.isnan(w[i]) else 1)
    order = sorted(mid, key=lambda i: (-key(i)[0], -key(i)[1], i))
    return sorted(list(range(sink)) + order[:keep - sink - recent] + list(range(length - recent, length)))


EVICT = [
    # B, hkv, length, max_t, keep, sink, recent
    (1, 2, [640], 640, 320, 4, 64),
    (1, 1, [1], 1, 1, 0, 0),
    (1, 1, [2], 5, 1, 0, 0),
    (2, 3, [50, 33], 60, 33, 1, 2),       # one sequence as long as keep
    (3, 2, [100, 5, 0], 100, 40, 0, 0),   # shorter than keep; empty
    (1, 4, [999], 1000, 998, 10, 10),     # one row goes
    (1, 2, [1000], 1000, 64, 32, 32),     # only sinks and recent rows stay
    (1, 2, [1000], 1000, 0, 0, 0),        # nothing stays
    (2, 16, [4097, 3000], 4100, 1025, 16, 100),
    (1, 2, [50000], 50001, 20000, 4, 64),  # a row of weights beyond shared memory
    (2, 40, [300, 299], 300, 100, 3, 5),  # wide slices (many heads)
]


@pytest.mark.parametrize("B,hkv,length,max_t,keep,sink,recent", EVICT)
@pytest.mark.parametrize("alias", [False, True], ids=["apart", "in_place"])
def test_evict_matches_its_definition(cuda_device, B, hkv, length, max_t, keep, sink, recent, alias):
    dev = cuda_device
    g = _gen(B * 7 + keep, dev)
    k, v = _caches(g, B, hkv, max_t, dev)
    # ties (rounded weights), zeros of both signs, NaN and infinities among the weights
    w = torch.round(torch.randn((B, hkv, max_t), generator=g, device=dev) * 8) / 8
    w[..., 3::17] = math.nan
    w[..., 5::101] = math.inf
    w[..., 6::103] = -math.inf
    w[..., 7::13] = -0.0
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    wo = w if alias else torch.full_like(w, 5.0)
    index = attention.kv_evict(w, k, v, _i32(length, dev), keep, sink=sink, recent=recent, weight_out=wo)
    assert index.shape == (B, hkv, keep)
    if not alias:
        assert torch.equal(torch.nan_to_num(w, 7.0), torch.nan_to_num(w0, 7.0))
    index = index.cpu()
    for b in range(B):
        for h in range(hkv):
            want = _evict_ref(w0[b, h].tolist(), length[b], keep, sink, recent)
            n = len(want)
            assert index[b, h].tolist() == want + [-1] * (keep - n)
            at = torch.tensor(want, dtype=torch.long, device=dev)
            for new, old in ((k, k0), (v, v0)):
                assert torch.equal(new[b, h, :n], old[b, h, at]) and torch.equal(new[b, h, n:], old[b, h, n:])
            assert torch.equal(torch.nan_to_num(wo[b, h, :n], 7.0), torch.nan_to_num(w0[b, h, at], 7.0))
            assert torch.count_nonzero(wo[b, h, n:]) == 0


@pytest.mark.parametrize("heads", [1, 3])
def test_move_rows(cuda_device, heads):
    """In place at each sequence's base; indices that do not point forward, or past the cache,
    move nothing."""
    dev, B, hkv, max_t, count = cuda_device, 2, 3, 50, 6
    g = _gen(13, dev)
    k, v = _caches(g, B, hkv, max_t, dev)
    k0, v0 = k.clone(), v.clone()
    base = [10, 44]
    idx = torch.tensor([[0, 2, 3, 7, 8, -1], [1, 2, 4, 5, 6, 9]], dtype=torch.int32, device=dev)
    if heads > 1:
        idx = torch.stack([idx, idx.clamp(max=4), torch.arange(6, device=dev).expand(2, 6).to(torch.int32)], 1)
    attention.kv_move_rows(k, v, idx.contiguous(), base=_i32(base, dev))
    for b in range(B):
        for h in range(hkv):
            row = (idx[b] if heads == 1 else idx[b, h]).tolist()
            for new, old in ((k, k0), (v, v0)):
                want = old[b, h].clone()
                for i, src in enumerate(row):
                    if src > i and base[b] + src < max_t:
                        want[base[b] + i] = old[b, h, base[b] + src]
                assert torch.equal(new[b, h], want)


# ---- blocks --------------------------------------------------------------------------------

def _blocks_ref(q, k, v, keys, pos, block, topk):
    B, t, hq, _ = q.shape
    hkv, max_t = k.shape[1], k.shape[2]
    g = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    index = torch.full((B, t, hkv, topk), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(t):
            at = int(pos[b]) + i
            if pos[b] < 0 or at >= max_t:
                continue
            own = at // block
            for h in range(hkv):
                s = (keys[b, h, :own].double() @ q[b, i, h * g:(h + 1) * g].double().sum(0)).tolist()
                key = [(-math.inf, 0) if math.isnan(x) else (x, 1) for x in s]
                best = sorted(sorted(range(own), key=lambda c: (-key[c][0], -key[c][1], c))[:topk])
                index[b, i, h, :len(best)] = torch.tensor(best, dtype=torch.int32)
                rows = [r for c in best for r in range(c * block, (c + 1) * block)] + list(range(own * block, at + 1))
                rows = torch.tensor(rows, device=q.device)
                seen = torch.ones((g, len(rows)), dtype=torch.bool, device=q.device)
                out[b, i, h * g:(h + 1) * g], _ = _softmax_rows(q[b, i, h * g:(h + 1) * g], k[b, h, rows], v[b, h, rows],
                                                               seen)
    return out, index


BLOCKS = [
    # B, t, hq, hkv, pos, max_t, block, topk
    (1, 1, 2, 2, [0], 1, 16, 1),
    (1, 1, 16, 2, [2000], 2048, 64, 4),
    (3, 1, 16, 16, [63, 64, 65], 100, 64, 2),   # at a block's border; fewer blocks than topk
    (2, 1, 40, 1, [700, 300], 800, 32, 5),      # a group of 40
    (1, 50, 16, 2, [500], 600, 16, 8),          # a chunk, every row its own blocks
    (2, 70, 12, 4, [0, 111], 200, 32, 3),       # a prompt from nothing, ragged
    (1, 3, 8, 1, [1000], 1100, 128, 20),        # topk beyond the blocks
    (2, 4, 4, 2, [98, -1], 100, 16, 2),         # rows past the cache; no sequence
    (6, 8, 16, 16, [900] * 6, 1000, 64, 3),     # more units than a split serves
]


@pytest.mark.parametrize("B,t,hq,hkv,pos,max_t,block,topk", BLOCKS)
def test_blocks_match_their_definition(cuda_device, B, t, hq, hkv, pos, max_t, block, topk):
    dev = cuda_device
    g = _gen(t + block + topk, dev)
    fill = [p + t if p >= 0 else 0 for p in pos]
    k, v = _caches(g, B, hkv, max_t, dev, fill=fill)
    q = torch.randn((B, t, hq, D), generator=g, device=dev) * 1.5
    keys = torch.full((B, hkv, -(-max_t // block), D), math.nan, device=dev)
    # the history in one call, the new rows in another, as a program appends them
    start = _i32([0 if p >= 0 else -1 for p in pos], dev)
    attention.block_keys(k, start, max(1, max(pos)), block, keys=keys)
    attention.block_keys(k, _i32(pos, dev), t, block, keys=keys)
    for b, n in enumerate(fill):
        done = min(max(n, max(pos) if pos[b] >= 0 else 0), max_t) // block
        mean = k[b, :, :done * block].double().view(hkv, done, block, D).mean(2)
        sure = min(n, max_t) // block
        assert torch.equal(keys[b, :, :sure], mean[:, :sure].float())
    ref, iref = _blocks_ref(q, k, v, keys, pos, block, topk)
    out, index = attention.attention_blocks(q, k, v, keys, _i32(pos, dev), block, topk)
    assert torch.equal(index.cpu(), iref)
    _close(out, ref)


def test_blocks_ties_go_to_the_lower_block(cuda_device):
    dev, block, topk, own = cuda_device, 16, 3, 9
    g = _gen(17, dev)
    k, v = _caches(g, 1, 1, 160, dev)
    keys = torch.zeros((1, 1, 10, D), device=dev)
    keys[0, 0, [2, 4, 5, 7], 0] = 1.0
    keys[0, 0, 1] = math.nan
    q = torch.zeros((1, 1, 2, D), device=dev)
    q[..., 0] = 1.0
    _, index = attention.attention_blocks(q, k, v, keys, _i32([own * block], dev), block, topk)
    assert index.flatten().tolist() == [2, 4, 5]
    _, index = attention.attention_blocks(-q, k, v, keys, _i32([own * block], dev), block, 6)
    assert index.flatten().tolist() == [0, 2, 3, 4, 6, 8]


def test_block_keys_touch_only_completed_blocks(cuda_device):
    dev = cuda_device
    g = _gen(18, dev)
    k, _ = _caches(g, 2, 2, 100, dev)
    keys = torch.full((2, 2, 7, D), 3.0, device=dev)
    attention.block_keys(k, _i32([30, 40], dev), 20, 16, keys=keys)  # rows 30..49 and 40..59
    for b, done in enumerate(([1, 2], [2])):
        for c in range(7):
            if c in done:
                assert torch.equal(keys[b, :, c], k[b, :, c * 16:c * 16 + 16].double().mean(1).float())
            else:
                assert torch.all(keys[b, :, c] == 3.0)


# ---- how they are called --------------------------------------------------------------------

def _case(dev, seed=21, B=2, hq=8, hkv=2, max_t=80, n=6):
    g = _gen(seed, dev)
    k, v = _caches(g, B, hkv, max_t, dev)
    cos, sin = _tables(max_t, dev)
    return dict(k=k, v=v, qkv=torch.randn((B, n, (hq + 2 * hkv) * D), generator=g, device=dev),
                q=torch.randn((B, 1, hq, D), generator=g, device=dev), cos=cos, sin=sin,
                parents=_i32([[-1, 0, 0, 1, 2, 2][:n]] * B, dev), pos=_i32([30, 17][:B], dev),
                w=torch.zeros((B, hkv, max_t), device=dev), keys=attention.block_keys(k, _i32([0] * B, dev), max_t, 16))


def _run_all(c):
    """Every operator once, on the case's own buffers."""
    a = attention.rope_attention_tree(c["qkv"], c["parents"], c["pos"], c["cos"], c["sin"], c["k"], c["v"])
    b = attention.attention_weights(c["q"], c["k"], c["v"], c["pos"], c["w"])
    d, index = attention.attention_blocks(c["q"], c["k"], c["v"], c["keys"], c["pos"], 16, 1)
    kept = attention.kv_evict(c["w"], c["k"], c["v"], c["pos"], 12, sink=2, recent=4, weight_out=c["w"])
    return a, b, d, index, kept


def test_operators_replay_from_a_cuda_graph_as_positions_grow(cuda_device):
    """One captured graph of all operators, replayed with other positions and inputs in place,
    and a second graph captured beside it: each equals the eager calls."""
    dev = cuda_device
    c1, c2 = _case(dev), _case(dev, seed=22, B=1, n=4)
    _run_all(_case(dev))  # kernel attributes before the capture
    graphs = []
    for c in (c1, c2):
        s, graph = torch.cuda.Stream(dev), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            outs = _run_all(c)
        graphs.append((graph, c, outs))
    for seed, pos in ((31, [40, 9]), (32, [60, 61])):
        fresh = [_case(dev, seed=seed), _case(dev, seed=seed + 5, B=1, n=4)]
        for (graph, c, outs), f in zip(graphs, fresh):
            f["pos"].copy_(_i32(pos[:f["pos"].numel()], dev))
            for name in c:
                c[name].copy_(f[name])
        torch.cuda.synchronize()
        for graph, _, _ in graphs:  # both in flight before either is looked at
            graph.replay()
        torch.cuda.synchronize()
        for (graph, c, outs), f in zip(graphs, fresh):
            for got, want in zip(outs, _run_all(f)):
                assert torch.equal(got, want)
            assert torch.equal(c["k"], f["k"]) and torch.equal(c["v"], f["v"]) and torch.equal(c["w"], f["w"])
    del graphs


def test_operators_on_two_streams_at_once(cuda_device):
    dev = cuda_device
    want = [_run_all(_case(dev, seed=s)) for s in (41, 42)]
    torch.cuda.synchronize()
    cases = [_case(dev, seed=s) for s in (41, 42)]
    streams = [torch.cuda.Stream(dev) for _ in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (c, s) in enumerate(zip(cases, streams)):
            fresh = _case(dev, seed=41 + i)
            torch.cuda.synchronize()
            for name in c:
                c[name].copy_(fresh[name])
            torch.cuda.synchronize()
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i] = _run_all(c)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for x, y in zip(g, w):
                assert torch.equal(x, y)


def test_results_repeat_bit_for_bit(cuda_device):
    dev = cuda_device
    runs = [_run_all(_case(dev, seed=51)) for _ in range(3)]
    for r in runs[1:]:
        for x, y in zip(r, runs[0]):
            assert torch.equal(x, y)


def test_single_sequence_caches_may_drop_the_batch(cuda_device):
    """[kv_heads, max_t, 128] caches, as Q8Decoder holds them."""
    dev = cuda_device
    a, b = _case(dev, seed=61, B=1), _case(dev, seed=61, B=1)
    b["k"], b["v"], b["w"] = b["k"][0], b["v"][0], b["w"][0]
    for x, y in zip(_run_all(a), _run_all(b)):
        assert torch.equal(x, y)


def test_outputs_and_workspaces_of_the_caller(cuda_device):
    dev = cuda_device
    L = _lib.lib()
    a, b = _case(dev, seed=71), _case(dev, seed=71)
    out = torch.full((2, 6, 8, D), 9.0, device=dev)
    ws = torch.full((L.q8lin_attention_tree_workspace_size(2, 6, 8, 2),), 0xab, dtype=torch.uint8, device=dev)
    got = attention.rope_attention_tree(a["qkv"], a["parents"], a["pos"], a["cos"], a["sin"], a["k"], a["v"], out=out,
                                        workspace=ws)
    assert got is out
    assert torch.equal(out, attention.rope_attention_tree(b["qkv"], b["parents"], b["pos"], b["cos"], b["sin"], b["k"],
                                                          b["v"]))
    with pytest.raises(Q8LinError) as e:
        attention.rope_attention_tree(a["qkv"], a["parents"], a["pos"], a["cos"], a["sin"], a["k"], a["v"],
                                      workspace=ws[:16])
    assert e.value.status == _lib.ERR_WORKSPACE


def test_tensors_that_do_not_fit_are_refused(cuda_device):
    dev = cuda_device
    c = _case(dev)
    tree = lambda **x: attention.rope_attention_tree(*[{**c, **x}[n] for n in
                                                       ("qkv", "parents", "pos", "cos", "sin", "k", "v")])
    for status, change in (
            (_lib.ERR_INVALID_ARGUMENT, {"qkv": c["qkv"].half()}),
            (_lib.ERR_INVALID_ARGUMENT, {"qkv": c["qkv"].transpose(0, 1)[:, ::1].transpose(0, 1)[:, ::2]}),
            (_lib.ERR_INVALID_ARGUMENT, {"parents": c["parents"].long()}),
            (_lib.ERR_INVALID_ARGUMENT, {"k": c["k"][:, :, ::2], "v": c["v"][:, :, ::2]}),
            (_lib.ERR_SHAPE, {"parents": c["parents"][:1]}),
            (_lib.ERR_SHAPE, {"pos": c["pos"][:1]}),
            (_lib.ERR_SHAPE, {"cos": c["cos"][:50]}),
            (_lib.ERR_SHAPE, {"v": c["v"][:, :1].contiguous()}),
            (_lib.ERR_SHAPE, {"qkv": c["qkv"][..., :5 * D].contiguous()}),  # 5 - 4 heads over 2
            (_lib.ERR_DEVICE, {"qkv": c["qkv"].cpu()}),
            (_lib.ERR_DEVICE, {"k": c["k"].cpu(), "v": c["v"].cpu()})):
        with pytest.raises(Q8LinError) as e:
            tree(**change)
        assert e.value.status == status, change.keys()
    with pytest.raises(Q8LinError):
        attention.attention_weights(c["q"], c["k"], c["v"], c["pos"], c["w"][:, :, :-1].contiguous())
    with pytest.raises(Q8LinError):
        attention.kv_evict(c["w"], c["k"], c["v"], c["pos"], 8, sink=5, recent=4)
    with pytest.raises(Q8LinError):
        attention.attention_blocks(c["q"], c["k"], c["v"], c["keys"], c["pos"], 24, 1)
    with pytest.raises(Q8LinError):
        attention.kv_move_rows(c["k"], c["v"], _i32([[0]], dev))


def test_a_wait_that_runs_out_reports_itself(cuda_device):
    """With a wait limit of 0 the tensor-core kernels give up at their first wait that is not over
    at once: fault bit 5, rows NaN or right, the context usable, and the next call with the
    usual limit right again."""
    import ctypes

    dev, L = cuda_device, _lib.lib()
    g = _gen(91, dev)
    B, t, hq, hkv, max_t = 2, 40, 16, 2, 700
    k, v = _caches(g, B, hkv, max_t, dev)
    q = torch.randn((B, t, hq, D), generator=g, device=dev)
    pos = [600, 300]
    flags = ctypes.c_uint32(0)
    _lib.check(L.q8lin_fault_status(0, ctypes.byref(flags), 1))
    ref, wref = _weights_ref(q, k, v, pos, torch.zeros((B, hkv, max_t), device=dev))
    old = L.q8lin_wait_limit_ns()
    try:
        assert L.q8lin_set_wait_limit_ns(0) == 0
        w = torch.zeros((B, hkv, max_t), device=dev)
        out = attention.attention_weights(q, k, v, _i32(pos, dev), w)
        torch.cuda.synchronize()
    finally:
        L.q8lin_set_wait_limit_ns(old)
    _lib.check(L.q8lin_fault_status(0, ctypes.byref(flags), 1))
    assert flags.value == 32
    # which of the kernels had to wait is a matter of timing; what one gave up on is NaN
    assert torch.isnan(out).any() or torch.isnan(w).any()
    _close(torch.where(torch.isnan(out), ref.to(out.dtype), out), ref)
    w = torch.zeros((B, hkv, max_t), device=dev)
    out = attention.attention_weights(q, k, v, _i32(pos, dev), w)
    _close(out, ref)
    _close(w, wref, "weight")
    _lib.check(L.q8lin_fault_status(0, ctypes.byref(flags), 1))
    assert flags.value == 0
