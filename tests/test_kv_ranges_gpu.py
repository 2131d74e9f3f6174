"""Sizes of queries, keys and values in the attention kernels over the KV caches: what a row does not
see may be of any size, what it sees may differ in size from key to key, and neither moves its result
beyond the error of its own scores.

Bounds.  Scores of ordinary size are held to the bound of tests/test_kv_attention_gpu.py.  Where scores
reach S in size, a score is a rounded product of two rounded operands, three halves of an f32 step (2^-24
of S each) and as much again for the pairs that the operands are split into (below 2^-22 of S): under
1.5 * 2^-21 * S, which is the relative error of its probability and, over rows of 128 dimensions
that all move together, at most that of the output: 1.5 * 2^-21 * S + 1e-5."""
import math

import pytest
import torch

from talechime_b200 import attention
from test_kv_attention_gpu import (D, REL_L2, ROOMY, _caches, _close, _gen, _i32, _paths, _tables, _tree_ref, _weights_ref)

pytestmark = pytest.mark.gpu

MAX = torch.finfo(torch.float32).max
SIZES = [2.0 ** 16, 2.0 ** 24, 2.0 ** 36, 1e30, MAX]
FORMS = [(12, 4, 2, 100), (40, 16, 2, 100), (40, 16, 2, ROOMY)]  # 16-row kernel, twice; tensor-core kernel


def _grow(x, size):
    """x at that size; the type's largest number in the signs of x."""
    return torch.sign(x) * MAX if size == MAX else x * size


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n,hq,hkv,max_t", FORMS)
def test_tree_rows_beside_unseen_rows_of_any_size(cuda_device, n, hq, hkv, max_t, size):
    """A draft whose key, value, or both are far larger than its siblings': rows that do not see it
    give what they give without it."""
    dev, p0 = cuda_device, 50
    parents = [-1, 0, 0, 1, 1, 2, 2] + [1 + (i % 2) for i in range(7, n)]
    free = [i for i, path in enumerate(_paths(parents, p0, max_t)) if 2 not in path]
    cos, sin = _tables(max_t, dev)
    for what in ("key", "value", "both"):
        g = _gen(101, dev)
        k, v = _caches(g, 1, hkv, max_t, dev)
        qkv = torch.randn((1, n, (hq + 2 * hkv) * D), generator=g, device=dev)
        ref, _, _ = _tree_ref(qkv, _i32([parents], dev), [p0], cos, sin, k, v, hq)
        rows = qkv.view(1, n, -1, D)[0, 2]
        if what != "value":
            rows[hq:hq + hkv] = _grow(rows[hq:hq + hkv], size)
        if what != "key":
            rows[hq + hkv:] = _grow(rows[hq + hkv:], size)
        out = attention.rope_attention_tree(qkv, _i32([parents], dev), _i32([p0], dev), cos, sin, k, v)
        _close(out[0, free], ref[0, free], what)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("t,hq,hkv,p0", [(3, 4, 2, 20), (3, 16, 4, 0), (40, 4, 2, 20), (70, 16, 2, 0)])
def test_prompt_rows_before_larger_rows(cuda_device, t, hq, hkv, p0, size):
    """Rows in front of far larger ones, the first of a prompt among them: two later rows whose keys and
    values are that much larger leave the outputs before them as they are."""
    dev, max_t = cuda_device, 100
    g = _gen(102, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    q = torch.randn((1, t, hq, D), generator=g, device=dev)
    zero = lambda: torch.zeros((1, hkv, max_t), device=dev)
    ref, _ = _weights_ref(q, k, v, [p0], zero())
    for row in {t - 1, max(1, t // 3)}:
        k[0, :, p0 + row] = _grow(k[0, :, p0 + row], size)
        v[0, :, p0 + row] = _grow(v[0, :, p0 + row], size)
    out = attention.attention_weights(q, k, v, _i32([p0], dev), zero())
    first = max(1, t // 3)
    _close(out[:, :first], ref[:, :first])
    if p0 == 0:
        _close(out[0, 0].view(hkv, -1, D), v[0, :, :1].double().expand(hkv, hq // hkv, D))


def _graded(dev, t, hq, hkv, L, drop, seed):
    """Queries and keys whose scores are -drop[j] and a little, values e^drop[j] times unit normal."""
    g = _gen(seed, dev)
    k, v = _caches(g, 1, hkv, L, dev)
    q = 0.1 * torch.randn((1, t, hq, D), generator=g, device=dev)
    q[..., 0] = math.sqrt(D)
    k *= 0.1
    k[..., 0] = -drop
    return q, k, v * torch.exp(drop)[:, None]


@pytest.mark.parametrize("size", [1.0, 2.0 ** 10, 2.0 ** 20, 2.0 ** 24, 2.0 ** 40])
@pytest.mark.parametrize("t,hq,hkv,L", [(1, 16, 2, 100), (2, 16, 2, 100), (1, 16, 16, 3000), (40, 16, 2, 100), (70, 16, 2, 1500)])
def test_equal_keys_share_the_weight_at_any_score(cuda_device, t, hq, hkv, L, size):
    """Keys that are all alike have scores that are all alike, however large: each row spreads its unit evenly
    and its output is the mean of the values, to the bound that scores of ordinary size have."""
    dev = cuda_device
    g = _gen(108, dev)
    k, v = _caches(g, 1, hkv, L, dev)
    k[:] = k[:, :, :1].clone()
    q = torch.randn((1, t, hq, D), generator=g, device=dev) * size
    w = torch.zeros((1, hkv, L), device=dev)
    out = attention.attention_weights(q, k, v, _i32([L - t], dev), w)
    seen = (torch.arange(L, device=dev) <= L - t + torch.arange(t, device=dev)[:, None]).double()
    p = seen / seen.sum(-1, keepdim=True)
    ref = torch.einsum("tl,bhld->bthd", p, v.double()).repeat_interleave(hq // hkv, 2)
    _close(out, ref)
    _close(w, (p.sum(0) * (hq // hkv)).expand(1, hkv, L), "weight")


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("kind", ["alternating", "by_tile", "by_range"])
def test_small_weights_of_large_values(cuda_device, t, kind):
    """Keys of low score with values as much larger: their share of the output is that of the others,
    beside each other in the cache, in tiles of their own, and over the whole of a long cache."""
    dev, hq, hkv, L = cuda_device, 16, 2, 700
    j = torch.arange(L, device=dev)
    S = 20.0  # values 2^29 times larger
    drop = {"alternating": (j % 2) * S, "by_tile": (j // 64 % 2) * S, "by_range": (j < 350) * S}[kind].float()
    q, k, v = _graded(dev, t, hq, hkv, L, drop, 103)
    w = torch.zeros((1, hkv, L), device=dev)
    ref, wref = _weights_ref(q, k, v, [L - t], w)
    out = attention.attention_weights(q, k, v, _i32([L - t], dev), w)
    bound = 1.5 * 2.0 ** -21 * S + REL_L2
    for i in range(t):
        assert float((out[0, i].double() - ref[0, i]).norm() / ref[0, i].norm()) <= bound, i
    assert float((w.double() - wref).norm() / wref.norm()) <= bound


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("small", [0.0, 1e-12, 1e-30])
def test_heavy_keys_with_small_values(cuda_device, t, small):
    """Keys that take all but 2^-43 of the weight, with values that are zero or next to it: the output is
    the other keys' and has its accuracy."""
    dev, hq, hkv, L = cuda_device, 16, 2, 300
    S = 30.0
    drop = torch.full((L,), S, device=dev)
    heavy = [0, 1, 70, 77]
    drop[heavy] = 0.0
    q, k, v = _graded(dev, t, hq, hkv, L, drop, 104)
    v = v / math.exp(S)
    v[:, :, heavy] *= small * math.exp(S)
    w = torch.zeros((1, hkv, L), device=dev)
    ref, _ = _weights_ref(q, k, v, [L - t], w)
    out = attention.attention_weights(q, k, v, _i32([L - t], dev), w)
    for i in range(t):
        assert float((out[0, i].double() - ref[0, i]).norm() / ref[0, i].norm()) <= 1.5 * 2.0 ** -21 * S + REL_L2, i


@pytest.mark.parametrize("qs,ks,vs", [(1e-18, 1e18, 1e30), (1e12, 1e-12, 1e-30), (1e-12, 1e12, 1e-25), (1.0, 1.0, 1e36)])
@pytest.mark.parametrize("t,L", [(1, 70), (40, 70), (40, 1500)])
def test_large_and_small_numbers_in_prompts(cuda_device, t, L, qs, ks, vs):
    """Queries, keys and values of very different sizes whose scores are ordinary, in a cache that one CTA
    takes whole and in one that several share."""
    dev, hq, hkv = cuda_device, 16, 2
    g = _gen(105, dev)
    k, v = _caches(g, 1, hkv, L, dev)
    q = torch.randn((1, t, hq, D), generator=g, device=dev)
    q, k, v = q * qs, k * ks, v * vs
    w = torch.zeros((1, hkv, L), device=dev)
    ref, wref = _weights_ref(q, k, v, [L - t], w)
    out = attention.attention_weights(q, k, v, _i32([L - t], dev), w)
    assert float((out.double() - ref).norm() / ref.norm()) <= REL_L2
    _close(w, wref, "weight")


@pytest.mark.parametrize("size", [1.0, 2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("n,hq,hkv,max_t", FORMS + [(2, 16, 2, 100)])
def test_tree_nodes_of_equal_keys_take_the_mean_at_any_score(cuda_device, n, hq, hkv, max_t, size):
    """A tree without rotation (cos 1, sin 0) whose keys are those of the history, all alike: a node's output is
    the mean of the values it sees, however large the scores."""
    dev, p0 = cuda_device, 50
    g = _gen(111, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    k[:] = k[:, :, :1].clone()
    qkv = torch.randn((1, n, (hq + 2 * hkv) * D), generator=g, device=dev)
    rows = qkv.view(n, hq + 2 * hkv, D)
    rows[:, :hq] *= size
    rows[:, hq:hq + hkv] = k[0, :, 0]
    one, zero = torch.ones((max_t, 64), device=dev), torch.zeros((max_t, 64), device=dev)
    parents = [(i - 1) // 2 if i else -1 for i in range(n)]
    ref = []
    for i, path in enumerate(_paths(parents, p0, max_t)):
        seen = torch.cat([v[0, :, :p0], rows[path, hq + hkv:].transpose(0, 1)], 1).double()
        ref.append(seen.mean(1).repeat_interleave(hq // hkv, 0))
    out = attention.rope_attention_tree(qkv, _i32([parents], dev), _i32([p0], dev), one, zero, k, v)
    _close(out[0], torch.stack(ref))


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** -24, 2.0 ** -36])
@pytest.mark.parametrize("t,L", [(64, 200), (130, 1500)])
def test_weights_of_query_rows_of_different_sizes(cuda_device, t, L, size):
    """Every third query that much smaller than its neighbours, over keys that give it ordinary scores and the
    others, but for a few, one key each: every row adds one unit, on the keys of its own softmax.

    A score of size S is off by 1.5 * 2^-21 * S at most (above), and so is the weight of a row whose
    weight is not all on one key; the rows whose is (to 1e-6 of it) are off by less than 1e-6 of that."""
    dev, hq, hkv = cuda_device, 16, 2
    g = _gen(106, dev)
    k, v = _caches(g, 1, hkv, L, dev)
    q = torch.randn((1, t, hq, D), generator=g, device=dev)
    q[:, ::3] *= size
    k /= size
    w = torch.zeros((1, hkv, L), device=dev)
    ref, wref = _weights_ref(q, k, v, [L - t], w)
    top, off = 0.0, 0
    for h in range(hq):
        s = (q[0, :, h].double() @ k[0, h // (hq // hkv)].double().T) / math.sqrt(D)
        s = s.masked_fill(torch.arange(L, device=dev) > L - t + torch.arange(t, device=dev)[:, None], -math.inf)
        large = [i for i in range(t) if i % 3]
        one = torch.softmax(s, -1).amax(-1)[large] > 1 - 1e-6
        top = max(top, float(s[large].masked_fill(s[large] == -math.inf, 0.0).abs().max()))
        off += int((~one).sum())
    out = attention.attention_weights(q, k, v, _i32([L - t], dev), w)
    _close(out[:, ::3], ref[:, ::3])
    bound = REL_L2 + (off * 1.5 * 2.0 ** -21 * top + t * hq * 1e-6) / float(wref.norm())
    assert float((w.double() - wref).norm() / wref.norm()) <= bound
    torch.testing.assert_close(w.sum(-1), torch.full((1, hkv), float(t * hq // hkv), device=dev), rtol=1e-5, atol=0)


@pytest.mark.parametrize("t,hq,hkv,p0", [(3, 16, 2, 61), (77, 16, 2, 61), (130, 12, 4, 0), (130, 16, 2, 1003)])
def test_every_row_adds_one_unit_of_weight(cuda_device, t, hq, hkv, p0):
    """Keys whose sizes differ by up to 2^30 within any group, queries whose scores reach 2^30: the weights of
    each row add up to 1 all the same (f32 sums of at most t * hq / hkv units: 1e-5)."""
    dev, max_t = cuda_device, p0 + t + 20
    g = _gen(109, dev)
    k, v = _caches(g, 1, hkv, max_t, dev, fill=[p0 + t])
    k *= torch.exp2(torch.randint(-30, 1, (1, hkv, max_t, 1), generator=g, device=dev).float())
    q = torch.randn((1, t, hq, D), generator=g, device=dev)
    q *= torch.exp2(torch.randint(0, 31, (1, t, hq, 1), generator=g, device=dev).float())
    w = torch.zeros((1, hkv, max_t), device=dev)
    out = attention.attention_weights(q, k, v, _i32([p0], dev), w)
    assert torch.isfinite(out).all() and torch.count_nonzero(w[..., p0 + t:]) == 0
    torch.testing.assert_close(w.double().sum(-1), torch.full((1, hkv), float(t * hq // hkv), device=dev).double(), rtol=1e-5,
                               atol=0)


def test_tree_of_one_path_among_many_sizes(cuda_device):
    """Nodes that grow by 2^10 from child to child: a node sees only smaller ones and itself, and its
    output is its own size's."""
    dev, n, hq, hkv, max_t, p0 = cuda_device, 12, 32, 2, ROOMY, 64
    g = _gen(107, dev)
    k, v = _caches(g, 1, hkv, max_t, dev)
    qkv = torch.randn((1, n, (hq + 2 * hkv) * D), generator=g, device=dev)
    size = torch.exp2(10.0 * torch.arange(n, device=dev))
    qkv.view(1, n, -1, D)[..., hq + hkv:, :] *= size[:, None, None]
    cos, sin = _tables(max_t, dev)
    parents = _i32([list(range(-1, n - 1))], dev)
    ref, _, _ = _tree_ref(qkv, parents, [p0], cos, sin, k, v, hq)
    out = attention.rope_attention_tree(qkv, parents, _i32([p0], dev), cos, sin, k, v)
    for i in range(n):
        _close(out[0, i], ref[0, i], str(i))


@pytest.mark.parametrize("B,t,hq,hkv,L", [(2, 1, 16, 2, 2000), (2, 1, 32, 2, 2000), (2, 60, 16, 2, 2000), (40, 60, 16, 2, 300)])
def test_ordinary_numbers_keep_the_accuracy_of_f32(cuda_device, B, t, hq, hkv, L):
    """Unit normal queries, keys and values, in units of 8 and 16 rows and on the tensor cores with and
    without a split.  What the pairs drop is below 2^-22 of each product, of either sign: 1.5e-7 of a
    score.  The tensor cores cut their sums at most 24 times, by less than 2^-23 of the sum so far, which
    is 0.58 of the whole on average: 1.7e-6 if every cut is as large as it can be.  Exponentials, sums
    and divisions add a few 2^-23.  So 2.5e-6, the probabilities' relative error, bounds the outputs'."""
    dev = cuda_device
    g = _gen(110, dev)
    k, v = _caches(g, B, hkv, L, dev)
    q = torch.randn((B, t, hq, D), generator=g, device=dev)
    w = torch.zeros((B, hkv, L), device=dev)
    ref, wref = _weights_ref(q, k, v, [L - t - 7 * b for b in range(B)], w)
    out = attention.attention_weights(q, k, v, _i32([L - t - 7 * b for b in range(B)], dev), w)
    assert float((out.double() - ref).norm() / ref.norm()) <= 2.5e-6
    assert float((w.double() - wref).norm() / wref.norm()) <= 2.5e-6
