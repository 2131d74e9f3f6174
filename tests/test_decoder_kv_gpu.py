"""Q8Decoder's trees of drafted tokens, tracked attention with eviction, and block-sparse modes."""
import numpy as np
import pytest
import torch

from talechime_b200 import Q8LinError, _lib, attention
from talechime_b200.decoder import DecoderConfig, Q8Decoder, synthetic_weights

pytestmark = pytest.mark.gpu

# whole-model logits of two GPU paths: one re-quantized activation block may flip
# (tests/test_decoder_gpu.py)
LOGITS_REL_L2 = 2e-3
FLIP_REL_L2 = 3e-2


def _cfg(**kw):
    return DecoderConfig(**{**dict(hidden=256, layers=2, heads=4, kv_heads=2, inter=512, vocab=1000, max_t=64), **kw})


def _rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm())


def _greedy(dec, n, mode="fused"):
    out = []
    for _ in range(n):
        dec.step(mode)
        out.append(int(dec.token.item()))
    return out


@pytest.fixture(scope="module")
def model():
    cfg = _cfg(max_pos=256)
    return cfg, synthetic_weights(cfg, seed=5)


PROMPT = [3, 141, 59, 26, 535, 897, 932, 384]


def test_tree_steps_give_the_tokens_of_plain_steps(cuda_device, model):
    """Drafts that are right, partly right and wrong: the same tokens as plain greedy steps, the
    caches of the accepted rows as plain steps leave them, and decoding goes on from there."""
    cfg, w = model
    plain = Q8Decoder(cfg, w, device=cuda_device)
    plain.prefill(PROMPT)
    first = int(plain.token.item())
    want = _greedy(plain, 12)
    dec = Q8Decoder(cfg, w, device=cuda_device)
    dec.prefill(PROMPT)
    bad = lambda t: (t + 1) % cfg.vocab
    got = []
    # a chain of right drafts behind wrong siblings: nodes 0, 2, 4, 5 are the path
    got += dec.step_tree([first, bad(want[0]), want[0], bad(want[1]), want[1], want[2], bad(want[2])],
                         [-1, 0, 0, 2, 2, 4, 4])
    assert got == want[:4] and int(dec.pos.item()) == len(PROMPT) + 4
    # all drafts wrong: one token
    got += dec.step_tree([got[-1], bad(want[4]), 7], [-1, 0, 1])
    assert got == want[:5]
    # no drafts; then the first branch holds
    got += dec.step_tree([got[-1]], [-1])
    got += dec.step_tree([got[-1], want[6], bad(want[6])], [-1, 0, 0])
    assert got == want[:8]
    n = int(dec.pos.item())
    assert n == len(PROMPT) + 8
    for li in range(cfg.layers):
        assert _rel(dec.k_cache[li][:, :n], plain.k_cache[li][:, :n]) <= FLIP_REL_L2
        assert _rel(dec.v_cache[li][:, :n], plain.v_cache[li][:, :n]) <= FLIP_REL_L2
    assert got + _greedy(dec, 4) == want


def test_tree_logits_equal_a_prefill_along_each_path(cuda_device, model):
    cfg, w = model
    tokens, parents = [11, 22, 33, 44, 55], [-1, 0, 0, 2, 1]
    dec = Q8Decoder(cfg, w, device=cuda_device)
    dec.prefill(PROMPT)
    nxt = dec.verify_tree(torch.tensor(tokens), torch.tensor(parents))
    assert nxt.shape == (5,) and dec.tree_logits.shape == (5, cfg.vocab)
    for path in ([0], [0, 1], [0, 2], [0, 2, 3], [0, 1, 4]):
        ref = Q8Decoder(cfg, w, device=cuda_device)
        ref.prefill(PROMPT)
        pick = ref.prefill([tokens[i] for i in path])
        assert _rel(dec.tree_logits[path[-1]], ref.logits) <= FLIP_REL_L2
        assert int(nxt[path[-1]]) == int(dec.tree_logits[path[-1]].argmax())
        assert int(pick) == int(ref.logits.argmax())
    assert int(dec.pos.item()) == len(PROMPT)  # verifying moves nothing on


def test_tree_launches_replay_from_a_cuda_graph(cuda_device, model):
    """The launches of a tree capture; a replay behind a longer history and with other tokens
    equals the eager call."""
    cfg, w = model
    dec, ref = (Q8Decoder(cfg, w, device=cuda_device) for _ in range(2))
    for d in (dec, ref):
        d.prefill(PROMPT)
        d.verify_tree([1, 2, 3], [-1, 0, 0])
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device=cuda_device)
    par = torch.tensor([[-1, 0, 0]], dtype=torch.int32, device=cuda_device)
    s, graph = torch.cuda.Stream(cuda_device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        nxt = dec._tree_launches(tok, par)
        logits = dec.tree_logits
    for d in (dec, ref):
        d.prefill([77, 78])
    tok.copy_(torch.tensor([9, 8, 7], dtype=torch.int32))
    par.copy_(torch.tensor([[-1, 0, 1]], dtype=torch.int32))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    want = ref.verify_tree([9, 8, 7], [-1, 0, 1])
    assert torch.equal(nxt, want) and torch.equal(logits, ref.tree_logits)
    del graph


def test_tree_refusals(cuda_device, model):
    cfg, w = model
    dec = Q8Decoder(cfg, w, device=cuda_device)
    dec.prefill(PROMPT)
    for tok, par in (([1, 2], [-1]), ([], []), ([1, 2], [-1, 1]), ([1, 2], [-1, -2]), ([[1]], [[-1]])):
        with pytest.raises(Q8LinError):
            dec.verify_tree(tok, par)
    with pytest.raises(Q8LinError) as e:
        dec.verify_tree(list(range(57)), [-1] * 57)  # 8 + 57 > 64
    assert e.value.status == _lib.ERR_SHAPE
    with pytest.raises(Q8LinError):
        dec.step_tree([int(dec.token.item()) + 1], [-1])
    with pytest.raises(Q8LinError):
        dec.step_tree([int(dec.token.item()), 5], [-1, -1])
    with pytest.raises(Q8LinError):
        dec.accept_path([0, 2, 1], 5)
    with pytest.raises(ValueError):
        Q8Decoder(cfg, w, device=cuda_device, batch=2).verify_tree([1], [-1])
    assert int(dec.pos.item()) == len(PROMPT)


def test_tracked_steps_and_prompts(cuda_device, model):
    """The tracked modes give the plain modes' logits, and every row and head adds one unit of
    weight per layer, none of it behind the last row."""
    cfg, w = model
    dec = Q8Decoder(cfg, w, device=cuda_device, track_weights=True)
    ref = Q8Decoder(cfg, w, device=cuda_device)
    dec.prefill(PROMPT, mode="tracked")
    ref.prefill(PROMPT)
    assert _rel(dec.logits, ref.logits) <= FLIP_REL_L2
    assert _greedy(dec, 3, "tracked") == _greedy(ref, 3)
    assert _rel(dec.logits, ref.logits) <= FLIP_REL_L2
    n = len(PROMPT) + 3
    for li in range(cfg.layers):
        kw = dec.kv_weight[li]
        assert kw.shape == (cfg.kv_heads, cfg.max_t)
        torch.testing.assert_close(kw.sum(-1), torch.full((cfg.kv_heads,), 2.0 * n, device=cuda_device), rtol=1e-5, atol=0)
        assert torch.count_nonzero(kw[:, n:]) == 0
    dec.reset()
    assert all(torch.count_nonzero(x) == 0 for x in dec.kv_weight)
    with pytest.raises(ValueError):
        ref.step("tracked")
    with pytest.raises(ValueError):
        ref.prefill(PROMPT, mode="tracked")
    with pytest.raises(ValueError):
        ref.evict(4)


@pytest.mark.parametrize("mode", ["fused", "unfused", "persistent", "tracked"])
def test_steps_after_an_eviction(cuda_device, model, mode):
    """evict() keeps the heaviest rows of every head; a step after it equals a step of a decoder
    whose caches were put together by hand and whose RoPE tables begin at the rows gone."""
    cfg, w = model
    dec = Q8Decoder(cfg, w, device=cuda_device, track_weights=True)
    dec.prefill(PROMPT * 4, mode="tracked")
    dec.step("tracked")
    dec.step("persistent")  # a program with the old position offset
    n, keep, sink, recent = len(PROMPT) * 4 + 2, 20, 2, 5
    hand = Q8Decoder(cfg, w, device=cuda_device, track_weights=True)
    hand.cos, hand.sin = dec.cos[n - keep:].contiguous(), dec.sin[n - keep:].contiguous()
    for li in range(cfg.layers):
        kw = dec.kv_weight[li].cpu().numpy()
        for h in range(cfg.kv_heads):
            mid = sorted(range(sink, n - recent), key=lambda i: (-kw[h, i], i))[:keep - sink - recent]
            rows = torch.tensor(list(range(sink)) + sorted(mid) + list(range(n - recent, n)), device=cuda_device)
            hand.k_cache[li][h, :keep] = dec.k_cache[li][h, rows]
            hand.v_cache[li][h, :keep] = dec.v_cache[li][h, rows]
            hand.kv_weight[li][h, :keep] = dec.kv_weight[li][h, rows]
    hand.pos.fill_(keep)
    hand.token.copy_(dec.token)
    assert dec.evict(keep, sink=sink, recent=recent) == n - keep
    assert int(dec.pos.item()) == keep and dec.evicted == n - keep
    for _ in range(2):
        dec.step(mode)
        hand.step(mode)
        assert torch.equal(dec.logits, hand.logits) and torch.equal(dec.token, hand.token)
    for li in range(cfg.layers):
        for a, b in ((dec.k_cache, hand.k_cache), (dec.v_cache, hand.v_cache), (dec.kv_weight, hand.kv_weight)):
            assert torch.equal(a[li][:, :keep + 2], b[li][:, :keep + 2])
    # prompts and trees run on from the same position
    dec.prefill([5, 6])
    hand.prefill([5, 6])
    assert torch.equal(dec.logits, hand.logits)
    assert torch.equal(dec.verify_tree([1, 2], [-1, 0]), hand.verify_tree([1, 2], [-1, 0]))
    assert torch.equal(dec.tree_logits, hand.tree_logits)


def test_eviction_makes_room_past_the_context_limit(cuda_device):
    """A cache of 24 rows serves 60 tokens; eviction that keeps everything changes nothing; tables
    that end too early refuse."""
    cfg = _cfg(max_t=24, max_pos=64)
    w = synthetic_weights(cfg, seed=6)
    dec = Q8Decoder(cfg, w, device=cuda_device, track_weights=True)
    dec.prefill(PROMPT, mode="tracked")
    before = [c.clone() for c in dec.k_cache]
    assert dec.evict(len(PROMPT)) == 0 and dec.evict(20, sink=1, recent=2) == 0 and dec.evicted == 0
    assert all(torch.equal(a, b) for a, b in zip(before, dec.k_cache))
    for _ in range(52):
        if int(dec.pos.item()) == cfg.max_t:
            dec.evict(14, sink=2, recent=6)
        dec.step("tracked")
        assert torch.isfinite(dec.logits).all()
    assert dec.evicted + int(dec.pos.item()) == len(PROMPT) + 52
    with pytest.raises(Q8LinError):
        dec.evict(1)
    with pytest.raises(Q8LinError):
        dec.evict(6, sink=4, recent=3)
    dec.reset(3)
    assert dec.evicted == 0 and int(dec.pos.item()) == 0


def test_eviction_of_a_batch(cuda_device, model):
    """Sequences of a batch keep rows of their own."""
    cfg, w = model
    toks = np.random.default_rng(8).integers(0, cfg.vocab, (3, 30))
    big = Q8Decoder(cfg, w, device=cuda_device, batch=3, track_weights=True)
    big.prefill(toks, mode="tracked")
    kept = [attention.kv_evict(x, k.clone(), v.clone(), big.pos.expand(3).contiguous(), 12, recent=3)
            for x, k, v in zip(big.kv_weight, big.k_cache, big.v_cache)]
    k0 = [k.clone() for k in big.k_cache]
    assert big.evict(12, recent=3) == 18
    for li in range(cfg.layers):
        for b in range(3):
            for h in range(cfg.kv_heads):
                assert torch.equal(big.k_cache[li][b, h, :12], k0[li][b, h, kept[li][b, h].long()])
    big.prefill(toks[:, :4], mode="tracked")
    assert torch.isfinite(big.prefill_logits).all()


def test_block_modes(cuda_device, model):
    """With as many blocks as there are, the blocks modes give the plain modes' logits; with fewer
    they attend over the chosen ones; keys kept up step by step equal keys made anew."""
    cfg, w = model
    ref = Q8Decoder(cfg, w, device=cuda_device)
    all_ = Q8Decoder(cfg, w, device=cuda_device, blocks=(16, 4))
    few = Q8Decoder(cfg, w, device=cuda_device, blocks=(16, 1))
    prompt = PROMPT * 4
    for d, m in ((ref, "dense"), (all_, "blocks"), (few, "blocks")):
        d.prefill(prompt, mode=m)
    assert _rel(all_.logits, ref.logits) <= FLIP_REL_L2
    want = _greedy(ref, 18)
    assert _greedy(all_, 18, "blocks") == want
    _greedy(few, 18, "blocks")
    assert torch.isfinite(few.logits).all()
    done = (len(prompt) + 18) // 16
    for d in (all_, few):
        for li in range(cfg.layers):
            k = d.k_cache[li][:, :done * 16].double().view(cfg.kv_heads, done, 16, 128).mean(2).float()
            assert torch.equal(d.block_keys[li][0, :, :done], k)
    # steps of another mode leave the keys behind; the next blocks step catches up
    all_.step("fused")
    for d in (ref, all_):
        d.step("fused" if d is ref else "blocks")
    with pytest.raises(ValueError):
        ref.step("blocks")
    with pytest.raises(ValueError):
        ref.prefill([1], mode="blocks")


def test_tracked_and_block_steps_replay_from_a_cuda_graph(cuda_device, model):
    cfg, w = model
    for mode in ("tracked", "blocks"):
        make = lambda: Q8Decoder(cfg, w, device=cuda_device, track_weights=True, blocks=(16, 1))
        a, b = make(), make()
        for d in (a, b):
            d.prefill(PROMPT * 2, mode=mode)
        want = _greedy(a, 6, mode)
        b.step(mode)  # warm-up
        s, graph = torch.cuda.Stream(cuda_device), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            b.step(mode)
        got = [want[0]]
        for _ in range(5):
            graph.replay()
            torch.cuda.synchronize()
            got.append(int(b.token.item()))
        assert got == want
        assert torch.equal(a.logits, b.logits)
        del graph
