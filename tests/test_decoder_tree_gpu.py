"""Q8Decoder's trees of drafted tokens: what step_tree keeps and what accept_path refuses."""
import pytest
import torch

from talechime_b200 import Q8LinError, _lib
from talechime_b200.decoder import Q8Decoder, synthetic_weights
from test_decoder_kv_gpu import FLIP_REL_L2, PROMPT, _cfg, _greedy, _rel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = _cfg(max_pos=256)
    return cfg, synthetic_weights(cfg, seed=5)


def test_step_tree_keeps_the_longer_of_two_equal_branches(cuda_device, model):
    cfg, w = model
    plain, dec = (Q8Decoder(cfg, w, device=cuda_device) for _ in range(2))
    for d in (plain, dec):
        d.prefill(PROMPT)
    first = int(plain.token.item())
    want = _greedy(plain, 5)
    got = dec.step_tree([first, want[0], want[0], want[1], want[2]], [-1, 0, 0, 2, 3])
    assert got == want[:4]
    assert int(dec.pos.item()) == len(PROMPT) + 4
    assert got + _greedy(dec, 1) == want
    n = len(PROMPT) + 4
    for li in range(cfg.layers):
        assert _rel(dec.k_cache[li][:, :n], plain.k_cache[li][:, :n]) <= FLIP_REL_L2


def test_accept_path_takes_paths_of_the_last_tree_alone(cuda_device, model):
    """Nodes the tree does not have, siblings, a path without its root, a tree that was accepted from, and one
    that a step, a prompt, an eviction or a reset has overtaken: refused, position, token and rows as they were."""
    cfg, w = model
    dec = Q8Decoder(cfg, w, device=cuda_device, track_weights=True)

    def refused(path):
        before = int(dec.pos.item()), int(dec.token.item()), [c.clone() for c in dec.k_cache]
        with pytest.raises(Q8LinError) as e:
            dec.accept_path(path, 5)
        assert e.value.status == _lib.ERR_INVALID_ARGUMENT
        assert (int(dec.pos.item()), int(dec.token.item())) == before[:2]
        assert all(torch.equal(a, b) for a, b in zip(dec.k_cache, before[2]))

    refused([0])  # no tree yet
    dec.prefill(PROMPT, mode="tracked")
    refused([0])
    tree = lambda: dec.verify_tree([11, 22, 33, 44], [-1, 0, 0, 2])
    tree()
    for path in ([4], [0, 4], [0, 500], [-1], [0, -1], [1], [0, 3], [0, 1, 2], [0, 1, 3], [0, 0], [2, 3], list(range(60))):
        refused(path)
    dec.accept_path([0, 2, 3], 5)
    assert int(dec.pos.item()) == len(PROMPT) + 3 and int(dec.token.item()) == 5
    refused([0])
    tree()
    dec.accept_path([], 6)  # none of it
    assert int(dec.pos.item()) == len(PROMPT) + 3 and int(dec.token.item()) == 6
    refused([0])
    for other in (lambda: dec.step("tracked"), lambda: dec.prefill([1, 2]), lambda: dec.evict(9),
                  lambda: (dec.reset(), dec.prefill(PROMPT + [1]))):
        tree()
        other()
        refused([0])


def test_accept_path_of_a_graph_that_moved_on(cuda_device, model):
    """A replayed step moves the position without the decoder's knowledge: the tree before it is not accepted."""
    cfg, w = model
    dec = Q8Decoder(cfg, w, device=cuda_device)
    dec.prefill(PROMPT)
    dec.step()
    s, graph = torch.cuda.Stream(cuda_device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        dec.step()
    dec.verify_tree([1, 2], [-1, 0])
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(Q8LinError):
        dec.accept_path([0], 3)
    del graph


def test_trees_of_any_size_behind_one_another(cuda_device):
    """Wide feed-forward layers (6144, the production width): a tree after a larger one, where another kernel
    serves the linears and needs more scratch, gives what it gives on its own."""
    cfg = _cfg(layers=1, inter=6144)
    w = synthetic_weights(cfg, seed=6)
    dec = Q8Decoder(cfg, w, device=cuda_device)
    dec.prefill(PROMPT)
    for n in (16, 8, 11, 2, 12, 9, 5, 33, 16, 8):
        tok, par = [(7 * i + n) % cfg.vocab for i in range(n)], [(i - 1) // 2 if i else -1 for i in range(n)]
        dec.verify_tree(tok, par)
        alone = Q8Decoder(cfg, w, device=cuda_device)
        alone.prefill(PROMPT)
        alone.verify_tree(tok, par)
        assert torch.equal(dec.tree_logits, alone.tree_logits), n
