"""Q8Decoder's block-sparse mode: keys that a capture leaves behind, and what a decoder refuses."""
import pytest
import torch

from talechime_b200.decoder import Q8Decoder, synthetic_weights
from test_decoder_kv_gpu import PROMPT, _cfg, _greedy

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = _cfg()
    return cfg, synthetic_weights(cfg, seed=5)


def test_a_capture_does_not_count_as_a_refresh(cuda_device, model):
    """A "blocks" step captured while the keys are out of date records their refresh: the graph's replays are
    right, and so is an eager step that comes before any of them."""
    cfg, w = model
    prompt = PROMPT * 4
    ref, eager, replayed = (Q8Decoder(cfg, w, device=cuda_device, blocks=(16, 1)) for _ in range(3))
    for d in (ref, eager, replayed):
        d.prefill(prompt)  # dense: no keys
    warm = Q8Decoder(cfg, w, device=cuda_device, blocks=(16, 1))
    warm.prefill(prompt)
    warm.step("blocks")  # kernel attributes before the captures
    graphs = []
    for d in (eager, replayed):
        s, graph = torch.cuda.Stream(cuda_device), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            d.step("blocks")
        graphs.append(graph)
    want = _greedy(ref, 4, "blocks")
    assert _greedy(eager, 4, "blocks") == want
    got = []
    for _ in range(4):
        graphs[1].replay()
        torch.cuda.synchronize()
        got.append(int(replayed.token.item()))
    assert got == want
    for d in (eager, replayed):
        assert torch.equal(d.logits, ref.logits)
        done = (len(prompt) + 4) // 16  # a refresh also writes blocks that are not complete, which nothing reads
        assert all(torch.equal(a[:, :, :done], b[:, :, :done]) for a, b in zip(d.block_keys, ref.block_keys))
    del graphs
