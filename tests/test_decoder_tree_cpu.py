"""Which drafts of a tree a decoder accepts (no GPU)."""
import random

import pytest

from talechime_b200.decoder import longest_path


def _by_search(tokens, parents, picks):
    """Every path from node 0 down, tried one by one."""
    best = [0]
    stack = [[0]]
    while stack:
        path = stack.pop()
        best = min(best, path, key=lambda p: (-len(p), p[-1]))
        stack += [path + [i] for i in range(len(tokens)) if i and parents[i] == path[-1] and tokens[i] == picks[path[-1]]]
    return best


def test_the_longer_branch_of_two_equal_siblings():
    # nodes 1 and 2 hold the same right token; only node 2 has a draft behind it, and that is right too
    assert longest_path([5, 7, 7, 9], [-1, 0, 0, 2], [7, 9, 9, 4]) == [0, 2, 3]
    # of two paths of one length the one that ends at the lower node
    assert longest_path([5, 7, 7], [-1, 0, 0], [7, 1, 1]) == [0, 1]


def test_paths_of_one_node():
    assert longest_path([5], [-1], [8]) == [0]
    assert longest_path([5, 6, 7], [-1, 0, 1], [8, 7, 0]) == [0]  # node 2 is right behind a wrong node


@pytest.mark.parametrize("seed", range(50))
def test_against_a_search(seed):
    rng = random.Random(seed)
    n = rng.randint(1, 24)
    tokens = [rng.randint(0, 2) for _ in range(n)]
    parents = [-1] + [rng.randint(max(0, i - 4), i - 1) for i in range(1, n)]
    picks = [rng.randint(0, 2) for _ in range(n)]
    assert longest_path(tokens, parents, picks) == _by_search(tokens, parents, picks)
