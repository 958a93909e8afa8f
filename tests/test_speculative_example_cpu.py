"""The n-gram draft trees of examples/speculative_decode.py."""
import importlib.util
import os

import numpy as np
import pytest

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_decode.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def paths(tokens, parents):
    out = []
    for i in range(1, len(tokens)):
        p, j = [], i
        while j > 0:
            p.append(tokens[j])
            j = parents[j]
        out.append(tuple(p[::-1]))
    return out


def test_no_earlier_place_gives_a_bare_root(example):
    assert example.ngram_tree([1, 2, 3], 8) == ([3], [-1])
    assert example.ngram_tree([3], 8) == ([3], [-1])


def test_the_longest_shared_context_comes_first(example):
    h = [5, 1, 2, 7, 9, 2, 8, 4, 1, 2]
    tokens, parents = example.ngram_tree(h, 8, depth=2)
    assert (tokens, parents) == ([2, 7, 9, 8, 4], [-1, 0, 1, 0, 3])


@pytest.mark.parametrize("n_nodes", [1, 2, 7, 16])
def test_trees_are_well_formed(example, n_nodes):
    rng = np.random.default_rng(n_nodes)
    for length in (1, 2, 5, 40, 200):
        h = rng.integers(0, 6, length).tolist()
        tokens, parents = example.ngram_tree(h, n_nodes)
        assert 1 <= len(tokens) == len(parents) <= n_nodes and tokens[0] == h[-1] and parents[0] == -1
        assert all(0 <= p < i for i, p in enumerate(parents) if i)
        ps = paths(tokens, parents)
        assert len(set(ps)) == len(ps) and all(len(p) <= example.DRAFT_DEPTH for p in ps)
        for p in ps:  # each path followed the root's token before
            assert any(tuple(h[i:i + len(p) + 1]) == (h[-1], *p) for i in range(len(h)))
