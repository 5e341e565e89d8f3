"""``tree_next_tokens``: the successors of every token in DFS order, against a
walk over every root-to-leaf path."""
import random

import numpy as np
import pytest

from tree_training_b200 import TreeNode, tree_next_tokens


def forest(seed):
    rng = random.Random(seed)

    def node(depth):
        n = TreeNode([rng.randrange(1000) for _ in range(rng.choice([0, 1, 1, 2, 5]))])
        if depth < 4:
            n.children = [node(depth + 1) for _ in range(rng.choice([0, 1, 2, 3]))]
        return n
    return [node(0) for _ in range(rng.randint(1, 3))]


def walk(roots):
    """Per token in DFS order: the tokens that follow it, in the order of the
    branches."""
    out, at = [], {}

    def first(n):
        return [n.token_ids[0]] if n.token_ids else [t for c in n.children for t in first(c)]

    def go(n):
        for i, _ in enumerate(n.token_ids):
            out.append([n.token_ids[i + 1]] if i + 1 < len(n.token_ids)
                       else [t for c in n.children for t in first(c)])
        for c in n.children:
            go(c)
    for r in roots:
        go(r)
    return out


@pytest.mark.parametrize("seed", range(12))
def test_successors(seed):
    roots = forest(seed)
    want = walk(roots)
    got = tree_next_tokens(roots, ignore=-7)
    assert got.dtype == np.int64 and got.shape[0] == len(want)
    assert got.shape[1] == max([1] + [len(w) for w in want])
    for row, w in zip(got, want):
        assert row[:len(w)].tolist() == w and (row[len(w):] == -7).all()


def test_a_chain_and_an_empty_forest():
    assert tree_next_tokens([TreeNode([5, 6, 7])]).tolist() == [[6], [7], [-100]]
    assert tree_next_tokens([]).shape == (0, 1)
    assert tree_next_tokens([TreeNode([])]).shape == (0, 1)
