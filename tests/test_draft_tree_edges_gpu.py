"""Drafted trees at the edges of what a call allows, against the plain implementations in 64 bits (tests/plain_tree.py)."""
import random

import pytest

import plain_tree
from test_draft_tree_gpu import ints, ops, random_tree  # noqa: F401

pytestmark = pytest.mark.gpu

# -- step maps ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("most", [1, 5, 64, 65, 130, 256])
def test_step_maps_of_portions_in_maps_made_for_trees(ops, most):  # noqa: F811
    """A portion is a tree whose nodes follow one another: behind a step of trees, the same maps have a chain's ancestors, not the trees' still."""
    rng = random.Random(most)
    B, R, page, blocks = 5, 6, 16, 30
    n_new, lengths = [most] + [rng.randint(0, most) for _ in range(B - 1)], [rng.randint(0, 200) for _ in range(R)]
    pages = [[rng.randrange(50) for _ in range(blocks)] for _ in range(R)]
    tokens = sum(n_new) + 3
    parents = [p for n in n_new for p in random_tree(n, rng)] + [0] * 3
    chain = [p for n in n_new for p in range(-1, n - 1)] + [0] * 3
    rows = rng.sample(range(R), B)
    maps = ops.StepMaps(B, tokens, blocks, most, tree=True)
    for parents_of in (parents, None, parents):
        ops.step_maps(maps, ints(rows), ints(n_new), ints(lengths), ints(pages), page, 50, None if parents_of is None else ints(parents_of))
        want = plain_tree.step_maps(rows, n_new, lengths, pages, page, 50, tokens, blocks, most, parents_of)
        if parents_of is None:
            want["ancestors"] = plain_tree.step_maps(rows, n_new, lengths, pages, page, 50, tokens, blocks, most, chain)["ancestors"]
        for name, value in want.items():
            assert getattr(maps, name).tolist() == value, name
