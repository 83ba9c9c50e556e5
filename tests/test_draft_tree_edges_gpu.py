"""Drafted trees at the edges of what a call allows: maps used for trees and portions in turn, values and scores that are not finite or next to it, positions and
lengths below zero, one request in several sequences; against the plain implementations in 64 bits (tests/plain_tree.py)."""
import math
import random

import pytest
import torch

import plain_tree
from test_draft_tree_gpu import DEV, DTYPES, WAYS, Case, ints, ops, random_tree  # noqa: F401

pytestmark = pytest.mark.gpu

LN2 = math.log(2.0)        # as the scale: scores are powers of two


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


# -- attention ----------------------------------------------------------------------------------------------------------------
def one_column_case(dtype, cached, nodes, H, Hkv, dim, page, **more):
    """Scores are the keys' first column in powers of two: all zero at first."""
    c = Case(dtype, cached, nodes, H, Hkv, dim, page, scale=LN2, **more)
    kv = Hkv * dim
    c.qkv[:, :-2 * kv] = 0.0
    c.qkv[:, 0:H * dim:dim] = 1.0
    c.qkv[:, H * dim:H * dim + kv:dim] = 0.0
    c.k_pages[:, 0:kv:dim] = 0.0
    return c


def way_case(dtype, seqs, Hkv, group, most, dim):
    rng = random.Random(most * dim + seqs)
    cached, nodes = [rng.choice([0, 1, 63, 64, 130, 257, 600]) for _ in range(seqs)], [most] + [rng.randint(0, 3) for _ in range(seqs - 1)]
    return one_column_case(dtype, cached, nodes, Hkv * group, Hkv, dim, rng.choice([1, 7, 16, 64]), seed=most + dim, extra_rows=1)


def same_with_what_is_not_finite(c, got):
    want, bound = c.want()
    rows = c.cu_q[-1]
    got = got.double().cpu()[:rows]
    want, bound = want[:rows], bound[:rows]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    odd = torch.isinf(want) | torch.isinf(got)
    assert torch.equal(got[odd], want[odd])
    plain = torch.isfinite(want)
    assert ((got - want).abs()[plain] <= bound[plain]).all()
    return want


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype,seqs,Hkv,group,most,dim,hint", WAYS)
def test_tree_attention_of_a_seen_value_that_is_not_finite_and_weighs_nothing(ops, dtype, seqs, Hkv, group, most, dim, hint, value):  # noqa: F811
    """Zero times infinity wherever the key lies: in a tile that all rows see in full or one of pages, nodes or ends that they do not."""
    c = way_case(dtype, seqs, Hkv, group, most, dim)
    for b in range(seqs):
        key, column = (slice(c.H * dim, c.H * dim + Hkv * dim, dim), slice(c.H * dim + Hkv * dim + 1, None, dim)), slice(1, None, dim)
        for at in {0, c.cached[b] // 2, c.cached[b] - 1} if c.cached[b] > 0 and b % 2 == 0 else ():
            row = c.tables[b][at // c.page] * c.page + at % c.page
            c.k_pages[row, 0::dim], c.v_pages[row, column] = -4096.0, value
        if c.nodes[b] > 0 and b % 2 == 1:
            c.qkv[c.cu_q[b], key[0]], c.qkv[c.cu_q[b], key[1]] = -4096.0, value
    want = same_with_what_is_not_finite(c, c.call(ops, c.device(), max_cached=hint))
    assert torch.isnan(want[:, 1]).any() and torch.isfinite(want[:, 0]).all()


@pytest.mark.parametrize("dtype,seqs,Hkv,group,most,dim,hint", WAYS)
def test_tree_attention_of_large_values_whose_keys_come_late(ops, dtype, seqs, Hkv, group, most, dim, hint):  # noqa: F811
    """The nodes' scores lie 7 (in powers of two) above those of the cache, the values of some nodes at a tenth of the largest number: what is added up stays below the
    type's largest, as with weights of at most one."""
    c = way_case(dtype, seqs, Hkv, group, most, dim)
    kv = Hkv * dim
    c.qkv[:, c.H * dim:c.H * dim + kv:dim] = 7.0
    for b in range(seqs):
        if c.nodes[b] > 0:
            c.qkv[c.cu_q[b], -kv:] = 3e37 * c.qkv[c.cu_q[b], -kv:].sign()
    c.check(c.call(ops, c.device(), max_cached=hint))


@pytest.mark.parametrize("dtype,seqs,Hkv,group,most,dim,hint", WAYS)
def test_tree_attention_of_keys_that_all_score_minus_infinity(ops, dtype, seqs, Hkv, group, most, dim, hint):  # noqa: F811
    """No weights can be found: NaN, as the formula has it; zeros are for rows that see nothing."""
    c = way_case(dtype, seqs, Hkv, group, most, dim)
    c.qkv[:, c.H * dim:c.H * dim + Hkv * dim:dim] = -math.inf
    c.k_pages[:, 0::dim] = -math.inf
    rng = random.Random(most)
    c.ancestors = [[0] * c.words if rng.random() < 0.4 else a for a in c.ancestors]
    for b in range(seqs):                 # (one sequence's pages are none, and a cache of one finite key)
        if b % 4 == 1:
            c.tables[b] = [-1] * len(c.tables[b])
        if b % 4 == 2 and c.cached[b] > 0:
            at = c.cached[b] // 3
            c.k_pages[c.tables[b][at // c.page] * c.page + at % c.page, 0::dim] = 3.0
    same_with_what_is_not_finite(c, c.call(ops, c.device(), max_cached=hint))
    c.window, c.positions = 5, [p + 3 for p in c.positions]
    same_with_what_is_not_finite(c, c.call(ops, c.device(), max_cached=hint))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_of_scores_next_to_the_least_number(ops, dtype):  # noqa: F811
    """Finite scores below all that a running maximum may begin with."""
    c = one_column_case(dtype, [40, 0], [6, 5], 2, 1, 32, 8, seed=3)
    c.qkv[:, 64:96:32] = -3.3e38
    c.k_pages[:, 0::32] = -3.3e38
    # (the scores are equal, so that the result is the mean of the values; their products' own error is as large as they are)
    got = c.call(ops, c.device()).double().cpu()
    c.qkv[:, 64:96:32], c.k_pages[:, 0::32] = 0.0, 0.0
    want, bound = c.want()
    assert ((got - want).abs() <= bound)[:11].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_of_positions_below_zero_and_the_widest_window(ops, dtype):  # noqa: F811
    c = Case(dtype, [100, 30], [9, 20], 4, 2, 64, 16, seed=5, window=2 ** 31 - 1)
    c.positions = [p - 200 for p in c.positions]
    c.check(c.call(ops, c.device()))


# -- acceptance ---------------------------------------------------------------------------------------------------------------
def accept(ops, choices, ids, parents, cu_q, cached, tables, page, n_pages, most, lengths, rows=None):  # noqa: F811
    B, T = len(cached), len(choices)
    kept, following, slots, path = ints([9] * B), ints([9] * B), ints([9] * T), torch.full((B, most), 9, dtype=torch.int32, device=DEV)
    ops.tree_accept(ints(choices), ints(ids), ints(parents), ints(cu_q), ints(cached), ints(tables), page, n_pages, kept, path, following, slots, lengths=lengths,
                    rows=None if rows is None else ints(rows))
    return [x.tolist() for x in (kept, path, following, slots)]


def test_tree_accept_takes_lengths_that_are_none_as_none(ops):  # noqa: F811
    """A cached length below zero is none, as step maps and attention take it; one near the largest number leaves room for the nodes, as step maps have it."""
    n, most = 6, 6
    chain, tables, lengths = [-1] + list(range(n - 1)), [[3, 1]] * 3, ints([-7] * 3)
    got = accept(ops, [4] * (3 * n), [4] * (3 * n), chain * 3, [0, n, 2 * n, 3 * n], [-3, 2, 2 ** 31 - 1], tables, 4, 9, most, lengths)
    want = plain_tree.accept([4] * (3 * n), [4] * (3 * n), chain * 3, [0, n, 2 * n, 3 * n], [0, 2, 2 ** 31 - 1], tables, 4, 9, most)
    assert got == list(want)
    assert lengths.tolist() == [6, 8, 2 ** 31 - 1]      # (the last: room for six nodes, all kept)


def test_tree_accept_of_one_request_in_several_sequences_gives_page_rows_to_the_last(ops):  # noqa: F811
    """Two sequences' keys in one row of the pages would be those that arrive last: the sequence whose length counts has them, the others' nodes go nowhere."""
    B, n, R = 130, 3, 7
    rng = random.Random(1)
    rows = [rng.randrange(-1, R + 1) for _ in range(B)]
    cached, tables = [rng.randint(0, 40) for _ in range(B)], [[rng.randrange(20) for _ in range(4)] for _ in range(B)]
    choices, ids, parents, cu_q = [4] * (B * n), [rng.choice([4, 5]) for _ in range(B * n)], [-1, 0, 1] * B, list(range(0, B * n + 1, n))
    lengths = ints([-7] * R)
    got = accept(ops, choices, ids, parents, cu_q, cached, tables, 16, 20, n, lengths, rows)
    want = list(plain_tree.accept(choices, ids, parents, cu_q, cached, tables, 16, 20, n))
    last = {r: b for b, r in enumerate(rows)}
    for b, r in enumerate(rows):
        if 0 <= r < R and last[r] != b:
            want[3][b * n:(b + 1) * n] = [-1] * n
    assert got == want
    assert lengths.tolist() == [cached[last[r]] + want[0][last[r]] if r in last else -7 for r in range(R)]


def test_tree_accept_of_rows_in_front_of_the_first_sequence(ops):  # noqa: F811
    """Rows of no sequence go nowhere, in front of the first sequence as behind the last."""
    T, cu_q = 300, [170, 172, 175]
    parents, tables, lengths = [-1] * T, [[1, 2], [3, 4]], ints([0, 0])
    for b in (0, 1):
        for i in range(1, cu_q[b + 1] - cu_q[b]):
            parents[cu_q[b] + i] = i - 1
    args = [4] * T, [4] * T, parents, cu_q, [3, 5], tables, 4, 9, 3
    assert accept(ops, *args, lengths) == list(plain_tree.accept(*args))
    assert lengths.tolist() == [5, 8]


@pytest.mark.parametrize("dtype,seqs,Hkv,group,most,dim,hint", WAYS)
def test_tree_attention_of_an_infinite_value_whose_key_scores_minus_infinity(ops, dtype, seqs, Hkv, group, most, dim, hint):  # noqa: F811
    """Zero times infinity too where all keys that a part of the call looks at score so: every key but the nodes' and the first of the cache."""
    c = way_case(dtype, seqs, Hkv, group, most, dim)
    for b in range(seqs):
        for at in range(1, c.cached[b]):
            c.k_pages[c.tables[b][at // c.page] * c.page + at % c.page, 0::dim] = -math.inf
        if c.cached[b] > 1 and b % 2 == 0:
            at = 1 + (7 * b + 40) % (c.cached[b] - 1)
            c.v_pages[c.tables[b][at // c.page] * c.page + at % c.page, 1::dim] = math.inf
    want = same_with_what_is_not_finite(c, c.call(ops, c.device(), max_cached=hint))
    assert torch.isfinite(want[:, 0]).all()
