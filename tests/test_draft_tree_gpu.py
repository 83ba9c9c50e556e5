"""The step over trees of drafted tokens: step_maps, rotary, tree_attention and tree_accept against their plain implementations in 64
bits (tests/plain_tree.py), and a run of them together against the same model token by token."""
import math
import random

import pytest
import torch

import plain_tree

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}       # half a step of the type


@pytest.fixture(scope="module")
def ops():
    from mini_llm_amd.kernels import ops as o
    return o


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def random_tree(n, rng):
    reach = rng.choice([1, 3, n])
    return [-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, n)] if n else []


# -- step maps ----------------------------------------------------------------------------------------------------------------
def check_maps(ops, rows, n_new, lengths, pages, page_size, n_pages, tokens, max_blocks, max_new, parents, stride=0):
    maps = ops.StepMaps(len(n_new), tokens, max_blocks, max_new, tree=parents is not None)
    for name in ("cu_q", "cached", "ctx_len", "token_seq", "positions", "slots", "block_tables"):
        getattr(maps, name).fill_(-77)
    table = torch.full((len(lengths), len(pages[0]) + stride), 12345, dtype=torch.int32, device=DEV)[:, :len(pages[0])]
    table.copy_(ints(pages))
    ops.step_maps(maps, None if rows is None else ints(rows), ints(n_new), ints(lengths), table, page_size, n_pages, None if parents is None else ints(parents))
    want = plain_tree.step_maps(rows, n_new, lengths, pages, page_size, n_pages, tokens, max_blocks, max_new, parents)
    for name, value in want.items():
        if name != "ancestors" or parents is not None:
            assert getattr(maps, name).tolist() == value, name
    return maps


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("B,R,most,page,longest,spare,stride", [(1, 1, 1, 16, 0, 0, 0), (1, 3, 1, 1, 5, 0, 1), (3, 3, 16, 16, 100, 5, 0), (7, 9, 64, 24, 1000, 3, 3),
                                                                (5, 5, 65, 8, 777, 0, 1), (4, 6, 256, 16, 40000, 40, 2), (300, 301, 5, 64, 5000, 9, 0),
                                                                (2, 2, 200, 7, 20000, 1, 0), (20, 20, 129, 1, 3000, 0, 0)])
def test_step_maps(ops, tree, B, R, most, page, longest, spare, stride):
    rng = random.Random(B * 1000 + most)
    rows = rng.sample(range(R), B) if R > B or rng.random() < 0.5 else None
    n_new = [rng.randint(0, most) for _ in range(B)]
    n_new[rng.randrange(B)] = most
    lengths = [rng.randint(0, longest) for _ in range(R)]
    blocks = -(-(longest + most) // page)
    n_pages = max(2, min(R * blocks, 1 << 24))
    pages = [[rng.randrange(n_pages) for _ in range(blocks + 2)] for _ in range(R)]
    parents = [p for n in n_new for p in random_tree(n, rng)] + [rng.randint(-5, 300) for _ in range(spare)] if tree else None
    check_maps(ops, rows, n_new, lengths, pages, page, n_pages, max(1, sum(n_new) + spare), blocks, most, (parents or [0]) if tree else None, stride)


def test_step_maps_of_long_portions(ops):
    check_maps(ops, [1, 0], [5000, 1], [3, 700], [[(7 * i) % 400 for i in range(400)], [(11 * i) % 400 for i in range(400)]], 16, 400, 5003, 400, 5000, None)


@pytest.mark.parametrize("tree", [False, True])
def test_step_maps_takes_what_names_nothing_as_none(ops, tree):
    """Rows outside the requests, counts below zero and above the limits, lengths below zero, pages outside the pool, positions behind
    the table, parents behind their children."""
    rows, n_new, lengths = [2, -1, 0, 7, 1, 2], [3, 4, -2, 5, 9, 9], [30, -4, 61]
    pages = [[1, 2, 3, 4], [5, 99, -1, 0], [7, 8, -3, 2 ** 31 - 1]]
    parents = [-1, 0, 5, -9, 0, 1, 2, 3, 300, 1, 0] if tree else None
    check_maps(ops, rows, n_new, lengths, pages, 16, 20, 11, 4, 6, parents)
    check_maps(ops, rows, n_new, lengths, pages, 16, 20, 2, 3, 6, parents[:2] if tree else None)


# -- rotary -------------------------------------------------------------------------------------------------------------------
SCALINGS = [None, dict(kind="linear", factor=4.0), dict(kind="base", factor=8.0), dict(kind="by_turns", factor=8.0, original=4096, fast=32.0, slow=1.0),
            dict(kind="by_pair", factor=32.0, original=4096, fast=32.0, slow=1.0)]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["kind"] if s else "plain")
@pytest.mark.parametrize("rot", [4, 18, 32, 128])
def test_rotary_freqs(ops, scaling, rot):
    got = ops.rotary_freqs(rot, 10000.0, scaling, device="cpu")
    want = plain_tree.frequencies(rot, 10000.0, scaling)
    shares = torch.tensor([(x % 2 ** 64) * 2.0 ** -64 for x in got.tolist()], dtype=torch.float64) * 2 * math.pi
    # a power, a quotient and a mixture in 64 bits on either side, of numbers up to 1: 2^-48 is 32 roundings
    assert (shares - want).abs().max() <= 2.0 ** -48


def check_rotary(ops, dtype, T, H, dim, rot, interleaved, positions, amplitude=1.0, in_place=False, scaling=None, shift=0, pad=0):
    g = torch.Generator().manual_seed(T * 100 + dim + rot)
    data = torch.randn(T, H * dim + pad + shift, generator=g).to(dtype)
    buf = data.to(DEV)
    x = buf[:, shift:shift + H * dim]
    out = x if in_place else torch.full((T, H * dim + pad), 7.0, dtype=dtype, device=DEV)[:, :H * dim]
    freqs = plain_tree.frequencies(rot, 10000.0, scaling)
    assert ops.rotary(x, ints(positions), ops.rotary_freqs(rot, 10000.0, scaling), H, dim, out, interleaved=interleaved, amplitude=amplitude) is out
    src = data[:, shift:shift + H * dim]
    want, size, first, second = plain_tree.rotary(src, torch.tensor(positions), freqs, H, dim, interleaved, amplitude)
    # Of each coefficient: the angle's share of a turn 2 pi 2^-33 and its frequency |p| 2 pi 2^-65, its float and the constant's (0.79 rad, half a step each), the
    # series (2e-9), four roundings in it and one by the amplitude: under 8 half steps. Then two products and a sum, then the type's rounding.
    angle = 1e-9 + max(abs(p) for p in positions) * 2.0 ** -53
    got = out.double().cpu().view(T, H, dim)
    turned = torch.zeros(dim, dtype=torch.bool)
    bound = torch.zeros(T, H, dim, dtype=torch.float64)
    for cols in (first, second):
        turned[cols] = True
        bound[..., cols] = size * (10 * 2.0 ** -24 + angle)
    want = want.view(T, H, dim)
    if dtype == torch.bfloat16:
        bound = bound + (want.abs() + bound) * HALF[dtype]
    assert ((got - want).abs() <= bound).all()
    assert torch.equal(got[..., ~turned], src.double().view(T, H, dim)[..., ~turned])
    rest = buf.cpu()
    assert torch.equal(rest[:, :shift], data[:, :shift]) and torch.equal(rest[:, shift + H * dim:], data[:, shift + H * dim:])
    if not in_place:
        assert torch.equal(rest, data)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T,H,dim,rot", [(1, 1, 2, 2), (1, 12, 64, 64), (5, 3, 96, 32), (7, 5, 80, 80), (3, 2, 64, 18), (33, 40, 128, 128), (2, 3, 30, 10), (200, 18, 96, 32), (4, 1, 256, 256)])
def test_rotary(ops, dtype, interleaved, in_place, T, H, dim, rot):
    rng = random.Random(T)
    check_rotary(ops, dtype, T, H, dim, rot, interleaved, [rng.randint(0, 5000) for _ in range(T)], in_place=in_place)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shift,pad", [(0, 16), (8, 24), (1, 0), (3, 2)])
def test_rotary_of_columns_of_wider_rows(ops, dtype, interleaved, shift, pad):
    check_rotary(ops, dtype, 9, 4, 64, 48, interleaved, list(range(9)), in_place=True, shift=shift, pad=pad)
    check_rotary(ops, dtype, 9, 4, 64, 48, interleaved, list(range(9)), shift=shift, pad=pad)


@pytest.mark.parametrize("scaling", SCALINGS[1:], ids=lambda s: s["kind"])
def test_rotary_far_positions_and_scalings(ops, scaling):
    positions = [0, 1, -1, 2 ** 24 + 1, 10 ** 6, 131071, 3, 2 ** 31 - 1, -2 ** 31]
    check_rotary(ops, torch.float32, 9, 2, 64, 64, False, positions, amplitude=1.2, scaling=scaling)
    check_rotary(ops, torch.bfloat16, 9, 2, 64, 32, True, positions, amplitude=0.9, scaling=scaling)


# -- attention ----------------------------------------------------------------------------------------------------------------
class Case:
    """Inputs of one call on the CPU, and the call."""

    def __init__(self, dtype, cached, nodes, H, Hkv, dim, page, seed=0, window=0, extra_rows=0, scale=None, std=1.0):
        g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
        self.dtype, self.H, self.Hkv, self.dim, self.page, self.window = dtype, H, Hkv, dim, page, window
        self.cached, self.nodes, self.scale = cached, nodes, dim ** -0.5 if scale is None else scale
        self.cu_q = [sum(nodes[:b]) for b in range(len(nodes) + 1)]
        self.T = T = self.cu_q[-1] + extra_rows
        blocks = [max(1, -(-(c + n) // page)) for c, n in zip(cached, nodes)]
        self.n_pages = sum(blocks) + 3
        order = rng.sample(range(1, self.n_pages), self.n_pages - 1)      # (page 0 stands behind the tables' ends)
        self.tables = []
        for n in blocks:
            self.tables.append([order.pop() for _ in range(n)] + [0] * (max(blocks) - n))
        kv = Hkv * dim
        self.k_pages, self.v_pages = (torch.randn(self.n_pages * page, kv, generator=g).to(dtype) for _ in range(2))
        self.qkv = (torch.randn(T, H * dim + 2 * kv, generator=g) * std).to(dtype)
        self.parents = [random_tree(n, rng) for n in nodes]
        self.words = (max(max(nodes), 1) + 63) // 64
        maps = plain_tree.step_maps(None, nodes, cached, self.tables, page, self.n_pages, max(T, 1), max(blocks), max(max(nodes), 1), [p for t in self.parents for p in t])
        self.positions, self.ancestors = maps["positions"][:T], maps["ancestors"][:T]

    def split(self):
        kv = self.Hkv * self.dim
        return self.qkv[:, :-2 * kv], self.qkv[:, -2 * kv:-kv], self.qkv[:, -kv:]

    def device(self):
        kv = self.Hkv * self.dim
        qkv = self.qkv.to(DEV)
        return dict(q=qkv[:, :-2 * kv], k=qkv[:, -2 * kv:-kv], v=qkv[:, -kv:], k_pages=self.k_pages.to(DEV), v_pages=self.v_pages.to(DEV), block_tables=ints(self.tables),
                    cached=ints(self.cached), cu_q=ints(self.cu_q), ancestors=torch.tensor(self.ancestors, dtype=torch.int64, device=DEV),
                    positions=ints(self.positions), out=torch.full((self.T, self.H * self.dim), 55.0, dtype=self.dtype, device=DEV))

    def call(self, ops, d, max_cached=None):
        return ops.tree_attention(d["q"], d["k"], d["v"], self.H, self.Hkv, self.dim, d["k_pages"], d["v_pages"], self.page, d["block_tables"], d["cached"],
                                  d["cu_q"], d["ancestors"], d["positions"], self.scale, d["out"], max_new=max(max(self.nodes), 1),
                                  max_cached=max(self.cached) if max_cached is None else max_cached, window=self.window)

    def want(self):
        q, k, v = self.split()
        out, spread, top, mass = plain_tree.attention(q, k, v, self.H, self.Hkv, self.dim, self.k_pages, self.v_pages, self.page, self.tables, self.cached, self.cu_q,
                                                      self.ancestors, self.positions, self.scale, self.window)
        # A score: dim fused additions and the scale, each off by 2^-24 of at most the sum of their sizes. Its exponential: that much relative,
        # plus the difference to the maximum (a rounding of a number up to twice the largest score) and two steps of the function. The sums: a rounding a key,
        # of at most the largest value. Each is in the numerator and the denominator.
        keys = max(self.cached) + max(max(self.nodes), 1)
        score = (self.dim + 2) * 2.0 ** -24 * mass + 3 * mass * 2.0 ** -24 + 2 ** -22
        bound = 2 * top * score + 2 * top * (keys + 8) * 2.0 ** -24
        if self.dtype == torch.bfloat16:
            # the weights and the result are rounded once each; the bare hardware exponential is off by 2^-22 of its value at most
            bound = bound + (spread + out.abs()) * HALF[self.dtype] + 2 * top * 2.0 ** -21
        return out, bound

    def check(self, got):
        want, bound = self.want()
        rows = self.cu_q[-1]
        got = got.double().cpu()
        assert torch.isfinite(got[:rows]).all()
        assert ((got - want).abs()[:rows] <= bound[:rows]).all(), ((got - want).abs()[:rows] / bound[:rows].clamp(min=1e-30)).max()
        assert (got[rows:] == 55.0).all()


SIZES = [([0], [1], 1, 1, 8, 16), ([5], [1], 2, 2, 16, 16), ([1], [3], 4, 1, 32, 1), ([31], [2], 2, 2, 64, 16), ([32], [17], 3, 3, 64, 32), ([33, 0, 64], [16, 5, 1], 2, 1, 64, 8),
         ([500], [26], 12, 12, 64, 16), ([70, 3, 200, 0], [9, 1, 33, 64], 4, 2, 128, 24), ([100, 90], [65, 3], 2, 1, 80, 7), ([257], [130], 2, 1, 48, 64), ([40], [256], 1, 1, 96, 16),
         ([300, 20], [7, 12], 7, 1, 256, 16), ([64], [40], 8, 1, 40, 16), ([95, 97], [31, 33], 2, 2, 24, 16), ([129], [20], 4, 4, 160, 32), ([65, 66], [16, 15], 3, 1, 192, 16), ([1200], [4], 4, 2, 72, 256),
         ([128], [64], 4, 2, 112, 16), ([60, 61, 62], [0, 2, 0], 2, 2, 64, 16), ([50], [90], 5, 5, 224, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cached,nodes,H,Hkv,dim,page", SIZES)
def test_tree_attention(ops, dtype, cached, nodes, H, Hkv, dim, page):
    c = Case(dtype, cached, nodes, H, Hkv, dim, page, seed=dim + len(cached))
    c.check(c.call(ops, c.device()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 15, 33, 100, 1000])
def test_tree_attention_window(ops, dtype, window):
    c = Case(dtype, [150, 0, 40], [21, 70, 3], 4, 2, 64, 24, seed=window, window=window)
    c.check(c.call(ops, c.device()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_of_long_contexts(ops, dtype):
    c = Case(dtype, [9000, 4500, 1], [5, 2, 1], 2, 1, 64, 16, seed=4)
    c.check(c.call(ops, c.device()))
    c = Case(dtype, [6000], [40], 4, 1, 128, 64, seed=5, window=5000)
    c.check(c.call(ops, c.device()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hint", [0, 10, 400, 100000])
def test_tree_attention_is_right_whatever_longest_cache_it_is_told(ops, dtype, hint):
    c = Case(dtype, [400, 33], [19, 5], 4, 2, 64, 16, seed=6)
    c.check(c.call(ops, c.device(), max_cached=hint))


F32, BF16 = torch.float32, torch.bfloat16
WAYS = [(F32, 8, 9, 3, 11, 16, 13500), (F32, 7, 1, 1, 17, 16, 12990), (F32, 8, 9, 5, 39, 16, 13719), (F32, 8, 1, 5, 13, 16, 14134), (F32, 8, 9, 4, 9, 64, 30013), (F32, 8, 1, 1, 17, 64, 26878),
        (F32, 8, 5, 7, 55, 64, 15668), (F32, 8, 1, 5, 13, 64, 17465), (F32, 6, 1, 1, 17, 96, 13968), (F32, 8, 9, 2, 49, 96, 17738), (F32, 7, 1, 3, 11, 96, 28560), (F32, 3, 1, 1, 17, 200, 21231),
        (F32, 7, 1, 3, 11, 200, 7632), (BF16, 8, 9, 3, 11, 16, 14426), (BF16, 8, 1, 1, 17, 16, 22620), (BF16, 8, 9, 5, 26, 16, 10698), (BF16, 8, 1, 5, 13, 16, 23888), (BF16, 7, 1, 3, 11, 64, 20672),
        (BF16, 5, 1, 1, 17, 64, 26912), (BF16, 8, 9, 3, 43, 64, 28923), (BF16, 6, 1, 5, 13, 64, 25474), (BF16, 7, 1, 1, 17, 96, 22611), (BF16, 7, 1, 3, 11, 96, 11395), (BF16, 8, 9, 5, 27, 96, 27689),
        (BF16, 7, 1, 5, 13, 96, 18633), (BF16, 6, 1, 1, 17, 200, 25666), (BF16, 6, 1, 3, 11, 200, 3984),
        (F32, 8, 5, 7, 55, 16, 28308), (F32, 8, 10, 3, 11, 64, 21717), (BF16, 8, 10, 3, 43, 96, 27944)]


@pytest.mark.parametrize("dtype,seqs,Hkv,group,most,dim,hint", WAYS)
def test_tree_attention_in_every_way_of_sharing_it_out(ops, dtype, seqs, Hkv, group, most, dim, hint):
    """A case of every kernel that there is beside the smallest of each width, by the longest cache the call is told; the caches are short and ragged."""
    rng = random.Random(most * dim)
    cached, nodes = [rng.choice([0, 1, 63, 64, 65, 130, 257]) for _ in range(seqs)], [most] + [rng.randint(0, 3) for _ in range(seqs - 1)]
    c = Case(dtype, cached, nodes, Hkv * group, Hkv, dim, rng.choice([1, 8, 16, 24]), seed=most + dim, extra_rows=1)
    c.check(c.call(ops, c.device(), max_cached=hint))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_rows_that_see_nothing(ops, dtype):
    """Masks of any bits: rows without one and without a cache get zeros, rows without one and with a cache their cache alone."""
    c = Case(dtype, [0, 50], [70, 66], 4, 2, 64, 16, seed=7, extra_rows=5)
    rng = random.Random(8)
    c.ancestors = [[0, 0] if rng.random() < 0.3 else [rng.getrandbits(64) - 2 ** 63, rng.getrandbits(2)] for _ in range(c.T)]
    c.check(c.call(ops, c.device()))
    c.window, c.positions = 3, [p + 1000 for p in c.positions]     # (windows in front of which everything lies but the nodes)
    c.check(c.call(ops, c.device()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("window", [0, 20])
def test_tree_attention_of_bad_values_where_nothing_is_seen(ops, dtype, bad, window):
    """Unseen: pages' rows behind the cache, rows of no sequence, and nodes in nobody's path (whose own rows alone see them)."""
    c = Case(dtype, [45, 17], [37, 20], 4, 2, 64, 16, seed=9, window=window, extra_rows=4)
    own = [c.cu_q[0] + 36, c.cu_q[1] + 19]                 # the last nodes, which have no children
    kv = c.Hkv * c.dim
    for t in own + list(range(c.cu_q[-1], c.T)):
        c.qkv[t, -2 * kv:] = bad
    unseen = list(range(c.page))                           # page 0
    for b, cached in enumerate(c.cached):
        places = list(range(cached, len(c.tables[b]) * c.page)) + (list(range(max(0, cached - window + 1))) if window else [])
        unseen += [c.tables[b][at // c.page] * c.page + at % c.page for at in places]
    c.k_pages[unseen] = c.v_pages[unseen] = bad
    d = c.device()
    got = c.call(ops, d)
    rows = [t for t in range(c.cu_q[-1]) if t not in own]
    want, bound = c.want()
    got = got.double().cpu()
    assert torch.isfinite(got[rows]).all()
    assert ((got - want).abs()[rows] <= bound[rows]).all()
    if math.isnan(bad):
        assert torch.isnan(got[own]).all()
    assert (got[c.cu_q[-1]:] == 55.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_of_a_bad_value_that_some_rows_see(ops, dtype):
    """One infinite value of a node: in the rows that see it its column is infinite, in the others nothing changes."""
    c = Case(dtype, [30], [60], 2, 1, 64, 16, seed=10)
    clean = c.call(ops, c.device()).double().cpu()
    c.qkv[20, -64 + 5] = math.inf
    got = c.call(ops, c.device()).double().cpu()
    sees = torch.tensor([bool(a[0] >> 20 & 1) for a in c.ancestors])
    for h in range(2):
        assert (got[sees][:, 64 * h + 5] == math.inf).all()
        others = torch.ones(64, dtype=torch.bool)
        others[5] = False
        assert torch.equal(got[:, 64 * h:64 * h + 64][:, others], clean[:, 64 * h:64 * h + 64][:, others])
    assert torch.equal(got[~sees], clean[~sees])


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_of_pages_that_are_none(ops, dtype):
    """A table's entry outside the pool holds nothing that is seen; a cache longer than its table ends with it."""
    c = Case(dtype, [100, 64], [5, 40], 4, 2, 64, 16, seed=11)
    c.tables[0][2], c.tables[0][4], c.tables[1][0] = -1, c.n_pages, 2 ** 31 - 1
    c.check(c.call(ops, c.device()))
    c.cached = [5000, 64]
    c.check(c.call(ops, c.device()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("std,scale", [(30.0, 1.0), (1.0, 0.0), (1e-3, -4.0), (200.0, 0.125)])
def test_tree_attention_of_large_and_flat_scores(ops, dtype, std, scale):
    c = Case(dtype, [130, 20], [25, 9], 4, 2, 64, 16, seed=12, std=std, scale=scale)
    c.check(c.call(ops, c.device()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_of_scores_that_rise_along_the_cache(ops, dtype):
    """Every key beats the ones in front of it by far: each tile moves the maximum."""
    c = Case(dtype, [600], [18], 2, 1, 64, 16, seed=13, scale=1.0)
    c.qkv[:, :128] = 1.0
    for at in range(600):
        c.k_pages[c.tables[0][at // 16] * 16 + at % 16] = at / 64.0
    c.check(c.call(ops, c.device()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_beyond_32_bits(ops, dtype):
    """Pages whose elements lie more than 2^31 elements (and 2^32 bytes) from the pool's first."""
    c = Case(dtype, [70], [9], 4, 4, 128, 16, seed=14)
    kv, far = 512, (2 ** 31 // 512 + 4096) // 16
    d = c.device()
    big = {}
    for name in ("k_pages", "v_pages"):
        big[name] = torch.empty((far + 40) * 16, kv, dtype=dtype, device=DEV)
        for page in range(c.n_pages):
            big[name][(far + 2 * page) * 16:(far + 2 * page + 1) * 16] = d[name][page * 16:(page + 1) * 16]
    near = c.call(ops, d).clone()
    d.update(big, block_tables=ints([[far + 2 * p for p in row] for row in c.tables]))
    d["out"].fill_(55.0)
    assert torch.equal(c.call(ops, d), near)
    c.check(near)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cached,nodes,H,Hkv", [([5000, 300], [6, 3], 4, 2), ([200, 90], [33, 20], 8, 1)])
def test_tree_attention_streams_and_graphs(ops, dtype, cached, nodes, H, Hkv):
    """On another stream; twice the same bits; two captured graphs, replayed in turn with new inputs and with eager work between."""
    cases = [Case(dtype, cached, nodes, H, Hkv, 64, 16, seed=s) for s in (20, 21, 22)]
    data = [c.device() for c in cases]
    eager = [c.call(ops, d).clone() for c, d in zip(cases, data)]
    cases[0].check(eager[0])
    assert torch.equal(cases[0].call(ops, data[0]), eager[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = cases[1].call(ops, data[1]).clone()
    torch.cuda.synchronize()
    assert torch.equal(other, eager[1])
    graphs, places = [], [cases[0].device(), cases[1].device()]
    for place in places:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cases[0].call(ops, place)
        graphs.append(graph)
    order = [(0, 0), (1, 1), (0, 2), (1, 0), (0, 1)]
    for g, n in order:
        kv = Hkv * 64
        places[g]["q"]._base.copy_(cases[n].qkv)
        for name in ("k_pages", "v_pages", "block_tables", "ancestors", "positions"):
            places[g][name].copy_(data[n][name])
        places[g]["out"].fill_(55.0)
        torch.cuda.synchronize()
        graphs[g].replay()
        busy = cases[2].call(ops, data[2])
        torch.cuda.synchronize()
        assert torch.equal(places[g]["out"], eager[n]) and torch.equal(busy, eager[2])
    # both at once, on two streams
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for place in places:
            place["out"].fill_(55.0)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(places[0]["out"], eager[1]) and torch.equal(places[1]["out"], eager[0])


def test_tree_attention_of_one_node_is_decode_attention(ops):
    """A tree of one node beside paged_attention, which reads the token's own key from its pages."""
    c = Case(torch.float32, [300, 41, 7], [1, 1, 1], 4, 2, 64, 16, seed=23)
    d = c.device()
    got = c.call(ops, d)
    slots = ints([plain_tree.slot(c.tables[b], 99, 16, c.n_pages, c.cached[b]) for b in range(3)])
    out = torch.empty_like(got)
    ops.paged_attention(d["q"]._base, 0, 4, 2, 64, d["k_pages"], d["v_pages"], 16, d["block_tables"], ints([0, 1, 2]), d["cached"], c.scale, 0, out, max_q_len=1,
                        max_ctx_len=301, append=(256, 384, slots))
    want, bound = c.want()
    assert ((out - got).abs().double().cpu() <= 2 * bound).all()


# -- acceptance ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("most,page", [(1, 16), (5, 1), (26, 16), (64, 24), (65, 16), (200, 8), (256, 16)])
def test_tree_accept(ops, seed, most, page):
    rng = random.Random(seed * 1000 + most)
    B, spare = rng.choice([1, 3, 17]), rng.choice([0, 4])
    nodes = [rng.randint(0, most) for _ in range(B)]
    nodes[0] = most
    cached = [rng.randint(0, 500) for _ in range(B)]
    cu_q = [sum(nodes[:b]) for b in range(B + 1)]
    T, blocks = cu_q[-1] + spare, -(-(500 + most) // page)
    words = rng.choice([2, 5, 1000])                 # few tokens: siblings that carry the same one
    parents = [p for n in nodes for p in random_tree(n, rng)] + [0] * spare
    if seed % 4 == 3:                                # second roots, parents behind their children
        parents = [p if rng.random() < 0.9 else rng.randint(-3, 300) for p in parents]
        for b in range(B):
            for i in range(nodes[b]):
                p = parents[cu_q[b] + i]
                parents[cu_q[b] + i] = p if p < i else i + 1
    ids, choices = [rng.randrange(words) for _ in range(T)], [rng.randrange(words) for _ in range(T)]
    for b in range(B):
        for i in range(nodes[b]):
            p = parents[cu_q[b] + i]
            if 0 <= p < i and rng.random() < 0.7:
                choices[cu_q[b] + p] = ids[cu_q[b] + i]
    tables = [[rng.randrange(-1, 900) for _ in range(blocks)] for _ in range(B)]
    rows = rng.sample(range(B + 2), B) if seed % 2 else None
    if rows and seed % 3 == 0:
        rows[0] = -1
    kept, following, slots = ints([9] * B), ints([9] * B), ints([9] * T) if T else ints([9])
    if T == 0:
        return
    path, lengths = torch.full((B, most), 9, dtype=torch.int32, device=DEV), ints([-5] * (B + 2 if rows else B))
    for _ in range(2):
        ops.tree_accept(ints(choices), ints(ids), ints(parents), ints(cu_q), ints(cached), ints(tables), page, 900, kept, path, following, slots, lengths=lengths,
                        rows=None if rows is None else ints(rows))
    want = plain_tree.accept(choices, ids, parents, cu_q, cached, tables, page, 900, most)
    assert [kept.tolist(), path.tolist(), following.tolist(), slots.tolist()] == list(want)
    ends = [-5] * lengths.numel()
    for b in range(B):
        r = b if rows is None else rows[b]
        if r >= 0:
            ends[r] = cached[b] + want[0][b]
    assert lengths.tolist() == ends
    slots.fill_(9)
    ops.tree_accept(ints(choices), ints(ids), ints(parents), ints(cu_q), ints(cached), ints(tables), page, 900, kept, path, following, slots)
    assert slots.tolist() == want[3]


def test_tree_accept_of_a_chain_and_of_more_nodes_than_the_path_has_room_for(ops):
    n = 256
    args = [ints([7] * n), ints([7] * n), ints([-1] + list(range(n - 1))), ints([0, n]), ints([10]), ints([list(range(20))]), 16, 20]
    kept, path, following, slots = ints([0]), torch.empty(1, n, dtype=torch.int32, device=DEV), ints([0]), ints([0] * n)
    ops.tree_accept(*args, kept, path, following, slots)
    assert kept.tolist() == [n] and path.tolist() == [list(range(n))] and slots.tolist() == list(range(10, 10 + n)) and following.tolist() == [7]
    path = torch.empty(1, 5, dtype=torch.int32, device=DEV)
    ops.tree_accept(*args, kept, path, following, slots)
    assert kept.tolist() == [5] and path.tolist() == [[0, 1, 2, 3, 4]] and slots.tolist() == [10, 11, 12, 13, 14] + [-1] * (n - 5)


# -- together -----------------------------------------------------------------------------------------------------------------
class Model:
    """A small decoder of two layers on the package's own operations, with rotary positions and shared keys."""
    D, H, HKV, DIM, V, LAYERS, PAGE, BLOCKS, REQUESTS = 96, 6, 2, 16, 211, 2, 8, 12, 4

    def __init__(self, ops, dtype):
        self.ops, self.dtype = ops, dtype
        g = torch.Generator().manual_seed(1)
        w = lambda *s: (torch.randn(s, generator=g) * s[-1] ** -0.5).to(dtype).to(DEV)      # noqa: E731
        self.kv = self.HKV * self.DIM
        self.emb = (torch.randn(self.V, self.D, generator=g)).to(dtype).to(DEV)
        self.layers = [(w(self.D + 2 * self.kv, self.D), w(self.D, self.D), w(4 * self.D, self.D), w(self.D, 4 * self.D)) for _ in range(self.LAYERS)]
        self.head = w(self.V, self.D) * 4
        self.one = torch.ones(self.D, device=DEV)
        self.freqs = ops.rotary_freqs(self.DIM, 10000.0, SCALINGS[3])
        self.n_pages = self.REQUESTS * self.BLOCKS
        self.k_pages, self.v_pages = ([torch.zeros(self.n_pages * self.PAGE, self.kv, dtype=dtype, device=DEV) for _ in range(self.LAYERS)] for _ in range(2))
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        self.pages = order.view(self.REQUESTS, self.BLOCKS).to(DEV)
        self.lengths = torch.zeros(self.REQUESTS, dtype=torch.int32, device=DEV)

    def forward(self, ids, maps, tree, max_new, max_cached):
        """The token chosen at every row; the layers' rows of queries, keys and values (of a tree: not in the pages yet)."""
        o, T = self.ops, ids.numel()
        x = torch.empty(T, self.D, device=DEV)
        o.embed(ids, None, self.emb, None, x)
        rows = []
        for n, (wqkv, wo, w1, w2) in enumerate(self.layers):
            qkv = torch.empty(T, self.D + 2 * self.kv, dtype=self.dtype, device=DEV)
            o.ln_linear(x, self.one, None, 1e-5, wqkv, None, qkv)
            turned = qkv[:, :self.D + self.kv]
            o.rotary(turned, maps.positions, self.freqs, self.H + self.HKV, self.DIM, turned)
            att = torch.empty(T, self.D, dtype=self.dtype, device=DEV)
            if tree:
                o.tree_attention(qkv[:, :self.D], qkv[:, self.D:self.D + self.kv], qkv[:, self.D + self.kv:], self.H, self.HKV, self.DIM, self.k_pages[n], self.v_pages[n],
                                 self.PAGE, maps.block_tables, maps.cached, maps.cu_q, maps.ancestors, maps.positions, self.DIM ** -0.5, att, max_new=max_new,
                                 max_cached=max_cached)
            else:
                o.kv_append(qkv, self.D, self.D + self.kv, self.kv, self.k_pages[n], self.v_pages[n], maps.slots)
                o.paged_attention(qkv, 0, self.H, self.HKV, self.DIM, self.k_pages[n], self.v_pages[n], self.PAGE, maps.block_tables, maps.token_seq, maps.positions,
                                  self.DIM ** -0.5, 0, att, cu_q=maps.cu_q, ctx_len=maps.ctx_len, max_q_len=max_new, max_ctx_len=max_cached + max_new)
            o.linear(att, wo, None, x, "add_residual")
            h = torch.empty(T, 4 * self.D, dtype=self.dtype, device=DEV)
            o.ln_linear(x, self.one, None, 1e-5, w1, None, h, "gelu_tanh")
            o.linear(h, w2, None, x, "add_residual")
            rows.append(qkv)
        logits = torch.empty(T, self.V, device=DEV)
        o.ln_linear(x, self.one, None, 1e-5, self.head, None, logits, "store_f32")
        chosen = torch.empty(T, dtype=torch.int32, device=DEV)
        o.argmax(logits, chosen)
        return chosen, rows, logits


def test_tree_accept_of_one_request_twice(ops):
    """Of several sequences of one request the last one's length stands, whatever the order of arrival: 300 sequences of 7 requests."""
    B, R = 300, 7
    rows = [(5 * b + b // 11) % (R + 1) for b in range(B)]                     # (row R names nobody)
    cached = [10 * b for b in range(B)]
    kept, path, following, slots, lengths = (torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((B,), (B, 2), (B,), (B,), (R,)))
    for _ in range(3):
        lengths.fill_(-7)
        ops.tree_accept(ints([4] * B), ints([1] * B), ints([-1] * B), ints(range(B + 1)), ints(cached), ints([[3] * 200] * B), 16, 9, kept, path, following, slots, lengths, ints(rows))
        assert lengths.tolist() == [max(cached[b] for b in range(B) if rows[b] == r) + 1 for r in range(R)]
        assert kept.tolist() == [1] * B


def test_the_most_sequences_that_a_call_takes(ops):
    """65,536 sequences of one node: step maps (portions and trees), attention of nodes that see themselves alone, and paths of one node."""
    B, page, blocks = 65536, 4, 2
    n, at = torch.ones(B, dtype=torch.int32, device=DEV), torch.arange(B, dtype=torch.int32, device=DEV)
    lengths = at % 7
    pages = torch.stack([at, (at + 1) % B], 1).contiguous()
    rows = torch.flip(at, [0]).contiguous()
    for tree in (False, True):
        m = ops.StepMaps(B, B, blocks, 1, tree=tree)
        ops.step_maps(m, rows, n, lengths, pages, page, B, torch.full((B,), -1, dtype=torch.int32, device=DEV) if tree else None)
        want = lengths[rows.long()]
        assert torch.equal(m.cu_q, torch.arange(B + 1, dtype=torch.int32, device=DEV)) and torch.equal(m.token_seq, at)
        assert torch.equal(m.cached, want) and torch.equal(m.positions, want) and torch.equal(m.ctx_len, want + 1)
        if tree:
            assert (m.slots == -1).all() and (m.ancestors == 1).all()
        else:
            assert torch.equal(m.slots, pages[rows.long(), (want // page).long()] * page + want % page)
    kept, path, following, slots, ends = (torch.full(s, -7, dtype=torch.int32, device=DEV) for s in ((B,), (B, 1), (B,), (B,), (B,)))
    ops.tree_accept(at, at, torch.full((B,), -1, dtype=torch.int32, device=DEV), m.cu_q, m.cached, m.block_tables, page, B, kept, path, following, slots, ends, rows)
    assert (kept == 1).all() and torch.equal(path[:, 0], at) and torch.equal(following, at)
    assert torch.equal(ends[rows.long()], want + 1)
    q, k, v = (torch.randn(B, 16, device=DEV).to(torch.bfloat16) for _ in range(3))
    pool, out = torch.randn(B * page, 16, device=DEV).to(torch.bfloat16), torch.zeros(B, 16, dtype=torch.bfloat16, device=DEV)
    ops.tree_attention(q, k, v, 1, 1, 16, pool, pool, page, m.block_tables, torch.zeros_like(m.cached), m.cu_q, m.ancestors, None, 0.25, out, max_new=1, max_cached=0)
    assert torch.equal(out, v)


def token_by_token(ops, dtype, prompts, steps):
    m = Model(ops, dtype)
    texts, margins = [], []
    for r, prompt in enumerate(prompts):
        text, feed, margin = list(prompt), list(prompt), []
        for _ in range(steps):
            maps = ops.StepMaps(1, len(feed), m.BLOCKS, len(feed))
            ops.step_maps(maps, ints([r]), ints([len(feed)]), m.lengths, m.pages, m.PAGE, m.n_pages)
            chosen, _, logits = m.forward(ints(feed), maps, False, len(feed), 80)
            m.lengths[r] += len(feed)
            two = logits[-1].topk(2).values
            margin.append(float(two[0] - two[1]))
            feed = [int(chosen[-1])]
            text += feed
        texts.append(text)
        margins.append(margin)
    return m, texts, margins


@pytest.mark.parametrize("captured", [False, True])
def test_drafted_trees_give_the_text_of_token_by_token(ops, captured):
    """Three requests in 32 bits: trees drafted from the known text with wrong siblings and early ends give the same tokens and the same
    cache; lengths and tables of the next step come from the device. Captured: the whole step is one graph, replayed on new drafts."""
    prompts = [[5, 17, 3, 99, 140], [1], [7] * 20]
    steps, N, ROWS = 30, 12, [2, 0, 3]
    ref, texts, margins = token_by_token(ops, torch.float32, prompts, steps)
    # (rounding moves logits by about 1e-5: a choice between two closer than 1e-3 could turn over)
    assert min(min(m) for m in margins) > 1e-3, "choose another seed of weights"
    m = Model(ops, torch.float32)
    rows, B, T = ints(ROWS), 3, 3 * N
    for b, prompt in enumerate(prompts):                 # the prompts but for their last token, as portions
        if len(prompt) > 1:
            maps = ops.StepMaps(1, len(prompt) - 1, m.BLOCKS, len(prompt))
            ops.step_maps(maps, ints([ROWS[b]]), ints([len(prompt) - 1]), m.lengths, m.pages, m.PAGE, m.n_pages)
            m.forward(ints(prompt[:-1]), maps, False, len(prompt) - 1, 0)
            m.lengths[ROWS[b]] += len(prompt) - 1
    maps = ops.StepMaps(B, T, m.BLOCKS, N, tree=True)
    ids, parents, n_new = ints([0] * T), ints([0] * T), ints([N] * B)
    kept, following, path, slots = ints([0] * B), ints([0] * B), torch.empty(B, N, dtype=torch.int32, device=DEV), ints([0] * T)

    def step():
        ops.step_maps(maps, rows, n_new, m.lengths, m.pages, m.PAGE, m.n_pages, parents)
        chosen, layers, _ = m.forward(ids, maps, True, N, 80)
        ops.tree_accept(chosen, ids, parents, maps.cu_q, maps.cached, maps.block_tables, m.PAGE, m.n_pages, kept, path, following, slots, lengths=m.lengths, rows=rows)
        for n, qkv in enumerate(layers):
            ops.kv_append(qkv, m.D, m.D + m.kv, m.kv, m.k_pages[n], m.v_pages[n], slots)

    graph = None
    if captured:
        # (a first run that keeps nothing: no sequence brings a node)
        n_new.zero_()
        saved, stream = m.lengths.clone(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        assert torch.equal(m.lengths, saved) and kept.tolist() == [0] * B
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    rng = random.Random(3)
    have = [list(p) for p in prompts]
    while any(len(have[b]) < len(texts[b]) for b in range(B)):
        all_ids, all_parents, counts, expect = [], [], [], []
        for b in range(B):
            # the true text as far as it goes for some nodes, then guesses; beside it wrong siblings
            true = texts[b][len(have[b]):]
            good = rng.randint(0, 5)
            tree_ids, tree_parents, at = [have[b][-1]], [-1], 0
            n = rng.randint(1, N)
            reached = 1
            while len(tree_ids) < n:
                if rng.random() < 0.5 and reached <= min(good, len(true) - 1):
                    tree_ids.append(true[reached - 1])
                    tree_parents.append(at)
                    at, reached = len(tree_ids) - 1, reached + 1
                else:
                    tree_parents.append(rng.randrange(len(tree_ids)))
                    tree_ids.append((rng.choice(texts[b]) + 1 + rng.randrange(50)) % m.V)
            all_ids += tree_ids
            all_parents += tree_parents
            counts.append(n)
            expect.append(reached)
        ids.copy_(ints(all_ids + [0] * (T - len(all_ids))))
        parents.copy_(ints(all_parents + [0] * (T - len(all_parents))))
        n_new.copy_(ints(counts))
        torch.cuda.synchronize()
        if graph is not None:
            graph.replay()
        else:
            step()
        places, n_kept, after = path.tolist(), kept.tolist(), following.tolist()
        for b in range(B):
            assert n_kept[b] >= expect[b]
            new = [all_ids[i] for i in places[b][1:n_kept[b]]] + [after[b]]
            have[b] += new
            # (behind the known text's end nothing is known; the cache has room for a tree more)
            have[b] = have[b][:len(texts[b])] if len(have[b]) > len(texts[b]) else have[b]
            assert have[b] == texts[b][:len(have[b])], b
        lengths = m.lengths.tolist()
        for b in range(B):
            # one request may be ready before the others: it is set back by one token and drafts on from there
            if len(have[b]) == len(texts[b]):
                m.lengths[ROWS[b]] = len(texts[b]) - 2
                have[b] = texts[b][:-1] if any(len(have[x]) < len(texts[x]) for x in range(B)) else have[b]
            else:
                assert lengths[ROWS[b]] == len(have[b]) - 1
    for b in range(B):
        for at in range(len(texts[b]) - 2):
            mine, theirs = (x.pages[r][at // m.PAGE].item() * m.PAGE + at % m.PAGE for x, r in ((m, ROWS[b]), (ref, b)))
            for n in range(m.LAYERS):
                for pool, other in ((m.k_pages, ref.k_pages), (m.v_pages, ref.v_pages)):
                    assert (pool[n][mine] - other[n][theirs]).abs().max() <= 1e-3
