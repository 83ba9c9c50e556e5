"""What the operations over trees of drafted tokens refuse, without a GPU: the Python face by shapes and types, the native side (which
checks before it launches) by numbers; and their plain implementation against cases written out."""
import ctypes
import math

import pytest
import torch

import plain_tree
from mini_llm_amd.kernels import ops

I32, F = torch.int32, torch.float32


def i32(*shape):
    return torch.zeros(shape, dtype=I32)


def attention_args(**change):
    a = dict(q=torch.zeros(3, 64), k=torch.zeros(3, 32), v=torch.zeros(3, 32), n_heads=4, n_kv_heads=2, head_dim=16, k_pages=torch.zeros(32, 32), v_pages=torch.zeros(32, 32),
             page_size=16, block_tables=i32(2, 2), cached=i32(2), cu_q=i32(3), ancestors=torch.zeros(3, 1, dtype=torch.int64), positions=i32(3), scale=1.0, out=torch.zeros(3, 64),
             max_new=3, max_cached=20)
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(block_tables=i32(3, 2)), "block_tables"), (dict(block_tables=torch.zeros(2, 2)), "block_tables"), (dict(block_tables=i32(2, 4)[:, ::2]), "block_tables"),
    (dict(cu_q=i32(2)), "cu_q"), (dict(cached=torch.zeros(2)), "cached"), (dict(ancestors=torch.zeros(3, 1, dtype=I32)), "ancestors"),
    (dict(ancestors=torch.zeros(2, 1, dtype=torch.int64)), "ancestors"), (dict(positions=i32(2)), "positions"), (dict(positions=None, window=4), "positions"),
    (dict(q=torch.zeros(3, 128)[:, ::2]), "contiguous last"), (dict(q=torch.zeros(3, 64, dtype=torch.float16)), "dtype"), ({}, "not on the GPU")])
def test_tree_attention_refuses(change, match):
    with pytest.raises(ops.KernelError, match=match):
        ops.tree_attention(**attention_args(**change))


def native_attention(**change):
    """A native call whose checks fail in front of any launch; addresses are never read."""
    at = lambda i, dt, r, c, s=None: ops.Tensor2(1 << (20 + i), dt, r, c, c if s is None else s)      # noqa: E731
    a = ops.TreeAttentionC()
    dt = change.pop("dtype", 1)
    a.q, a.k, a.v, a.out = at(0, dt, 3, 64), at(1, dt, 3, 32), at(2, dt, 3, 32), at(3, dt, 3, 64)
    a.k_pages, a.v_pages, a.page_size = at(4, dt, 32, 32), at(5, dt, 32, 32), 16
    a.n_heads, a.n_kv_heads, a.head_dim, a.n_seqs, a.max_blocks, a.words, a.max_new, a.max_cached, a.scale = 4, 2, 16, 2, 2, 1, 3, 20, 1.0
    a.block_tables = a.cached = a.cu_q = a.ancestors = a.positions = 1 << 30
    for name, value in change.items():
        setattr(a, name, at(*value) if isinstance(value, tuple) else value)
    ops._ok(ops.engine_library().mllm_op_tree_attention(ctypes.byref(a), None))


@pytest.mark.parametrize("change,match", [
    (dict(n_kv_heads=3), "multiple"), (dict(n_heads=0), "multiple"), (dict(head_dim=12), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(q=(0, 1, 3, 32)), "q and out"),
    (dict(out=(3, 1, 2, 64)), "q and out"), (dict(out=(3, 0, 3, 64)), "one dtype"), (dict(k=(1, 1, 4, 32)), "k and v"), (dict(v=(2, 1, 3, 64)), "k and v"),
    (dict(k_pages=(4, 1, 48, 32)), "one shape"), (dict(k_pages=(4, 1, 32, 32, 64)), "contiguous"), (dict(page_size=24), "whole number"), (dict(page_size=0), "whole number"),
    (dict(q=(0, 1, 3, 64, 68)), "aligned"), (dict(words=5), "words"), (dict(words=0), "words"), (dict(max_new=65), "words"), (dict(max_new=0), "words"), (dict(max_cached=-1), "max_cached"),
    (dict(window=-1), "window"), (dict(window=3, positions=0), "positions"), (dict(cu_q=0), "needed"), (dict(ancestors=0), "needed"), (dict(n_seqs=0), "needed"),
    (dict(out=(0, 1, 3, 64)), "shares memory"), (dict(q=(0, 1, 3, 64, 32)), "apart"), (dict(q=(0, 7, 3, 64)), "dtype"), (dict(n_heads=1 << 20), "multiple")])
def test_native_tree_attention_refuses(change, match):
    with pytest.raises(ops.KernelError, match=match):
        native_attention(**change)


def test_native_tree_attention_wants_its_workspace():
    """Few rows of a long cache are split: the call is refused without its workspace. The longest cache that the numbers allow asks for no more
    than splits of it, and sizes that the call refuses for nothing."""
    size = ops.engine_library().mllm_op_tree_attention_workspace
    for dtype in (0, 1):
        assert 0 < size(3, 2, 4, 2, 16, 3, 2 ** 31 - 1, 0, dtype) < 2 ** 20
        with pytest.raises(ops.KernelError, match="workspace"):
            native_attention(dtype=dtype, max_cached=2 ** 31 - 1)
    assert [size(*s) for s in ((3, 2, 4, 0, 16, 3, 99999, 0, 1), (3, 2, 4, 3, 16, 3, 99999, 0, 1), (3, 2, 4, 2, 300, 3, 99999, 0, 1), (0, 0, 4, 2, 16, 3, 99999, 0, 1))] == [0] * 4


def test_structures_are_as_the_native_side_has_them():
    for form, c in ((ops._MAPS_BYTES, ops.StepMapsC), (ops._ACCEPT_BYTES, ops.TreeAcceptC), (ops._ATTENTION_BYTES, ops.TreeAttentionC), (ops._ROWS_BYTES, ops.Tensor2)):
        assert form.size == ctypes.sizeof(c)


def test_numbers_beyond_32_bits_are_refused():
    for name in ("max_cached", "page_size", "window"):
        with pytest.raises(ops.KernelError):
            ops.tree_attention(**attention_args(**{name: 2 ** 40}))


def maps_args(**change):
    maps = change.pop("maps", None) or ops.StepMaps(2, 8, 3, 4, tree=True, device="cpu")
    a = dict(maps=maps, rows=i32(2), n_new=i32(2), lengths=i32(5), pages=i32(5, 3), page_size=16, n_pages=9, parents=i32(8))
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(rows=i32(3)), "rows"), (dict(n_new=i32(1)), "n_new"), (dict(lengths=i32(4)), "lengths"), (dict(pages=i32(5, 2)), "blocks"), (dict(pages=torch.zeros(5, 3)), "pages"),
    (dict(pages=i32(5, 6)[:, ::2]), "pages"), (dict(parents=i32(7)), "parents"), (dict(maps=ops.StepMaps(2, 8, 3, 4, device="cpu")), "made for trees"), ({}, "not on the GPU")])
def test_step_maps_refuses(change, match):
    with pytest.raises(ops.KernelError, match=match):
        ops.step_maps(**maps_args(**change))


@pytest.mark.parametrize("args", [(0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)])
def test_step_maps_of_nothing_are_refused(args):
    with pytest.raises(ops.KernelError):
        ops.StepMaps(*args, device="cpu")


def test_step_maps_of_too_large_trees_are_refused():
    assert ops.tree_max_nodes() == 256
    with pytest.raises(ops.KernelError, match="256"):
        ops.StepMaps(1, 1, 1, 257, tree=True, device="cpu")
    assert ops.StepMaps(1, 9, 1, 256, tree=True, device="cpu").ancestors.shape == (9, 4)
    assert ops.StepMaps(1, 9, 1, 5000, device="cpu").ancestors is None


@pytest.mark.parametrize("change,match", [
    (dict(page_size=0), "pages of"), (dict(n_pages=1 << 28), "pages of"), (dict(n_pages=0), "pages of"), (dict(max_new=300), "at most 256"), (dict(words=0), "words"), (dict(words=5), "words"),
    (dict(n_seqs=1 << 30, max_new=256, words=4), "sequences"), (dict(slots=0), "missing"), (dict(rows=0, n_seqs=9), "without rows"), (dict(ld_pages=2), "apart")])
def test_native_step_maps_refuses(change, match):
    a = ops.StepMapsC(**dict({n: 1 << 20 for n, t in ops.StepMapsC._fields_ if t is ctypes.c_void_p}, ld_pages=3, n_seqs=2, n_requests=5, tokens=8, page_size=16, n_pages=9,
                             max_blocks=3, max_new=4, words=1, **{}) | change)
    with pytest.raises(ops.KernelError, match=match):
        ops._ok(ops.engine_library().mllm_op_step_maps(ctypes.byref(a), None))


def accept_args(**change):
    a = dict(choices=i32(6), ids=i32(6), parents=i32(6), cu_q=i32(3), cached=i32(2), block_tables=i32(2, 4), page_size=16, n_pages=9, kept=i32(2), path=i32(2, 3), next_token=i32(2),
             slots=i32(6), lengths=i32(2), rows=None)
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(ids=i32(5)), "ids"), (dict(parents=torch.zeros(6)), "parents"), (dict(slots=i32(7)), "slots"), (dict(kept=i32(3)), "kept"), (dict(next_token=i32(1)), "next_token"),
    (dict(cu_q=i32(2)), "cu_q"), (dict(block_tables=i32(3, 4)), "block_tables"), (dict(path=i32(3, 3)), "path"), (dict(path=i32(2, 0)), "path"), (dict(lengths=i32(5)), "lengths"),
    (dict(rows=i32(3)), "rows"), ({}, "not on the GPU"), (dict(rows=i32(2), lengths=i32(9)), "not on the GPU")])
def test_tree_accept_refuses(change, match):
    with pytest.raises(ops.KernelError, match=match):
        ops.tree_accept(**accept_args(**change))


@pytest.mark.parametrize("change,match", [(dict(max_new=257), "at most 256"), (dict(page_size=0), "pages of"), (dict(n_pages=1 << 28), "pages of"), (dict(tokens=0), "0 tokens"), (dict(kept=0), "missing"),
                                          (dict(rows=0, n_requests=1), "without rows")])
def test_native_tree_accept_refuses(change, match):
    a = ops.TreeAcceptC(**dict({n: 1 << 20 for n, t in ops.TreeAcceptC._fields_ if t is ctypes.c_void_p}, n_seqs=2, tokens=6, page_size=16, n_pages=9, max_blocks=4, max_new=3,
                               n_requests=2) | change)
    with pytest.raises(ops.KernelError, match=match):
        ops._ok(ops.engine_library().mllm_op_tree_accept(ctypes.byref(a), None))


def rotary_args(**change):
    x = torch.zeros(3, 64)
    a = dict(x=x, positions=i32(3), freqs=torch.zeros(4, dtype=torch.int64), n_heads=4, head_dim=16, out=x)
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(freqs=torch.zeros(4)), "freqs"), (dict(freqs=torch.zeros(0, dtype=torch.int64)), "freqs"), (dict(out=torch.zeros(3, 32)), "out"), (dict(positions=i32(4)), "positions"),
    (dict(x=torch.zeros(3, 64, dtype=torch.float64)), "dtype"), ({}, "not on the GPU")])
def test_rotary_refuses(change, match):
    with pytest.raises(ops.KernelError, match=match):
        ops.rotary(**rotary_args(**change))


@pytest.mark.parametrize("pairs,heads,dim,x,out,match", [
    (9, 4, 16, (0, 0, 3, 64), (0, 0, 3, 64), "pairs"), (0, 4, 16, (0, 0, 3, 64), (0, 0, 3, 64), "pairs"), (1, 4, 15, (0, 0, 3, 60), (0, 0, 3, 60), "even"), (4, 3, 16, (0, 0, 3, 64), (0, 0, 3, 64), "heads"),
    (4, 4, 16, (0, 0, 3, 64), (1, 1, 3, 64), "dtype"), (4, 4, 16, (0, 0, 3, 64), (0, 0, 3, 64, 80), "shares memory"), (4, 70000, 16, (0, 0, 3, 64), (0, 0, 3, 64), "heads")])
def test_native_rotary_refuses(pairs, heads, dim, x, out, match):
    t = lambda i, dt, r, c, s=None: ops.Tensor2(1 << (20 + i), dt, r, c, c if s is None else s)      # noqa: E731
    with pytest.raises(ops.KernelError, match=match):
        ops._ok(ops.engine_library().mllm_op_rotary(ctypes.byref(t(*x)), 1 << 30, 1 << 30, pairs, heads, dim, 0, 1.0, ctypes.byref(t(*out)), None))


@pytest.mark.parametrize("args", [(7,), (0,), (8, 0.0), (8, math.inf), (8, 1e4, dict(kind="other", factor=2.0)), (8, 1e4, dict(kind="linear")), (8, 1e4, dict(kind="linear", factor=0.0)),
                                  (8, 1e4, dict(kind="linear", factor=2.0, original=5)), (2, 1e4, dict(kind="base", factor=2.0)),
                                  (8, 1e4, dict(kind="by_turns", factor=2.0, original=4096, fast=1.0, slow=32.0)), (8, 1e4, dict(kind="by_pair", factor=2.0, original=0, fast=32.0, slow=1.0)),
                                  (8, 1.0, dict(kind="by_pair", factor=2.0, original=4096, fast=32.0, slow=1.0))])
def test_rotary_freqs_refuses(args):
    with pytest.raises(ops.KernelError):
        ops.rotary_freqs(*args, device="cpu")


def test_rotary_freqs_in_fixed_point():
    """A turn every 2 pi positions for the first pair; by a base of 16 in four pairs every next half as fast."""
    f = [x % 2 ** 64 for x in ops.rotary_freqs(8, 16.0, device="cpu").tolist()]
    assert abs(f[0] / 2 ** 64 - 1 / (2 * math.pi)) < 2.0 ** -52
    assert [f[0] >> i for i in range(4)] == f
    half = [x % 2 ** 64 for x in ops.rotary_freqs(8, 16.0, dict(kind="linear", factor=2.0), device="cpu").tolist()]
    assert half == [x >> 1 for x in f]


# -- the plain implementations against cases written out --------------------------------------------------------------------------
def test_plain_step_maps():
    m = plain_tree.step_maps([1, 0], [3, 2], [4, 2], [[5, 6], [7, 8]], 4, 9, 6, 2, 3, parents=[-1, 0, 0, -1, 0, 9])
    assert m == dict(cu_q=[0, 3, 5], cached=[2, 4], ctx_len=[5, 6], token_seq=[0, 0, 0, 1, 1, 0], positions=[2, 3, 3, 4, 5, 0], slots=[-1] * 6, block_tables=[[7, 8], [5, 6]],
                     ancestors=[[1], [3], [5], [1], [3], [0]])
    m = plain_tree.step_maps(None, [1, 2], [4, 2], [[5, 6], [7, 8]], 4, 9, 3, 2, 3)
    assert m["positions"] == [4, 2, 3] and m["slots"] == [24, 30, 31] and m["block_tables"] == [[5, 6], [7, 0]]


def test_plain_accept():
    # the root's choice 4 names nodes 1 and 2 (the first stands), node 1's choice 6 its child 3
    got = plain_tree.accept([4, 6, 6, 9], [0, 4, 4, 6], [-1, 0, 0, 1], [0, 4], [3], [[2, 5]], 4, 9, 4)
    assert got == ([3], [[0, 1, 3, -1]], [9], [11, 20, -1, 21])


def test_plain_attention():
    q = torch.tensor([[1.0], [1.0]], dtype=F)
    out = plain_tree.attention(q, torch.tensor([[0.0], [5.0]]), torch.tensor([[8.0], [2.0]]), 1, 1, 1, torch.tensor([[0.0], [math.nan]]), torch.tensor([[4.0], [math.nan]]), 1, [[0, 1]], [1],
                               [0, 2], [[1], [0]], [1, 2], 1.0, 0)[0]
    assert out.tolist() == [[6.0], [4.0]]


# -- arrays that share memory, and more sequences than a call takes ------------------------------------------------------------------
def native_ints(kind, op, sizes, **change):
    """A native call whose arrays lie a mebibyte apart, but for those of `change`."""
    a = kind(**dict({n: (i + 1) << 20 for i, n in enumerate(n for n, t in kind._fields_ if t is ctypes.c_void_p)}, **sizes) | change)
    ops._ok(getattr(ops.engine_library(), op)(ctypes.byref(a), None))


MAPS_SIZES = dict(ld_pages=3, n_seqs=2, n_requests=5, tokens=8, page_size=16, n_pages=9, max_blocks=3, max_new=4, words=1)
ACCEPT_SIZES = dict(n_seqs=2, tokens=6, page_size=16, n_pages=9, max_blocks=4, max_new=3, n_requests=2)


def test_step_maps_into_its_inputs_is_refused():
    """Several workgroups read a request's length: the context lengths of the step before cannot be this step's lengths in place."""
    names = [n for n, t in ops.StepMapsC._fields_ if t is ctypes.c_void_p]
    for out in ("cu_q", "cached", "ctx_len", "token_seq", "positions", "slots", "block_tables", "ancestors"):
        for other in names:
            if other != out:
                with pytest.raises(ops.KernelError, match="shares memory"):
                    native_ints(ops.StepMapsC, "mllm_op_step_maps", MAPS_SIZES, **{out: (names.index(other) + 1) << 20})
    with pytest.raises(ops.KernelError, match="ctx_len shares memory with lengths"):
        native_ints(ops.StepMapsC, "mllm_op_step_maps", MAPS_SIZES, ctx_len=(3 << 20) + 4 * 4)


def test_tree_accept_into_its_inputs_is_refused():
    names = [n for n, t in ops.TreeAcceptC._fields_ if t is ctypes.c_void_p]
    for out in ("kept", "path", "next", "slots", "lengths"):
        for other in names:
            if other != out:
                with pytest.raises(ops.KernelError, match="shares memory"):
                    native_ints(ops.TreeAcceptC, "mllm_op_tree_accept", ACCEPT_SIZES, **{out: (names.index(other) + 1) << 20})


def test_more_sequences_than_a_call_takes_are_refused():
    with pytest.raises(ops.KernelError, match="65537 sequences"):
        native_ints(ops.StepMapsC, "mllm_op_step_maps", MAPS_SIZES, n_seqs=65537)
    with pytest.raises(ops.KernelError, match="65537 sequences"):
        native_ints(ops.TreeAcceptC, "mllm_op_tree_accept", ACCEPT_SIZES, n_seqs=65537)
    with pytest.raises(ops.KernelError, match="65537 sequences"):
        native_attention(n_seqs=65537)


def test_step_maps_keep_their_arrays():
    """The kernel writes to addresses taken once: an array put in another's place would not be written, and the one gone would be."""
    m = ops.StepMaps(2, 8, 3, 4, tree=True, device="cpu")
    with pytest.raises(AttributeError, match="keep their arrays"):
        m.slots = i32(8)


def test_kernels_of_drafted_trees_keep_no_register_in_scratch():
    """Tree attention's outputs stay in one set of registers through the loop only as long as no branch in it is the scalar unit's; what spills waits for memory."""
    from test_kernel_resources import kernels
    for library, least in (("tree_attention", 30), ("rotary", 8), ("draft_tree", 2)):
        found = kernels(library)
        assert len(found) >= least
        assert {k: n for k, n in found.items() if n} == {}
