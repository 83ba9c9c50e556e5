"""Drafted trees at the edges of what a call allows, without a GPU: which words of a node's ancestors tree attention reads, what maps of
portions refuse, copies of step maps."""
import copy
import os
import pickle
import shutil
import subprocess

import pytest

from mini_llm_amd.kernels import ops
from test_draft_tree import MAPS_SIZES, native_ints

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tree_attention_reads_no_word_behind_a_rows_ancestors(tmp_path):
    """Of every kernel, for 1 to 256 nodes, the tiles of its last stage that lie behind the last node among them."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++ on this machine")
    exe = str(tmp_path / "tree_words")
    done = subprocess.run([cxx, "-std=c++17", "-O1", "-I" + os.path.join(ROOT, "mini_llm_amd", "csrc", "kernels"), os.path.join(ROOT, "tests", "native", "tree_words.cc"), "-o", exe],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.startswith("ok "), run.stdout + run.stderr


@pytest.mark.parametrize("change,match", [(dict(max_new=300), "at most 256"), (dict(words=0), "words"), (dict(max_new=65), "words"), (dict(words=5), "words"),
                                          (dict(ancestors=2 << 20), "ancestors shares memory")])
def test_ancestors_of_portions_are_checked_as_those_of_trees(change, match):
    """Step maps write the chains' ancestors of portions too, wherever there is an array for them."""
    with pytest.raises(ops.KernelError, match=match):
        native_ints(ops.StepMapsC, "mllm_op_step_maps", MAPS_SIZES, **dict(dict(parents=0), **change))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda m: pickle.loads(pickle.dumps(m))], ids=["copy", "deepcopy", "pickle"])
def test_copies_of_step_maps_are_filled_in_their_own_arrays(tree, again):
    """What the kernel is handed are the addresses of the object's own arrays, not those of the object it was copied from, which may be gone."""
    maps = ops.StepMaps(2, 8, 3, 4, tree=tree, device="cpu")
    other = again(maps)
    names = ("cu_q", "cached", "ctx_len", "token_seq", "positions", "slots", "block_tables", "ancestors")
    for m in (maps, other):
        assert m.addresses == tuple(0 if getattr(m, n) is None else getattr(m, n).data_ptr() for n in names)
    assert (other.addresses == maps.addresses) == (again is copy.copy)          # (a shallow copy shares them)
    assert [getattr(other, n) for n in ("n_seqs", "tokens", "max_blocks", "max_new", "words")] == [2, 8, 3, 4, 1]
    with pytest.raises(AttributeError, match="keep their arrays"):
        other.slots = maps.slots
    with pytest.raises(AttributeError, match="keep their arrays"):
        del other.slots
