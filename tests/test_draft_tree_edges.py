"""Drafted trees at the edges of what a call allows, without a GPU: which words of a node's ancestors tree attention reads, what maps of
portions refuse."""
import os
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
