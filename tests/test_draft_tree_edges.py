"""Drafted trees at the edges of what a call allows, without a GPU: which words of a node's ancestors tree attention reads."""
import os
import shutil
import subprocess

import pytest

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
