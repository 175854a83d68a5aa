"""Kernels that are launched programmatically are on the device before the kernel ahead of them has ended,
and that one may write what they read (accept_tree the lengths, fork_pages the tables, append_packed the
rows). So they read nothing through the read-only path, which is for data that nobody writes while the
kernel is there, and nothing before griddepcontrol.wait. Read from the source; no GPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voltattn_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", ["decode_tree.cuh", "decode_tree_tc.cuh", "cache_rows.cuh", "pages.cuh", "launch_cache.cu"])
def test_no_read_only_loads(name):
    assert not re.findall(r"__ldg\s*\(|ld\.global\.nc", code(name))


@pytest.mark.parametrize("name", ["decode_stream.cuh", "decode_tc.cuh", "decode_tcg.cuh", "decode_mma.cuh"])
def test_lengths_and_tables_of_the_decodes(name):
    """The single-token decodes read the same lengths and tables."""
    assert not re.findall(r"__ldg\s*\(\s*p\.(?:lens|block_table)[^;]*;", code(name))


@pytest.mark.parametrize("name", ["decode_stream.cuh", "decode_tc.cuh", "decode_tcg.cuh", "decode_mma.cuh"])
def test_the_decodes_wait_before_they_read_the_cache(name):
    """No build reads K and V ahead of the wait: the kernels that write rows release the next one early."""
    text = code(name)
    waits = re.findall(r"[^;{}]*\bgrid_dependency_wait\(\)\s*;", text)
    assert all(w.strip() == "grid_dependency_wait();" for w in waits), waits  # none under a condition
    assert "EARLY" not in text.upper(), "a build that starts copies early"
