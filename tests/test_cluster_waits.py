"""Waits for data that another block of the cluster gave have the cluster's scope.

``mbarrier.try_wait`` without a scope acquires for the block only, so what it guards
would be read without being ordered behind the other block's stores.  Which scope a
wait has shows in the source alone: the hardware's order hides the difference."""

import re
from pathlib import Path

import matrixman_b200

CSRC = Path(matrixman_b200.__file__).parent / "csrc"


def code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_group_norm_waits_at_the_clusters_scope():
    text = code("mm_group_norm_resident.cu")
    assert "st.async" in text  # blocks give each other their results
    waits = re.findall(r"mbarrier\.(?:try|test)_wait[\w.:]*", text)
    assert waits and all(".acquire.cluster." in w for w in waits), waits


def test_a_block_that_gave_up_waits_for_late_stores_before_it_leaves():
    text = code("mm_group_norm_resident.cu")
    kernels = re.findall(r"\n__global__ void.*?\n}\n", text, re.S)
    assert len(kernels) == 2
    for kernel in kernels:
        assert "given = gn_given(" in kernel
        assert kernel.rstrip().endswith("if (k.ranks > 1) gn_leave_cluster(&bar, given);\n}")
    leave = re.search(r"void gn_leave_cluster\(.*?\n}\n", text, re.S)[0]
    assert re.search(r"gn_wait\(\);\s*if \(!given\) gn_try\(bar\);", leave)
