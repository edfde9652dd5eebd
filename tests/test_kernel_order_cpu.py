"""Orders in the kernels' sources that no run can be asked to show: the wrong one hangs the GPU."""
from __future__ import annotations

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dnn-opt_b200", "csrc")


def kernels():
    """(file, name, text) of every kernel; the text ends where the next one begins."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            source = re.sub(r"//[^\n]*", "", f.read())
        for text in re.split(r"\b__global__\b", source)[1:]:
            name = re.search(r"(\w+_kernel)\s*\(", text)
            yield os.path.basename(path), name.group(1) if name else "?", text


HOLDERS = [k for k in kernels() if "tmem_alloc(" in k[2] and "pdl_launch_dependents()" in k[2]]


def test_kernels_are_found():
    assert len(HOLDERS) >= 4


@pytest.mark.parametrize("file,name,text", HOLDERS, ids=[f"{f}:{n}" for f, n, _ in HOLDERS])
def test_tensor_memory_is_held_before_dependents_start(file, name, text):
    """A dependent kernel that allocates tensor memory before it waits for this grid must find every
    CTA of this grid with its own: it would keep the columns until this grid ends."""
    held = text.index("tmem_alloc(")
    freed = text.index("pdl_launch_dependents()")
    assert held < freed
    assert "__syncthreads()" in text[held:freed]
