"""Orders within the tensor-core kernels that no run shows to be missing: read from their sources."""

from __future__ import annotations

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "deformops_b200" / "csrc"


def code(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


KERNELS = [path for path in sorted(CSRC.glob("*.cu")) if "tensor_core.cuh" in path.read_text()]


def test_there_are_kernels():
    assert len(KERNELS) >= 3


@pytest.mark.parametrize("path", KERNELS, ids=lambda p: p.name)
def test_dependents_begin_after_tensor_memory_is_taken(path):
    """A CTA lets the next kernel in as soon as one of its threads does.  Were that before its tensor memory is taken, a CTA of
    that kernel could take it and wait for this one to end: only tmem_alloc itself may let it in, as the last thing."""
    text = code(path)
    assert "tmem_alloc(" in text and "launch_dependents" not in text
    alloc = re.search(r"void tmem_alloc\(.*?\n}", code(CSRC / "tensor_core.cuh"), re.S).group(0)
    assert alloc.index("tcgen05.alloc") < alloc.index("griddepcontrol.launch_dependents")


@pytest.mark.parametrize("path", KERNELS, ids=lambda p: p.name)
def test_barriers_are_there_for_the_asynchronous_units(path):
    """Loads and products arrive on barriers through another path than the plain stores that made them: whoever makes them
    fences in the same block, after the last one."""
    text = code(path)
    at = text.rindex("barrier_init(")
    depth, end = 0, at
    while depth >= 0:       # the end of the block that the last barrier is made in
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
    assert "fence_async_shared();" in text[at:end]
