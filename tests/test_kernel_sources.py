"""Rules that the CUDA sources keep and no run can show: a kernel that breaks one may pass every test on one
compiler and fail on the next."""

import re
from pathlib import Path

import pytest

SOURCES = sorted((Path(__file__).resolve().parents[1] / "opendm_b200" / "csrc").glob("*.cu"))


def _code(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


def _kernels(code):
    """(name, parameters, body) of each __global__ function."""
    for m in re.finditer(r"__global__\s+void\b", code):
        body = code.index("{", m.end())
        head = code[m.end():body]
        at = re.search(r"(\w+)\(((?:[^()]|\([^()]*\))*)\)\s*$", head)
        depth, end = 1, body + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(code[end], 0)
            end += 1
        yield at.group(1), at.group(2), code[body:end]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.stem)
def test_overlapped_kernels_take_no_restrict_pointers(path):
    """A kernel that waits for its predecessor inside runs while that one still writes what it will read: a
    ``const __restrict__`` pointer promises the opposite, and its loads need not stay behind the wait."""
    for name, parameters, body in _kernels(_code(path)):
        if "wait_previous()" in body:
            assert "__restrict__" not in parameters, name


def test_overlapped_launches_are_of_kernels_that_wait():
    found = set()
    for path in SOURCES:
        code = _code(path)
        waiting = {name for name, _, body in _kernels(code) if "wait_previous()" in body}
        for m in re.finditer(r"launch_overlapped\(\s*\"[^\"]*\",\s*(\w+)", code):
            assert m.group(1) in waiting, m.group(1)
            found.add(m.group(1))
    assert found == {"radix_scatter_kernel", "heads_kernel", "sum_kernel", "join_kernel", "list_scale_kernel"}
