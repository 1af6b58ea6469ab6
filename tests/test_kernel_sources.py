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


def test_shared_arrays_of_narrow_types_state_their_alignment():
    """Shared arrays of floats, 16-bit counts and bytes are stored and cleared in wider words, which fault where the
    array starts between two of them; a declaration alone promises no more than its element's alignment."""
    code = "".join(map(_code, [p for p in SOURCES if p.stem in ("embedding", "grad_clip")]))
    declared = re.findall(r"__shared__([^;=]*?)\b(float|uint16_t|unsigned char)\s+(\w+)\[", code)
    declared += re.findall(r"\n((?: *__align__\(16\))? *)(uint16_t)\s+(counts)\[RS_WARPS\]\[RS_BINS\];", code)
    assert {"red", "counts", "ring", "raw"} <= {name for _, _, name in declared}
    for qualifiers, _, name in declared:
        assert "__align__(16)" in qualifiers, name
