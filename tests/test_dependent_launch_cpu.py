"""Programmatic dependent launch, read from the kernels' source: a grid launched as a dependent must wait for
its prerequisite on every path, or the launch behind it (and the memory that the prerequisite still
writes) is ordered behind nothing."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "tokenfactory_b200", "csrc")


def _bodies(path):
    """(name, body) of the file's kernels, comments removed"""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)
    for m in re.finditer(r"__global__\b[^;{]*?(\w+)\s*\(", text):
        at = text.index("{", m.end())
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        yield m.group(1), text[at:end]


@pytest.mark.parametrize("name", ["paged_fp8_rows.cu", "paged_decode_mma.cu"])
def test_dependent_grids_wait_before_any_exit(name):
    waits = 0
    for kernel, body in _bodies(os.path.join(CSRC, name)):
        at = body.find("griddepcontrol.wait")
        if at < 0:
            continue
        waits += 1
        assert "return" not in body[:at], f"{kernel} may return before it has waited"
    assert waits > 0
