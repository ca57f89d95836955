"""Kernels started by ``launch_pdl`` may begin while the kernel in front of them still runs: each has to wait for it,
whatever its arguments, before it touches global memory (``csrc/common.cuh``). Read from the sources, no GPU needed."""

import glob
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "mdlc_b200", "csrc")


def body_at(text, at):
    """The braced block that opens at or after `at`."""
    i = text.index("{", at)
    depth, j = 0, i
    while True:
        depth += {"{": 1, "}": -1}.get(text[j], 0)
        j += 1
        if depth == 0:
            return text[i:j]


def kernels():
    """(file, kernel, body) of every __global__ function that is not launched the ordinary way."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        ordinary = set(re.findall(r"(\w+)\s*(?:<[^;<>]*>)?\s*<<<", text))
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
            if m.group(1) not in ordinary:
                depth, j = 1, m.end()
                while depth:
                    depth += {"(": 1, ")": -1}.get(text[j], 0)
                    j += 1
                found.append((os.path.basename(path), m.group(1), body_at(text, j)))
    return found


def test_kernels_are_found():
    names = {k for _, k, _ in kernels()}
    assert {"attn_tc_kernel", "attn_chunk_kernel", "attn_chunk_join_kernel", "attn_narrow_kernel", "attn_split_kernel", "page_plan_kernel",
            "rope_append_kernel", "gemv_w4_kernel"} <= names


@pytest.mark.parametrize("file,kernel,body", kernels(), ids=lambda v: v if isinstance(v, str) and len(v) < 60 else "")
def test_every_kernel_waits_for_the_one_in_front(file, kernel, body):
    """A pdl_wait() that stands by itself: a statement of the kernel's outermost block, not of a branch."""
    body = body.replace('asm volatile("griddepcontrol.wait;" ::: "memory");', "pdl_wait();")
    depth, outer = 0, ""
    for c in body:
        depth += {"{": 1, "}": -1}.get(c, 0)
        if depth == 1:
            outer += c
    assert re.search(r"[;{}]\s*pdl_wait\(\);", outer), f"{file}: {kernel} does not wait"
    # no __ldg and no named helper that reads the lengths in front of it
    assert not re.search(r"__ldg|find_tile|request_of|split_walk", outer[:outer.index("pdl_wait()")])
