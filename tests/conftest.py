"""Shared fixtures and markers.

``-m gpu`` tests need a B200 and the built ``libmdlc_b200.so``; everything else
runs on CPU. Golden fixtures live in ``tests/golden`` (made by
``tests/golden/make_golden.py`` from the reference implementation).
"""

from __future__ import annotations

import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA B200 and the built sm_100a library")


# Tests that stay as they were written although one value in them is wrong; the right one is tested elsewhere.
HOLD_A_WRONG_VALUE = {
    "tests/test_paged_gpu.py::test_page_plan_corners":
        "its third case wants kv_lens 4 for a request of which one row is left: attention would place that row at position 3, the plan "
        "itself at 0 (test_page_plan_gpu.py: test_cut_requests_count_as_if_they_brought_their_rows, test_attention_over_a_cut_request)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid in HOLD_A_WRONG_VALUE:
            item.add_marker(pytest.mark.xfail(reason=HOLD_A_WRONG_VALUE[item.nodeid], raises=AssertionError, strict=True))


@pytest.fixture
def rng():
    return np.random.default_rng(1234)


def golden(case: str) -> dict:
    with np.load(os.path.join(GOLDEN, f"{case}.npz")) as z:
        return {k: z[k] for k in z.files}
