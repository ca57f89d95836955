"""The paged decoder operators' tests in the bounds-checked build (``python -m mdlc_b200.build --check``): block tables, free lists, cache
rows, outputs, partial sums, 4-bit weights and the split x are indexed inside their tensors, or the error word would say so."""

import os
import re
import subprocess
import sys

import pytest

from conftest import ROOT

CHECK_LIB = os.path.join(ROOT, "mdlc_b200", "libmdlc_b200_check.so")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "mdlc_b200", "csrc", name)).read())


@pytest.mark.parametrize("name,checks", [("paged.cu", 4), ("w4.cu", 6), ("paged_attn.cuh", 6)])
def test_kernels_have_index_checks(name, checks):
    assert source(name).count("MDLC_CHECK_IDX(") >= checks


@pytest.mark.parametrize("name,stores", [("paged_attn.cu", ("table_ok(", "out_ok(", "part_ok(")), ("paged_attn_tc.cu", ("table_ok(", "out_ok(", "part_ok("))])
def test_attention_kernels_use_them(name, stores):
    assert all(source(name).count(s) >= 2 for s in stores)


@pytest.mark.gpu
@pytest.mark.skipif(not os.path.exists(CHECK_LIB), reason="checked build not built")
def test_paged_operators_under_bounds_checks():
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-p", "no:cacheprovider", "-m", "gpu", "-k", "not decoder", "tests/test_paged_gpu.py",
                        "tests/test_paged_tight_gpu.py", "tests/test_page_plan_gpu.py", "tests/test_paged_mixed_gpu.py", "tests/test_w4_exact_gpu.py"],
                       cwd=ROOT, env=dict(os.environ, MDLC_B200_LIB="check"), capture_output=True, text=True, timeout=1200)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]
    assert "libmdlc_b200_check.so" in subprocess.run([sys.executable, "-c", "from mdlc_b200 import _lib; print(_lib.load()._name)"], cwd=ROOT,
                                                     env=dict(os.environ, MDLC_B200_LIB="check"), capture_output=True, text=True, timeout=300).stdout
