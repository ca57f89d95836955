"""The paged decoder descriptors mirror the header (no GPU needed), and the workspace size is a host answer."""

import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT
from mdlc_b200 import _lib as L

STRUCTS = {"mdlc_page_desc": "PageDesc", "mdlc_rope_desc": "RopeDesc", "mdlc_attn_desc": "AttnDesc", "mdlc_w4_desc": "W4Desc"}


def test_struct_layouts_match_header(tmp_path):
    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mdlc_b200.h"', "int main(void) {"]
    for cname, pname in STRUCTS.items():
        lines.append(f'printf("{pname} size %zu\\n", sizeof({cname}));')
        for field, _ in getattr(L, pname)._fields_:
            lines.append(f'printf("{pname} {field} %zu\\n", offsetof({cname}, {field}));')
    lines += ["return 0;", "}"]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    seen = 0
    for line in filter(None, out):
        pname, field, value = line.split()
        cls = getattr(L, pname)
        assert (C.sizeof(cls) if field == "size" else getattr(cls, field).offset) == int(value), (pname, field)
        seen += 1
    assert seen == sum(1 + len(getattr(L, p)._fields_) for p in STRUCTS.values())


def test_request_limit_matches_header():
    text = open(os.path.join(ROOT, "include", "mdlc_b200.h")).read()
    assert int(re.search(r"#define MDLC_MAX_REQUESTS (\d+)", text).group(1)) == L.MAX_REQUESTS


def test_attention_workspace():
    d = dict(batch=4, tokens=4, heads=8, kv_heads=2, head_dim=128, page=16, pages=99, table_stride=30, max_q=1, max_kv=400, dtype=L.BF16,
             scale=0.1, q_stride=1024, out_stride=1024)
    small = L.paged_attn_workspace(L.AttnDesc(**d))
    assert small % 16 == 0 and 0 < small < 64 << 20
    assert L.paged_attn_workspace(L.AttnDesc(**{**d, "batch": 400, "tokens": 400})) > small   # grows with the requests
    assert L.paged_attn_workspace(L.AttnDesc(**{**d, "max_kv": 200})) == small                # not with their lengths
    for bad in (dict(head_dim=12), dict(kv_heads=3), dict(batch=0), dict(dtype=L.U8), dict(q_stride=1000)):
        with pytest.raises(L.MdlcError):
            L.paged_attn_workspace(L.AttnDesc(**{**d, **bad}))
