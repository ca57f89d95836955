"""4-bit quantisation and rotation tables on the host; the example decoder on the GPU against its dense form."""

import importlib.util
import os

import numpy as np
import pytest

from conftest import ROOT
from mdlc_b200 import paged


def load_example():
    spec = importlib.util.spec_from_file_location("paged_decoder", os.path.join(ROOT, "examples", "paged_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (7, 256, 64), (16, 384, 128)])
def test_quantize_w4_round_trip(rng, n, k, group, zeros):
    """Every weight is within half a step of its code's value (a step more at the rounded scale's clipped ends)."""
    w = rng.standard_normal((n, k)).astype(np.float32)
    codes, bits, z = paged.quantize_w4(w, group, zeros)
    assert codes.shape == (n, k // 2) and codes.dtype == np.uint8 and bits.shape == (n, k // group) and (z is not None) == zeros
    scale = (bits.astype(np.uint32) << 16).view(np.float32)
    err = abs(paged.dequantize_w4(codes, bits, z) - w).reshape(n, k // group, group).max(-1)
    assert (err <= scale * (1.01 if zeros else 0.54)).all()


def test_quantize_w4_corners():
    codes, bits, z = paged.quantize_w4(np.zeros((2, 64), np.float32), 32)
    assert not paged.dequantize_w4(codes, bits, z).any()
    with pytest.raises(ValueError):
        paged.quantize_w4(np.zeros((2, 48), np.float32), 32)


def test_rope_table():
    t = paged.rope_table(50, 16, 100.0)
    assert t.shape == (50, 8, 2) and t.dtype == np.float32
    np.testing.assert_allclose(t[..., 0] ** 2 + t[..., 1] ** 2, 1, rtol=1e-6)
    np.testing.assert_allclose(t[3, 2], [np.cos(3 * 100.0 ** -0.25), np.sin(3 * 100.0 ** -0.25)], rtol=1e-6)
    assert (t[0, :, 0] == 1).all() and not t[0, :, 1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(window=40, sinks=4), dict(heads=4, kv_heads=4, head_dim=32, page=8)])
def test_decoder_fp32_matches_its_dense_form(kw):
    """Chunked prompts, decoding and released pages together: fp32 logits within the few hundred rounded sums of two layers."""
    seqs, worst = load_example().run(steps=6, dtype="fp32", check=True, **kw)
    assert worst < 1e-4
    assert min(len(s) for s in seqs) >= 7


@pytest.mark.gpu
def test_decoder_bf16():
    """bf16 activations: a dozen roundings of 2^-8 per layer."""
    _, worst = load_example().run(steps=4, dtype="bf16", check=True)
    assert worst < 0.1


@pytest.mark.gpu
def test_cache_refuses_what_does_not_fit():
    from mdlc_b200 import _lib as L
    ctx = L.Context(0)
    c = paged.PagedCache(ctx, layers=1, batch=2, pages=3, page=4, heads=1, kv_heads=1, head_dim=8, max_tokens=16, max_len=12, dtype=L.F32)
    c.plan([4, 5])
    with pytest.raises(L.MdlcError) as e:
        c.plan([1, 0])
    assert e.value.status == L.ERR_NOMEM
    for bad in ([0, 0], [1], [-1, 2], [9, 0], [17, 0]):
        with pytest.raises(ValueError):
            c.plan(bad)
    c.release(1)
    c.plan([1, 0])
    assert list(c.lens) == [5, 0] and len(c.free) == 1
    ctx.sync()
    c.close()
    ctx.close()
