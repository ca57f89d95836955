"""The bounds of ``attn_bounds.py`` on the CPU: what the kernels' arithmetic does stays inside them, and what a mistake would do
does not."""

import numpy as np
import pytest

from attn_bounds import attn_bounds, visible
from oracle import reference as oref


def tf32(x):
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) & np.uint32(0xFFFFE000)).view(np.float32).astype(np.float64)


def bf16(x):
    return oref.round_bf16(np.asarray(x, np.float32)).astype(np.float64)


def forward(q, k, v, seen, scale, form):
    """(out, lse) of attention in 64 bits with one step of it done worse."""
    vv = tf32(v) if form in ("tf32", "values_tf32") else v
    s = scale * (tf32(q) @ tf32(k).T if form in ("tf32", "scores_tf32") else q @ k.T)
    s = np.where(seen, s, -np.inf)
    top = s.max(1, keepdims=True)
    w = np.exp(s - top)
    total = w.sum(1, keepdims=True)
    lse = (top + np.log(total))[:, 0]
    if form in ("tf32", "weights_tf32"):
        w = tf32(w)
    elif form == "weights_bf16":
        w = bf16(w)
    elif form == "lost_key":
        w[:, k.shape[0] // 2] = 0
    elif form == "lost_block":
        w[:, 16:32] = 0
    out = (w @ vv) / total
    return (bf16(out) if form == "weights_bf16" else out.astype(np.float32).astype(np.float64)), lse


def outside(got, want):
    return (abs(got[0] - want[0]) > want[2]).any() or (abs(got[1] - want[1]) > want[3]).any()


SHAPES = [(1, 700, 64), (1, 4000, 128), (60, 300, 64), (40, 1700, 128), (8, 190, 128)]


@pytest.mark.parametrize("n,m,d", SHAPES)
def test_fp32_bound(rng, n, m, d):
    """Values of one sign: what is cut off adds up."""
    q, k = (rng.standard_normal(s).astype(np.float32).astype(np.float64) for s in ((n, d), (m, d)))
    v = rng.uniform(1, 2, (m, d)).astype(np.float32).astype(np.float64)
    seen, scale = visible(n, m), d ** -0.5
    want = attn_bounds(q, k, v, seen, scale, "f32")
    assert not outside(forward(q, k, v, seen, scale, "exact"), want)
    for bad in ("tf32", "scores_tf32", "weights_tf32", "values_tf32", "lost_key", "lost_block"):
        assert outside(forward(q, k, v, seen, scale, bad), want), bad


@pytest.mark.parametrize("n,m,d", SHAPES)
def test_bf16_bound(rng, n, m, d):
    """Equal weights and one-hot values: every key has its part of one column."""
    q, k = (bf16(rng.standard_normal(s)) for s in ((n, d), (m, d)))
    v = np.zeros((m, d))
    v[np.arange(m), np.arange(m) % d] = 1.0
    seen = visible(n, m)
    for scale in (d ** -0.5, 0.0):
        want = attn_bounds(q, k, v, seen, scale, "bf16")
        assert not outside(forward(q, k, v, seen, scale, "weights_bf16"), want)
    for bad in ("lost_key", "lost_block"):
        assert outside(forward(q, k, v, seen, 0.0, bad), want), bad


def test_rows_that_see_nothing():
    q, k, v = np.ones((3, 8)), np.ones((1, 8)), np.ones((1, 8))
    out, lse, err, lerr = attn_bounds(q, k, v, visible(3, 1), 1.0, "f32")
    assert not out[:2].any() and np.isneginf(lse[:2]).all() and np.isfinite(err).all() and out[2, 0] == 1 and np.isfinite(lerr).all()
