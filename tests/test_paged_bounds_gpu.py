"""Paged attention of requests that have more tokens than the call's bounds: the rows within them are computed where they stand."""

import math

import numpy as np
import pytest

from attn_bounds import attn_bounds, visible
from mdlc_b200 import _lib as L
from test_paged_gpu import ET, RAW, ctx, dev, store  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("bf16", 5), ("f32", 16)])
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("new,max_q,tokens", [
    ([3, 1], 1, 4), ([9, 2], 4, 11), ([150, 1], 100, 151), ([150, 40], 150, 180), ([2, 300], 280, 302), ([5, 7], 6, 9), ([70, 1], 1, 71)])
def test_rows_within_the_bounds_keep_their_positions(dev, rng, dtype, page, window, new, max_q, tokens):  # noqa: F811
    """`max_q` or `tokens` cut a request: its first rows are the definition's, the others are left as they were."""
    c, d, h, kvh, cached = dev.ctx, 64, 4, 2, [130, 21]
    kv = [a + b for a, b in zip(cached, new)]
    need = [-(-x // page) for x in kv]
    pages, stride = sum(need), max(need)
    table = np.full((2, stride), -1, np.int32)
    kc, vc = (store(rng.standard_normal((pages, kvh, page, d)), dtype) for _ in range(2))
    table[0, :need[0]], table[1, :need[1]] = np.arange(need[0]), need[0] + np.arange(need[1])
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    raw, val = store(rng.standard_normal((tokens, h, d)), dtype)
    scale = 1 / math.sqrt(d)
    desc = L.AttnDesc(batch=2, tokens=tokens, heads=h, kv_heads=kvh, head_dim=d, page=page, pages=pages, table_stride=stride, max_q=max_q,
                      max_kv=max(kv), window=window, dtype=ET[dtype], scale=scale, q_stride=h * d, out_stride=h * d)
    out, lse = dev.out((tokens, h, d), RAW[dtype]), dev.out((tokens, h), np.float32)
    c.paged_attn(desc, dev.put(raw), dev.put(kc[0]), dev.put(vc[0]), dev.put(table), dev.put(starts), dev.put(np.array(kv, np.int32)), out, lse,
                 dev.out(L.paged_attn_workspace(desc), np.uint8))
    c.sync()
    got, gl = dev.floats(out, (tokens, h, d), dtype), c.download(lse, (tokens, h), np.float32)
    for i in range(2):
        rows = min(max_q, max(0, min(int(starts[i + 1]), tokens) - int(starts[i])))
        at = slice(starts[i], starts[i] + rows)
        for e in range(h):
            k, v = (x[1][table[i, :need[i]], e // (h // kvh)].reshape(-1, d)[:kv[i]].astype(np.float64) for x in (kc, vc))
            want, wl, err, lerr = attn_bounds(val[at, e].astype(np.float64), k, v, visible(new[i], kv[i], window)[:rows], scale, dtype)
            assert (abs(got[at, e] - want) <= err).all() and (abs(gl[at, e] - wl) <= lerr).all()
        left = slice(starts[i] + rows, min(int(starts[i + 1]), tokens))
        assert np.isnan(got[left]).all() and np.isnan(gl[left]).all()     # as they were
