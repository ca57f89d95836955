"""Paged attention against bounds that a lost low part, a lost key or a share joined wrongly would pass (``attn_bounds.py``), over the
kernels' forms: decodes in one piece and in many, joined ones, chunks in one and several shares, windows."""

import numpy as np
import pytest

from attn_bounds import attn_bounds, visible
from mdlc_b200 import _lib as L
from test_paged_gpu import ET, RAW, ctx, dev, store  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

SHAPES = [
    # cached, new, heads, kv_heads, head_dim, page, window, sinks
    ([700], [1], 2, 2, 64, 16, 0, 0), ([4000], [1], 4, 1, 128, 16, 0, 0), ([9000, 37], [1, 1], 8, 2, 64, 32, 0, 0),
    ([300] * 40, [1] * 40, 4, 2, 128, 16, 0, 0), ([2500, 0, 900], [3, 4, 1], 16, 2, 128, 16, 0, 0), ([1200], [9], 4, 1, 96, 7, 0, 0),
    ([240], [60], 1, 1, 64, 16, 0, 0), ([1660], [130], 2, 1, 128, 16, 0, 0), ([5000], [40], 2, 2, 64, 16, 0, 0),
    ([4000, 100, 2000], [70, 1, 150], 4, 2, 64, 64, 0, 0), ([0, 500], [300, 20], 3, 1, 80, 5, 0, 0), ([700, 3000], [100, 1], 8, 1, 128, 16, 0, 0),
    ([2000] * 16, [40] * 16, 8, 8, 64, 16, 0, 0),   # many tiles, cut finely
    ([3000, 50], [1, 120], 4, 2, 64, 16, 500, 20), ([1000], [300], 2, 1, 128, 32, 129, 4)]


def attend(dev, rng, dtype, shape, k_of, v_of, scale):
    """Runs one batch; yields (request, q, k, v, seen, out, lse) per request and head, as stored."""
    cached, new, h, kvh, d, page, window, sinks = shape
    b, kv = len(cached), [c + n for c, n in zip(cached, new)]
    need = [-(-x // page) for x in kv]
    pages, stride, tokens = sum(need) + 2, max(need), sum(new)
    ids, table = rng.permutation(pages), np.full((b, stride), -1, np.int32)
    kc, vc = (np.zeros((pages, kvh, page, d), np.float32) for _ in range(2))
    keys, at = [], 0
    for i, x in enumerate(kv):
        keys.append([store(f((x, kvh, d)), dtype)[1] for f in (k_of, v_of)])
        table[i, :need[i]] = ids[at:at + need[i]]
        at += need[i]
        for src, dst in zip(keys[i], (kc, vc)):
            full = np.zeros((need[i] * page, kvh, d), np.float32)
            full[:x] = src
            dst[table[i, :need[i]]] = full.reshape(need[i], page, kvh, d).transpose(0, 2, 1, 3)
    raw, val = store(rng.standard_normal((tokens, h, d)), dtype)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    desc = L.AttnDesc(batch=b, tokens=tokens, heads=h, kv_heads=kvh, head_dim=d, page=page, pages=pages, table_stride=stride, max_q=max(new),
                      max_kv=max(kv), window=window, sinks=sinks, dtype=ET[dtype], scale=scale, q_stride=h * d, out_stride=h * d)
    out, lse = dev.out((tokens, h, d), RAW[dtype]), dev.out((tokens, h), np.float32)
    dev.ctx.paged_attn(desc, dev.put(raw), dev.put(store(kc, dtype)[0]), dev.put(store(vc, dtype)[0]), dev.put(table), dev.put(starts),
                       dev.put(np.array(kv, np.int32)), out, lse, dev.out(L.paged_attn_workspace(desc), np.uint8))
    dev.ctx.sync()
    got, gl = dev.floats(out, (tokens, h, d), dtype).astype(np.float64), dev.ctx.download(lse, (tokens, h), np.float32)
    for i in range(b):
        rows = slice(starts[i], starts[i + 1])
        for e in range(h):
            k, v = (x[:, e // (h // kvh)].astype(np.float64) for x in keys[i])
            yield i, val[rows, e].astype(np.float64), k, v, visible(new[i], kv[i], window, sinks), got[rows, e], gl[rows, e]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[1])}on{max(s[0])}h{s[2]}-{s[3]}d{s[4]}")
def test_fp32_keeps_every_low_part(dev, rng, shape):  # noqa: F811
    scale = shape[4] ** -0.5
    for i, q, k, v, seen, out, lse in attend(dev, rng, "f32", shape, rng.standard_normal, lambda s: rng.uniform(1, 2, s), scale):
        want, wl, err, lerr = attn_bounds(q, k, v, seen, scale, "f32")
        assert (abs(out - want) <= err).all(), (i, (abs(out - want) / err).max())
        assert (abs(lse - wl) <= lerr).all(), (i, (abs(lse - wl) / lerr).max())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("equal", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[1])}on{max(s[0])}h{s[2]}-{s[3]}d{s[4]}")
def test_every_key_has_its_weight(dev, rng, shape, equal, dtype):  # noqa: F811
    """One-hot values: a column is the weight of the keys that it stands for, all of them alike with `equal`."""
    def one_hot(s):
        v = np.zeros(s)
        j = np.arange(s[0])
        v[j, :, j % s[2]] = 1.0
        return v
    scale = 0.0 if equal else shape[4] ** -0.5
    for i, q, k, v, seen, out, lse in attend(dev, rng, dtype, shape, rng.standard_normal, one_hot, scale):
        want, wl, err, lerr = attn_bounds(q, k, v, seen, scale, dtype)
        assert (abs(out - want) <= err).all(), (i, (abs(out - want) / err).max())
        assert (abs(lse - wl) <= lerr).all(), (i, (abs(lse - wl) / lerr).max())
    if not equal:
        return
    # a positive scale on keys of zero: the chunk form on tcgen05 with equal weights too
    for i, q, k, v, seen, out, lse in attend(dev, rng, dtype, shape, np.zeros, one_hot, 1.0):
        want, wl, err, lerr = attn_bounds(q, k, v, seen, 1.0, dtype)
        assert (abs(out - want) <= err).all(), (i, (abs(out - want) / err).max())
