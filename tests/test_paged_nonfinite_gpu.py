"""Non-finite queries and keys in paged attention: a NaN or an infinity that a token sees is not lost, whichever column of a
product it stands in, and one that it does not see changes nothing."""

import math

import numpy as np
import pytest

from mdlc_b200 import _lib as L
from test_paged_gpu import ET, H, RAW, U, attn_definition, ctx, dev, store  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

PAGE = 16
# decoding, several rows per request, chunks
NEWS = [1, 6, 200]


def attend(dev, dtype, q, k, v, window=0, sinks=0):
    """One request, its new tokens `q` [n, h, d] (fp32) on keys and values [kv, kvh, d]: (q, k, v as stored, out, lse)."""
    n, h, d = q.shape
    kv, kvh = k.shape[:2]
    pages = -(-kv // PAGE)

    def paged(x):
        c = np.zeros((pages * PAGE, kvh, d), np.float32)
        c[:kv] = x
        return np.ascontiguousarray(c.reshape(pages, PAGE, kvh, d).transpose(0, 2, 1, 3))
    (qr, qv), (kr, _), (vr, _) = store_all(q, dtype), store_all(paged(k), dtype), store_all(paged(v), dtype)
    desc = L.AttnDesc(batch=1, tokens=n, heads=h, kv_heads=kvh, head_dim=d, page=PAGE, pages=pages, table_stride=pages, max_q=n, max_kv=kv,
                      window=window, sinks=sinks, dtype=ET[dtype], scale=1 / math.sqrt(d), q_stride=h * d, out_stride=h * d)
    out, lse = dev.out((n, h, d), RAW[dtype], 0), dev.out((n, h), np.float32, 0)
    dev.ctx.paged_attn(desc, dev.put(qr), dev.put(kr), dev.put(vr), dev.put(np.arange(pages, dtype=np.int32)),
                       dev.put(np.array([0, n], np.int32)), dev.put(np.array([kv], np.int32)), out, lse, dev.out(L.paged_attn_workspace(desc), np.uint8))
    dev.ctx.sync()
    return qv, store_all(k, dtype)[1], store_all(v, dtype)[1], dev.floats(out, (n, h, d), dtype), dev.ctx.download(lse, (n, h), np.float32)


def store_all(x, dtype):
    """`store` for arrays with NaN in them (a quiet NaN's upper half is one too)."""
    raw, val = store(np.where(np.isnan(x), 0, x), dtype)
    raw, val = raw.copy(), val.copy()
    raw[np.isnan(x)] = 0x7FC0 if dtype == "bf16" else np.nan
    val[np.isnan(x)] = np.nan
    return raw, val


def tolerance(dtype, v):
    return (64 * U if dtype == "f32" else 2.5 * H) * abs(v[np.isfinite(v)]).max() + 1e-5


@pytest.mark.parametrize("new", NEWS)
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 64), ("f32", 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("window", [0, 90])
def test_bad_key_reaches_the_tokens_that_see_it(dev, rng, dtype, d, new, bad, window):  # noqa: F811
    """One key of which every token with a positive first query element gets a score of NaN or +inf, at each index modulo 32."""
    h, kvh, kv = 4, 2, 300
    q, k, v = (rng.standard_normal(s).astype(np.float32) for s in ((new, h, d), (kv, kvh, d), (kv, kvh, d)))
    q[..., 0] = 1.0
    for at in range(kv - min(new, 60) - 32, kv - min(new, 60)):
        k1 = k.copy()
        k1[at, :, 0] = bad
        qv, kk, vv, out, lse = attend(dev, dtype, q, k1, v, window)
        p = kv - new + np.arange(new)
        sees = (p >= at) & ((window == 0) | (at > p - window))
        assert sees.any()
        assert np.isnan(out[sees]).all() and not np.isfinite(lse[sees]).any()
        if np.isnan(bad):
            assert np.isnan(lse[sees]).all()
        if (~sees).any():
            kk[at] = 0
            want, wl = attn_definition(qv.astype(np.float64), kk.astype(np.float64), vv.astype(np.float64), kv, window, 0, 1 / math.sqrt(d))
            assert abs(out[~sees] - want[~sees]).max() <= tolerance(dtype, vv)
            assert np.isfinite(lse[~sees]).all()


@pytest.mark.parametrize("new", NEWS)
@pytest.mark.parametrize("d", [64, 128])
def test_key_of_minus_infinity_weighs_nothing(dev, rng, d, new):  # noqa: F811
    """bf16: a score of -inf is a weight of 0, like a key that is not there."""
    h, kvh, kv = 4, 2, 300
    q, k, v = (rng.standard_normal(s).astype(np.float32) for s in ((new, h, d), (kv, kvh, d), (kv, kvh, d)))
    q[..., 0] = 1.0
    gone = np.arange(33, 66)
    k[gone, :, 0] = -np.inf
    qv, kk, vv, out, lse = attend(dev, "bf16", q, k, v)
    want, wl = attn_definition(qv.astype(np.float64), kk.astype(np.float64), vv.astype(np.float64), kv, 0, 0, 1 / math.sqrt(d))
    assert abs(out - want).max() <= tolerance("bf16", vv)
    assert abs(lse - wl).max() <= 1e-4


@pytest.mark.parametrize("new", NEWS)
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 64), ("f32", 128)])
def test_nan_query_is_its_own_rows(dev, rng, dtype, d, new):  # noqa: F811
    h, kvh, kv = 4, 2, 300
    q, k, v = (rng.standard_normal(s).astype(np.float32) for s in ((new, h, d), (kv, kvh, d), (kv, kvh, d)))
    q[new // 2, 1, 3] = np.nan
    qv, kk, vv, out, lse = attend(dev, dtype, q, k, v)
    assert np.isnan(out[new // 2, 1]).all() and np.isnan(lse[new // 2, 1])
    qv[new // 2, 1] = 0
    want, wl = attn_definition(qv.astype(np.float64), kk.astype(np.float64), vv.astype(np.float64), kv, 0, 0, 1 / math.sqrt(d))
    rest = np.ones((new, h), bool)
    rest[new // 2, 1] = False
    assert abs(out[rest] - want[rest]).max(initial=0) <= tolerance(dtype, vv)
    assert abs(lse[rest] - wl[rest]).max(initial=0) <= 1e-4


@pytest.mark.parametrize("d", [64, 128])
def test_hidden_keys_weigh_nothing_beside_large_values(dev, rng, d):  # noqa: F811
    """Values near the type's largest behind the mask: a weight of 2^-126 in place of 0 would show."""
    new = kv = 200
    q, k, v = (rng.standard_normal(s).astype(np.float32) for s in ((new, 2, d), (kv, 1, d), (kv, 1, d)))
    v[120:] = 3e38
    qv, kk, vv, out, lse = attend(dev, "bf16", q, k, v)
    want, _ = attn_definition(qv.astype(np.float64), kk.astype(np.float64), vv.astype(np.float64), kv, 0, 0, 1 / math.sqrt(d))
    assert abs(out[:120] - want[:120]).max() <= tolerance("bf16", vv[:120])
