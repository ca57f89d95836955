"""4-bit products: every product is exact, so the error follows the sum of their magnitudes and nothing else, in every form the
kernel takes (one or two row tiles, x whole or in two buffers, several chunks of rows, several workspace batches).

The bound. The parts of x are exact. A group's products are added in the tensor core, 16 at a time in at most two steps that each
cut off below 2^-23 of the largest of what is added: 2 group / 16 steps. The scaled groups are then added in fp32 with rounding: a
warp has every eighth step of 128 columns, then three levels of a tree, three parts and the bias, 2^-24 each. So
  |error| <= 2^-23 (group / 8 + (k / 1024 + 1) (128 / group) / 2 + 4) sum |x w|   (+ |bias|),
and a bf16 output is one that some value within that distance rounds to."""

import numpy as np
import pytest

from mdlc_b200 import _lib as L
from oracle import reference as oref
from test_paged_gpu import ET, RAW, ctx, dev, store  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def product(dev, raw, codes, sraw, z, bv, xt, yt, group, k):
    m, n = raw.shape[0], codes.shape[0]
    y = dev.out((m, n), RAW[yt])
    d = L.W4Desc(m=m, n=n, k=k, group=group, x_type=ET[xt], y_type=ET[yt], x_stride=raw.shape[1], y_stride=n)
    dev.ctx.gemv_w4(d, dev.put(raw), dev.put(codes), dev.put(sraw), 0 if z is None else dev.put(z), 0 if bv is None else dev.put(bv), y)
    dev.ctx.sync()
    return dev.floats(y, (m, n), yt)


def weights(codes, sval, z, group):
    n, groups = sval.shape
    q = np.stack([codes & 15, codes >> 4], -1).reshape(n, groups, group).astype(np.float64)
    return ((q - (8 if z is None else z[..., None])) * sval[..., None].astype(np.float64)).reshape(n, -1)


def check(got, x, w, bv, yt, group):
    k = w.shape[1]
    b = 0 if bv is None else bv.astype(np.float64)
    want, mag = x @ w.T + b, abs(x) @ abs(w).T + abs(b)
    tol = 2.0 ** -23 * (group / 8 + (k / 1024 + 1) * (128 / group) / 2 + 4) * mag
    lo, hi = want - tol, want + tol
    if yt == "bf16":
        lo, hi = (oref.round_bf16(v.astype(np.float32)) for v in (lo, hi))
    assert ((got >= lo) & (got <= hi)).all(), (abs(got - want) / mag).max()


def random_case(rng, m, n, k, group, zeros, bias, xt):
    raw, val = store(rng.standard_normal((m, k)), xt)
    codes = rng.integers(0, 256, (n, k // 2)).astype(np.uint8)
    sraw, sval = store(rng.uniform(0.002, 0.03, (n, k // group)), "bf16")
    z = rng.integers(0, 16, sval.shape).astype(np.uint8) if zeros else None
    return raw, val, codes, sraw, sval, z, rng.standard_normal(n).astype(np.float32) if bias else None


@pytest.mark.parametrize("xt,m,n,k,group,zeros,bias", [
    # x in two buffers, one and several tiles per block, rounds of the warps that end inside one
    ("bf16", 16, 300, 14336, 64, 0, 1), ("bf16", 16, 5003, 14336, 128, 1, 0), ("f32", 16, 2500, 4096, 64, 0, 0), ("f32", 8, 300, 14336, 32, 1, 1),
    ("f32", 7, 5003, 2912, 32, 1, 1), ("f32", 13, 2400, 3200, 128, 0, 1), ("bf16", 40, 2500, 4128, 32, 1, 0), ("f32", 1, 9472, 8192, 64, 0, 0),
    # two row tiles per block
    ("bf16", 1, 9472, 256, 128, 0, 0), ("bf16", 1, 9600, 544, 32, 1, 1), ("f32", 1, 18944, 384, 64, 1, 0), ("bf16", 8, 20011, 256, 64, 0, 1),
    ("bf16", 16, 20000, 640, 128, 1, 0), ("f32", 16, 9500, 256, 32, 0, 0), ("f32", 3, 19000, 288, 32, 1, 0),
    # a single row that is too long for the blocks to split themselves
    ("bf16", 1, 40, 24576, 128, 1, 0), ("f32", 1, 40, 8192, 32, 0, 1), ("f32", 1, 40, 16384, 32, 0, 1), ("f32", 1, 40, 12288, 64, 1, 0),
    # chunks of rows, and more of them than the workspace holds at a time
    ("bf16", 49, 70, 256, 64, 1, 0), ("bf16", 160, 33, 1024, 128, 0, 1), ("f32", 200, 40, 14336, 128, 1, 0), ("bf16", 500, 17, 14336, 64, 0, 0),
    # so long that fewer column tiles go into the workspace
    ("f32", 16, 20, 100352, 128, 0, 0)])
def test_forms(dev, rng, xt, m, n, k, group, zeros, bias):  # noqa: F811
    raw, val, codes, sraw, sval, z, bv = random_case(rng, m, n, k, group, zeros, bias, xt)
    for yt in ("f32", "bf16"):
        check(product(dev, raw, codes, sraw, z, bv, xt, yt, group, k), val.astype(np.float64), weights(codes, sval, z, group), bv, yt, group)


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 14, 2.0 ** 20, 1e30])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("xt,m", [("bf16", 1), ("bf16", 5), ("f32", 1), ("f32", 5)])
def test_large_channels_over_zero_weights(dev, rng, xt, m, group, size):  # noqa: F811
    """A channel in every group that is far above the others and whose weights are zero adds nothing, also no error."""
    n, k = 64, 1024
    raw, val, codes, sraw, sval, z, _ = random_case(rng, m, n, k, group, 1, 0, xt)
    val = val.copy()
    q = np.stack([codes & 15, codes >> 4], -1).reshape(n, k)
    for c in range(group // 3, k, group):
        val[:, c] = size * rng.choice([-1.0, 1.0], m)
        q[:, c] = z[:, c // group]
    raw, val = store(val, xt)
    codes = (q[:, 0::2] | (q[:, 1::2] << 4)).astype(np.uint8)
    check(product(dev, raw, codes, sraw, z, None, xt, "f32", group, k), val.astype(np.float64), weights(codes, sval, z, group), None, "f32", group)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("xt,m", [("bf16", 1), ("bf16", 9), ("f32", 1), ("f32", 9)])
def test_identity_gives_every_bit_back(dev, rng, xt, m, group):  # noqa: F811
    """One weight of 1 per output: y is x, all 24 bits of it, over 60 orders of magnitude in one row."""
    k = 256
    raw, val = store(rng.standard_normal((m, k)) * 10.0 ** rng.uniform(-30, 30, (m, k)), xt)
    q = np.full((k, k), 8, np.uint8)
    q[np.arange(k), np.arange(k)] = 9
    codes = q[:, 0::2] | (q[:, 1::2] << 4)
    got = product(dev, raw, codes, store(np.ones((k, k // group)), "bf16")[0], None, None, xt, "f32", group, k)
    np.testing.assert_array_equal(got, val)


def test_products_that_fp32_sums_only_when_scaled(dev):  # noqa: F811
    """x near the type's largest under a small scale: no sum overflows on the way."""
    k, n = 256, 16
    x = np.full((1, k), 3e38, np.float32)
    codes = np.full((n, k // 2), 0xFF, np.uint8)
    s = np.full((n, k // 128), 2.0 ** -13, np.float32)
    got = product(dev, x, codes, store(s, "bf16")[0], None, None, "f32", "f32", 128, k)
    np.testing.assert_allclose(got, k * 7 * 3e38 * 2.0 ** -13, rtol=1e-5)


@pytest.mark.parametrize("xt", ["bf16", "f32"])
def test_infinities_of_both_signs(dev, xt):  # noqa: F811
    """As in IEEE arithmetic: inf - inf and inf x 0 are NaN, one sign alone is that infinity, other rows see nothing of it."""
    n, k = 16, 128
    x = np.ones((6, k), np.float32)
    x[0, 3], x[0, 77] = np.inf, -np.inf
    x[1, 3] = x[1, 77] = -np.inf
    x[2, 9] = np.inf                   # over a weight of 0
    x[3, 5] = np.inf                   # over a weight of -1
    raw, _ = store(np.where(np.isfinite(x), x, 0), xt)
    raw = raw.copy()
    for v, b16 in ((np.inf, 0x7F80), (-np.inf, 0xFF80)):
        raw[x == v] = b16 if xt == "bf16" else v
    q = np.full((n, k), 9, np.uint8)
    q[:, 9], q[:, 5] = 8, 7
    got = product(dev, raw, q[:, 0::2] | (q[:, 1::2] << 4), store(np.ones((n, 1)), "bf16")[0], None, None, xt, "f32", 128, k)
    assert np.isnan(got[0]).all() and np.isneginf(got[1]).all() and np.isnan(got[2]).all() and np.isneginf(got[3]).all()
    assert (got[4:] == k - 3).all()


def test_group_past_the_end_with_an_infinite_scale_before_it(dev, rng):  # noqa: F811
    """k ends inside a step of 128 columns: the missing columns take no scale, an infinite last one least of all."""
    n, k, group = 16, 96, 32
    x = np.ones((1, k), np.float32)
    s = np.ones((n, 3), np.float32)
    s[:, 2] = np.inf
    sraw = (s.view(np.uint32) >> 16).astype(np.uint16)
    got = product(dev, x, np.full((n, k // 2), 0x99, np.uint8), sraw, None, None, "f32", "f32", group, k)
    assert np.isposinf(got).all()
