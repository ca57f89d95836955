"""The paged decoder operators through the C ABI against plain forms in 64 bits.

Tolerances, from the formats (u = 2^-24: a rounding to fp32, relative; to bf16: 2 h with h = 2^-9):

* page plans are integers and must be equal;
* a rotated element x c - y s is two fp32 products, one sum and one rounding:
  |error| <= 4 u (|x| + |y|) + the output's own rounding (2 h |x'| in bf16);
* attention in bf16: the weights and the output are rounded to bf16, errors of both signs that partly cancel
  in the weighted mean: |error| <= 2.5 h max|v|; in fp32 the scores are off by at most d 2^-21 |q||k| scale
  (three tf32 products, each dropping 2^-22 of a product) plus the base-2 scaling's 2 u |s|, so the weights
  by as much relative, twice (weight and sum): |error| <= (2 eps_s + 64 u) max|v|, lse: eps_s + 8 u (1 + |lse|);
* 4-bit products: exact products and fp32 sums in a tree of at most k / 16 truncated steps per group:
  |error| <= 2^-23 (k / 16 + 16) sum |x w|; a bf16 output is one that some value within that
  distance rounds to.
"""

import math

import numpy as np
import pytest

from mdlc_b200 import _lib as L
from oracle import reference as oref

pytestmark = pytest.mark.gpu

U, H = 2.0 ** -24, 2.0 ** -9


def bits(x):
    return (oref.round_bf16(np.asarray(x, np.float32)).view(np.uint32) >> 16).astype(np.uint16)


def unbits(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def store(x, dtype):
    """(array to upload, the values it stands for) of fp32 x."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x, x
    b = bits(x)
    return b, unbits(b)


class Dev:
    """Device arrays of one test: uploaded values, poisoned outputs, freed at its end."""

    def __init__(self, ctx):
        self.ctx, self.made = ctx, []

    def put(self, arr):
        self.made.append(self.ctx.to_device(arr))
        return self.made[-1]

    def out(self, shape, dtype, fill=0xFF):
        n = int(np.prod(shape)) * np.dtype(dtype).itemsize
        self.made.append(self.ctx.alloc(max(n, 16)))
        self.ctx.memset(self.made[-1], fill, max(n, 16))
        return self.made[-1]

    def floats(self, p, shape, dtype):
        return self.ctx.download(p, shape, np.float32) if dtype == "f32" else unbits(self.ctx.download(p, shape, np.uint16))


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    ctx.sync()
    for p in d.made:
        ctx.free(p)


ET = {"bf16": L.BF16, "f32": L.F32}
RAW = {"bf16": np.uint16, "f32": np.float32}


# ------------------------------------------------------------------ page plans
def plan_definition(cached, new, free, n_free, table, page, tokens):
    table = table.copy()
    slots, positions = np.full(tokens, -1, np.int32), np.zeros(tokens, np.int32)
    starts, kv, asked, taken, refused = [0], [], 0, 0, 0
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        held, need = -(-c // page), -(-(c + n) // page)
        fits = need <= table.shape[1]
        first = asked
        asked += need - held if fits else 0
        ok = fits and (need == held or asked <= n_free)
        if ok:
            for j in range(held, need):
                table[b, j] = free[first + j - held]
            taken = max(taken, asked if need > held else 0)
        refused += not ok
        for i in range(n):
            t = starts[-1] + i
            if t < tokens:
                positions[t] = c + i
                slots[t] = table[b, (c + i) // page] * page + (c + i) % page if ok else -1
        starts.append(min(starts[-1] + n, tokens))
        kv.append(c + n if ok else c)
    return table, np.array(starts, np.int32), np.array(kv, np.int32), slots, positions, np.array([taken, refused], np.int32)


def run_plan(dev, cached, new, free, n_free, table, page, tokens, *, count_ptr=True, repeat=1):
    ctx, (b, stride) = dev.ctx, table.shape
    i32 = lambda a: dev.put(np.asarray(a, np.int32))  # noqa: E731
    td = i32(table)
    outs = [dev.out(n, np.int32) for n in (b + 1, b, tokens, tokens, 2)]
    d = L.PageDesc(batch=b, page=page, table_stride=stride, tokens=tokens, free_pages=len(free))
    fl, cl, nl, fc = i32(free) if len(free) else 0, i32(cached), i32(new), i32([n_free]) if count_ptr else 0
    for _ in range(repeat):
        ctx.page_plan(d, cl, nl, fl, fc, td, *outs)
    ctx.sync()
    return (ctx.download(td, table.shape, np.int32), *(ctx.download(o, (n,), np.int32) for o, n in zip(outs, (b + 1, b, tokens, tokens, 2))))


@pytest.mark.parametrize("batch,page,spread,pad,short", [
    (1, 16, 1, 0, 0), (1, 1, 40, 3, 0), (2, 1024, 3000, 0, 0), (64, 16, 1, 0, 0), (37, 7, 90, 11, 0),
    (513, 32, 60, 5, 0), (1025, 8, 9, 0, 0), (64, 16, 100, 2, 40), (300, 4, 30, 0, 900), (8192, 16, 2, 1, 0), (8192, 16, 3, 0, 300)])
def test_page_plan(dev, rng, batch, page, spread, pad, short):
    cached = rng.integers(0, 5 * page + 3, batch)
    new = rng.integers(0, spread + 1, batch)          # requests without new tokens among them
    need = -(-(cached + new) // page)
    stride = max(1, int(need.max()) - (1 if short else 0))   # with `short`, the longest do not fit their row either
    ids = rng.permutation(100000)[: int(need.sum()) + 7].astype(np.int32)
    table = np.full((batch, stride), -1, np.int32)
    at = 0
    for b in range(batch):
        h = min(-(-int(cached[b]) // page), stride)
        table[b, :h] = ids[at:at + h]
        at += h
    free = ids[at:]
    n_free = max(0, len(free) - short)
    tokens = max(1, int(new.sum()) + pad)
    got = run_plan(dev, cached, new, free, n_free, table, page, tokens, repeat=2)
    want = plan_definition(cached.tolist(), new.tolist(), free, n_free, table, page, tokens)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)


def test_page_plan_corners(dev):
    # no free page at all; negative lengths count as 0; more tokens than rows: the rest is cut
    table = np.array([[5, -1], [6, -1], [7, 8]], np.int32)
    for cached, new, free, tokens, ptr in (([3, -2, 8], [1, 0, -4], [], 4, False), ([4, 4, 4], [1, 1, 1], [9, 10], 3, True),
                                           ([4, 0, 8], [4, 4, 0], [9, 10, 11], 5, False)):
        got = run_plan(dev, cached, new, free, len(free), table, 4, tokens, count_ptr=ptr)
        want = plan_definition(cached, new, np.array(free, np.int32), len(free), table, 4, tokens)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g, w)


def test_page_plan_refuses(ctx):
    ok = dict(batch=2, page=16, table_stride=4, tokens=8, free_pages=3)
    for bad in (dict(batch=0), dict(batch=L.MAX_REQUESTS + 1), dict(page=0), dict(page=1025), dict(table_stride=0), dict(tokens=0),
                dict(free_pages=-1), dict(table_stride=2 ** 28, page=1024)):
        with pytest.raises(L.MdlcError) as e:
            ctx.page_plan(L.PageDesc(**{**ok, **bad}), *[256] * 10)
        assert e.value.status == L.ERR_INVALID
    for null in (0, 1, 2, 4, 9):
        args = [256] * 10
        args[null] = 0
        with pytest.raises(L.MdlcError):
            ctx.page_plan(L.PageDesc(**ok), *args)


# ------------------------------------------------------------------ rotation and cache write
def rope_definition(x, positions, table, sections, rot, interleaved):
    """x [t, h, d] float64; returns (rotated, bound of the fp32 arithmetic before the output's rounding)."""
    y, err, pair = x.copy(), np.zeros_like(x), 0
    for axis, n in enumerate(sections):
        for i in range(pair, pair + n):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
            c, s = (table[positions[axis], i, k].astype(np.float64)[:, None] for k in (0, 1))
            y[..., a] = x[..., a] * c - x[..., b] * s
            y[..., b] = x[..., b] * c + x[..., a] * s
            err[..., a] = err[..., b] = 4 * U * (abs(x[..., a]) + abs(x[..., b]))
        pair += n
    return y, err


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("t,h,kvh,d,rot,sections,inter,page,slack", [
    (1, 1, 1, 64, 64, [32], 0, 16, 0), (5, 8, 2, 128, 128, [16, 24, 24], 0, 16, 0), (7, 7, 1, 80, 80, [40], 0, 7, 0),
    (3, 4, 4, 96, 48, [4, 0, 10, 10], 0, 1, 0), (9, 4, 2, 64, 32, [16], 1, 32, 0), (2, 3, 1, 64, 0, [0], 0, 16, 0),
    (700, 6, 2, 64, 64, [32], 0, 64, 0), (1301, 28, 4, 128, 128, [10, 27, 27], 0, 32, 8), (33, 2, 1, 6, 2, [1], 1, 3, 1),
    (33, 5, 5, 30, 18, [4, 5], 0, 5, 3), (640, 3, 3, 24, 24, [12], 1, 8, 0), (1, 64, 8, 256, 256, [128], 0, 16, 0)])
def test_rope_append(dev, rng, dtype, t, h, kvh, d, rot, sections, inter, page, slack):
    """`slack`: elements between a token's packed heads and the next token's."""
    ctx, width = dev.ctx, (h + 2 * kvh) * d + slack
    raw, val = store(rng.standard_normal((t, width)), dtype)
    esz = raw.itemsize
    max_pos, pages = 61, -(-t // page) + 2
    table = rng.uniform(-1, 1, (max_pos, max(rot // 2, 1), 2)).astype(np.float32)
    pos = rng.integers(0, max_pos, (len(sections), t)).astype(np.int32)
    slots = rng.permutation(pages * page)[:t].astype(np.int32)
    slots[rng.random(t) < 0.15] = -1
    kc0, _ = store(rng.standard_normal((pages, kvh, page, d)), dtype)
    vc0, _ = store(rng.standard_normal((pages, kvh, page, d)), dtype)
    p, kc, vc = dev.put(raw), dev.put(kc0), dev.put(vc0)
    qo = dev.out((t, h * d + slack), RAW[dtype])
    desc = L.RopeDesc(tokens=t, heads=h, kv_heads=kvh, head_dim=d, rot_dim=rot, interleaved=inter, axes=len(sections), max_pos=max_pos,
                      page=page, pages=pages, dtype=ET[dtype], q_stride=width, k_stride=width, v_stride=width, out_stride=h * d + slack)
    desc.section[:len(sections)] = sections
    ctx.rope_append(desc, p, p + h * d * esz, p + (h + kvh) * d * esz, dev.put(pos), dev.put(table), dev.put(slots), qo, kc, vc)
    ctx.sync()
    x = val[:, :(h + 2 * kvh) * d].reshape(t, h + 2 * kvh, d).astype(np.float64)
    want, err = rope_definition(x[:, :h + kvh], pos, table, sections, rot, inter)
    err = err + (2 * H * abs(want) if dtype == "bf16" else U * abs(want))
    got = dev.floats(qo, (t, h * d + slack), dtype)
    assert (abs(got[:, :h * d].reshape(t, h, d) - want[:, :h]) <= err[:, :h]).all()
    for cache, before, lo, exact in ((kc, kc0, h, False), (vc, vc0, h + kvh, True)):
        after = ctx.download(cache, before.shape, RAW[dtype])
        flat, old = (a.transpose(0, 2, 1, 3).reshape(-1, kvh, d) for a in (after, before))
        live = slots[slots >= 0]
        rest = np.setdiff1d(np.arange(pages * page), live)
        np.testing.assert_array_equal(flat[rest], old[rest])
        mine = flat[live] if dtype == "f32" else unbits(flat[live])
        if exact:
            np.testing.assert_array_equal(mine, x[slots >= 0, lo:lo + kvh].astype(np.float32))
        else:
            assert (abs(mine - want[slots >= 0, lo:lo + kvh]) <= err[slots >= 0, lo:lo + kvh]).all()
    # in place: the queries where they lie
    ctx.rope_append(_with(desc, out_stride=width), p, p + h * d * esz,
                    p + (h + kvh) * d * esz, dev.put(pos), dev.put(table), dev.put(slots), p, kc, vc)
    ctx.sync()
    np.testing.assert_array_equal(dev.floats(p, (t, width), dtype)[:, :h * d], got[:, :h * d])


def _with(desc, **kw):
    new = type(desc).from_buffer_copy(bytes(desc))
    for k, v in kw.items():
        setattr(new, k, v)
    return new


def test_rope_append_checks_what_it_reads(dev, rng):
    """A position or slot outside its range is skipped and recorded; the other tokens are written."""
    ctx = dev.ctx
    t, d, page, pages, max_pos = 4, 64, 8, 2, 10
    x = rng.standard_normal((t, 3 * d)).astype(np.float32)
    p = dev.put(x)
    desc = L.RopeDesc(tokens=t, heads=1, kv_heads=1, head_dim=d, rot_dim=d, axes=1, max_pos=max_pos, page=page, pages=pages,
                      dtype=L.F32, q_stride=3 * d, k_stride=3 * d, v_stride=3 * d, out_stride=d)
    desc.section[0] = d // 2
    table = dev.put(np.stack([np.ones((max_pos, d // 2)), np.zeros((max_pos, d // 2))], -1).astype(np.float32))
    kc, vc, qo = (dev.out(s, np.float32, 0) for s in ((pages * page, d), (pages * page, d), (t, d)))
    ctx.rope_append(desc, p, p + d * 4, p + 2 * d * 4, dev.put(np.array([0, max_pos, -1, 3], np.int32)), table,
                    dev.put(np.array([0, 1, 2, pages * page], np.int32)), qo, kc, vc)
    with pytest.raises(L.MdlcError) as e:
        ctx.sync()
    assert e.value.status == L.ERR_DEVICE
    q, k = ctx.download(qo, (t, d), np.float32), ctx.download(kc, (pages * page, d), np.float32)
    np.testing.assert_array_equal(q, np.where(np.array([1, 0, 0, 1])[:, None], x[:, :d], 0))
    assert (k[0] == x[0, d:2 * d]).all() and not k[1:].any()


def test_rope_append_refuses(ctx):
    ok = dict(tokens=2, heads=4, kv_heads=2, head_dim=64, rot_dim=64, axes=1, max_pos=8, page=16, pages=4, dtype=L.BF16, q_stride=512,
              k_stride=512, v_stride=512, out_stride=256)

    def call(section=(32, 0, 0, 0), ptrs=(256,) * 9, **bad):
        d = L.RopeDesc(**{**ok, **bad})
        d.section[:] = section
        with pytest.raises(L.MdlcError) as e:
            ctx.rope_append(d, *ptrs)
        assert e.value.status == L.ERR_INVALID
    for bad in (dict(tokens=0), dict(heads=0), dict(kv_heads=0), dict(head_dim=257), dict(rot_dim=63), dict(rot_dim=66), dict(axes=0),
                dict(axes=5), dict(max_pos=0), dict(page=0), dict(pages=0), dict(interleaved=2), dict(dtype=L.S8), dict(q_stride=255),
                dict(k_stride=127), dict(v_stride=127), dict(out_stride=255), dict(pages=2 ** 28)):
        call(**bad)
    call(section=(31, 0, 0, 0))
    call(axes=2, section=(33, -1, 0, 0))
    for i in (0, 1, 2, 3, 4, 5, 7, 8):
        call(ptrs=tuple(0 if j == i else 256 for j in range(9)))
    call(ptrs=(257,) + (256,) * 8)


# ------------------------------------------------------------------ attention
def attn_definition(q, k, v, kv_len, window, sinks, scale):
    """q [n, h, d], k / v [kv_len, kvh, d] float64 -> out, lse."""
    n, h, d = q.shape
    g = h // max(k.shape[1], 1)
    j, p = np.arange(kv_len)[None], (kv_len - n + np.arange(n))[:, None]
    seen = (j <= p) & ((window == 0) | (j > p - window) | (j < sinks))
    out, lse = np.zeros_like(q), np.full((n, h), -np.inf)
    rows = seen.any(1)
    if not rows.any():
        return out, lse
    for i in range(h):
        s = np.where(seen, scale * (q[:, i] @ k[:, i // g].T), -np.inf)[rows]
        top = s.max(1, keepdims=True)
        w = np.exp(s - top)
        lse[rows, i] = (top + np.log(w.sum(1, keepdims=True)))[:, 0]
        out[rows, i] = (w / w.sum(1, keepdims=True)) @ v[:, i // g]
    return out, lse


def attn_case(dev, rng, dtype, cached, new, h, kvh, d, page, window=0, sinks=0, scale=None, q_slack=0, out_slack=0, lse=True,
              poison=True, kv_cut=None, sharp=1.0):
    """Runs one batch and checks it; returns out. Slots past a request's keys, pages no token sees and
    unassigned pages hold NaN, table entries behind the window an id that does not exist."""
    ctx, b = dev.ctx, len(cached)
    kv = [c + n for c, n in zip(cached, new)] if kv_cut is None else kv_cut
    scale = 1 / math.sqrt(d) if scale is None else scale
    need = [-(-x // page) for x in kv]
    pages, stride = sum(need) + 3, max(1, max(need)) + 1
    ids = rng.permutation(pages)
    fill = np.nan if poison else 0.0
    kc = np.full((pages, kvh, page, d), fill, np.float32)
    vc = np.full((pages, kvh, page, d), fill, np.float32)
    table = np.full((b, stride), -7 if poison else 0, np.int32)
    keys, at = [], 0
    for i, x in enumerate(kv):
        k, v = (store(rng.standard_normal((x, kvh, d)) * s, dtype)[1] for s in (sharp, 1.0))
        keys.append((k, v))
        lo = max(0, x - new[i] - window + 1) if window else 0
        for j in range(need[i]):
            a, e = j * page, min((j + 1) * page, x)
            if poison and e <= lo and a >= sinks:
                continue                     # a page behind the window, given back
            table[i, j] = ids[at]
            kc[ids[at], :, :e - a], vc[ids[at], :, :e - a] = k[a:e].transpose(1, 0, 2), v[a:e].transpose(1, 0, 2)
            at += 1
    tokens = sum(new)
    raw, val = store(rng.standard_normal((max(tokens, 1), h * d + q_slack)), dtype)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    desc = L.AttnDesc(batch=b, tokens=max(tokens, 1), heads=h, kv_heads=kvh, head_dim=d, page=page, pages=pages, table_stride=stride,
                      max_q=max(1, max(new)), max_kv=max(kv), window=window, sinks=sinks, dtype=ET[dtype], scale=scale,
                      q_stride=h * d + q_slack, out_stride=h * d + out_slack)
    ws = dev.out(L.paged_attn_workspace(desc), np.uint8)
    out, ls = dev.out((max(tokens, 1), h * d + out_slack), RAW[dtype]), dev.out((max(tokens, 1), h), np.float32)
    ctx.paged_attn(desc, dev.put(raw), dev.put(store(kc, dtype)[0]), dev.put(store(vc, dtype)[0]), dev.put(table), dev.put(starts),
                   dev.put(np.array(kv, np.int32)), out, ls if lse else 0, ws)
    ctx.sync()
    got = dev.floats(out, (max(tokens, 1), h * d + out_slack), dtype)
    gl = ctx.download(ls, (max(tokens, 1), h), np.float32)
    for i in range(b):
        if not new[i]:
            continue
        rows = slice(starts[i], starts[i + 1])
        k, v = (x.astype(np.float64) for x in keys[i])
        q = val[rows, :h * d].reshape(-1, h, d).astype(np.float64)
        want, wl = attn_definition(q, k, v, kv[i], window, sinks, scale)
        top_v = abs(v).max() if v.size else 1.0
        qk = math.sqrt((q ** 2).sum(-1).max() * ((k ** 2).sum(-1).max() if k.size else 0.0)) * abs(scale)
        eps = (d * 2.0 ** -21 if dtype == "f32" else d * 2.0 ** -23) * qk + 4 * U * qk
        tol = (2 * eps + 64 * U) * top_v if dtype == "f32" else (2.5 * H + 2 * eps) * top_v
        assert np.isfinite(got[rows, :h * d]).all()
        assert abs(got[rows, :h * d].reshape(-1, h, d) - want).max() <= tol, (i, abs(got[rows, :h * d].reshape(-1, h, d) - want).max(), tol)
        if lse:
            assert (np.isinf(gl[rows]) == np.isinf(wl)).all()
            fin = np.isfinite(wl)
            if fin.any():
                assert (abs(gl[rows][fin] - wl[fin]) <= eps + 8 * U * (1 + abs(wl[fin])) + 1e-6).all()
    return got, gl, starts


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cached,new,h,kvh,d,page", [
    ([0], [1], 1, 1, 64, 16),                                  # a first token sees itself alone
    ([700], [1], 8, 2, 128, 16), ([127], [1], 4, 4, 64, 128), ([1], [1], 6, 1, 80, 3), ([300], [1], 7, 1, 96, 32),
    ([0, 5, 130, 1000], [1, 1, 1, 1], 8, 1, 64, 16), ([33] * 9, [1] * 9, 16, 2, 128, 8),
    ([40], [3], 8, 1, 64, 16), ([40, 0], [7, 2], 16, 4, 128, 16), ([200], [4], 64, 4, 64, 64), ([5], [1], 64, 1, 32, 16),
    ([5], [1], 65, 1, 8, 16),                                  # more query heads than a row group has
    ([0], [70], 1, 1, 64, 16), ([0], [129], 4, 2, 128, 16), ([500], [257], 2, 2, 128, 64), ([3], [300], 5, 1, 72, 7),
    ([1000, 0, 17, 255, 256], [1, 64, 1, 200, 33], 8, 2, 128, 32), ([10, 20, 30], [1, 0, 100], 4, 1, 64, 16),
    ([0, 0, 0], [40, 1, 90], 12, 12, 64, 16), ([4000], [1], 8, 8, 64, 256), ([2047], [129], 7, 1, 128, 128)])
def test_paged_attn(dev, rng, dtype, cached, new, h, kvh, d, page):
    attn_case(dev, rng, dtype, cached, new, h, kvh, d, page)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cached,new,h,kvh,d,page,window,sinks", [
    ([900], [1], 8, 2, 64, 16, 100, 4), ([900], [1], 8, 2, 128, 16, 1, 0), ([900], [1], 8, 2, 64, 16, 1, 1),
    ([900, 3, 60], [1, 1, 1], 4, 1, 128, 16, 64, 17), ([900], [150], 8, 2, 64, 16, 130, 4), ([900], [300], 4, 4, 128, 32, 7, 40),
    ([900], [300], 4, 1, 64, 16, 5000, 9), ([0], [400], 2, 1, 64, 8, 33, 0), ([2000, 100, 0], [1, 280, 90], 6, 2, 96, 16, 256, 130),
    ([700], [5], 4, 4, 64, 16, 40, 700), ([1500], [200], 8, 1, 128, 64, 1000, 300)])
def test_paged_attn_window(dev, rng, dtype, cached, new, h, kvh, d, page, window, sinks):
    attn_case(dev, rng, dtype, cached, new, h, kvh, d, page, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cached,new,kv", [([0], [5], [3]), ([0, 0], [1, 200], [0, 150]), ([0, 4], [1, 90], [0, 0]), ([0], [64], [1])])
def test_paged_attn_rows_without_keys(dev, rng, dtype, cached, new, kv):
    """Fewer keys than new tokens: the first rows see nothing and give 0 and -inf."""
    got, lse, starts = attn_case(dev, rng, dtype, cached, new, 4, 2, 64, 16, kv_cut=kv)
    for i, (n, x) in enumerate(zip(new, kv)):
        empty = slice(starts[i], starts[i] + max(0, n - x))
        assert not got[empty].any() and np.isneginf(lse[empty]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_paged_attn_strides_scale_and_no_lse(dev, rng, dtype):
    attn_case(dev, rng, dtype, [100, 30], [1, 150], 4, 2, 64, 16, q_slack=3 * 64, out_slack=8)
    attn_case(dev, rng, dtype, [100, 30], [1, 150], 4, 2, 128, 16, scale=0.5, lse=False)
    attn_case(dev, rng, dtype, [100, 30], [1, 150], 4, 2, 64, 16, scale=0.0)
    attn_case(dev, rng, dtype, [100, 30], [1, 150], 4, 2, 64, 16, scale=-0.3)
    attn_case(dev, rng, dtype, [900, 30], [1, 250], 4, 2, 128, 16, sharp=12.0)   # nearly all weight on few keys


def test_paged_attn_no_such_page(dev, rng):
    """An id outside the cache hides its keys and is recorded; the call stays in bounds."""
    ctx, d, page = dev.ctx, 64, 16
    for new in (1, 150):
        kv = 150 + 40
        q, k, v = (store(rng.standard_normal(s), "f32")[0] for s in ((new, d), (12, page, d), (12, page, d)))
        table = np.arange(12, dtype=np.int32)[None].copy()
        table[0, 2], table[0, 4] = 12, -1
        desc = L.AttnDesc(batch=1, tokens=new, heads=1, kv_heads=1, head_dim=d, page=page, pages=12, table_stride=12, max_q=new, max_kv=kv,
                          dtype=L.F32, scale=0.125, q_stride=d, out_stride=d)
        out = dev.out((new, d), np.float32)
        ctx.paged_attn(desc, dev.put(q), dev.put(k), dev.put(v), dev.put(table), dev.put(np.array([0, new], np.int32)),
                       dev.put(np.array([kv], np.int32)), out, 0, dev.out(L.paged_attn_workspace(desc), np.uint8))
        with pytest.raises(L.MdlcError):
            ctx.sync()
        got = ctx.download(out, (new, d), np.float32)
        kk, vv = (x.reshape(-1, d)[:kv].astype(np.float64) for x in (k, v))
        j, p = np.arange(kv)[None], (kv - new + np.arange(new))[:, None]
        seen = (j <= p) & (j // page != 2) & (j // page != 4)
        s = np.where(seen, 0.125 * (q.astype(np.float64) @ kk.T), -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        np.testing.assert_allclose(got, (w / w.sum(1, keepdims=True)) @ vv, atol=1e-4)


@pytest.mark.parametrize("bad", [12, -1, -2, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_paged_attn_no_such_page_ids(dev, rng, dtype, new, bad):
    """Every id outside the cache is recorded and its keys hidden, whatever its value, in every type and form."""
    ctx, d, page, kv = dev.ctx, 64, 16, 190
    (q, qv), (k, kval), (v, vval) = (store(rng.standard_normal(s), dtype) for s in ((new, d), (12, page, d), (12, page, d)))
    table = np.arange(12, dtype=np.int32)[None].copy()
    table[0, 3] = bad
    desc = L.AttnDesc(batch=1, tokens=new, heads=1, kv_heads=1, head_dim=d, page=page, pages=12, table_stride=12, max_q=new, max_kv=kv,
                      dtype=ET[dtype], scale=0.125, q_stride=d, out_stride=d)
    out = dev.out((new, d), RAW[dtype])
    ctx.paged_attn(desc, dev.put(q), dev.put(k), dev.put(v), dev.put(table), dev.put(np.array([0, new], np.int32)),
                   dev.put(np.array([kv], np.int32)), out, 0, dev.out(L.paged_attn_workspace(desc), np.uint8))
    with pytest.raises(L.MdlcError):
        ctx.sync()
    got = dev.floats(out, (new, d), dtype)
    kk, vv = (x.reshape(-1, d)[:kv].astype(np.float64) for x in (kval, vval))
    j, p = np.arange(kv)[None], (kv - new + np.arange(new))[:, None]
    s = np.where((j <= p) & (j // page != 3), 0.125 * (qv.astype(np.float64) @ kk.T), -np.inf)
    w = np.exp(s - s.max(1, keepdims=True))
    qk = 0.125 * math.sqrt((qv.astype(np.float64) ** 2).sum(-1).max() * (kk ** 2).sum(-1).max())
    eps = (d * 2.0 ** -21 if dtype == "f32" else d * 2.0 ** -23) * qk + 4 * U * qk
    tol = ((2 * eps + 64 * U) if dtype == "f32" else (2.5 * H + 2 * eps)) * abs(vv).max()
    assert abs(got - (w / w.sum(1, keepdims=True)) @ vv).max() <= tol


def test_paged_attn_refuses(ctx):
    ok = dict(batch=2, tokens=4, heads=8, kv_heads=2, head_dim=64, page=16, pages=9, table_stride=4, max_q=2, max_kv=60, dtype=L.BF16,
              scale=0.1, q_stride=512, out_stride=512)
    for bad in (dict(batch=0), dict(batch=L.MAX_REQUESTS + 1), dict(tokens=0), dict(heads=0), dict(kv_heads=3), dict(head_dim=0), dict(head_dim=60),
                dict(head_dim=136), dict(page=0), dict(page=1025), dict(pages=0), dict(table_stride=0), dict(max_q=0), dict(max_kv=-1),
                dict(window=-1), dict(sinks=-1), dict(dtype=L.S8), dict(q_stride=504), dict(out_stride=516), dict(pages=2 ** 27)):
        d = L.AttnDesc(**{**ok, **bad})
        with pytest.raises(L.MdlcError) as e:
            ctx.paged_attn(d, *[256] * 9)
        assert e.value.status == L.ERR_INVALID
        with pytest.raises(L.MdlcError):
            L.paged_attn_workspace(d)
    for i in (0, 1, 2, 3, 4, 5, 6, 8):
        with pytest.raises(L.MdlcError):
            ctx.paged_attn(L.AttnDesc(**ok), *[0 if j == i else 256 for j in range(9)])
    for i in (0, 1, 2, 6, 8):
        with pytest.raises(L.MdlcError):
            ctx.paged_attn(L.AttnDesc(**ok), *[264 if j == i else 256 for j in range(9)])


# ------------------------------------------------------------------ 4-bit products
@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("m,n,k,group,zeros,bias,slack", [
    (1, 1, 32, 32, 0, 0, 0), (1, 16, 128, 128, 0, 1, 0), (1, 33, 96, 32, 1, 0, 8), (2, 100, 64, 64, 1, 1, 0), (3, 47, 192, 64, 0, 1, 16),
    (5, 250, 2912, 32, 1, 1, 0), (8, 513, 1152, 128, 1, 0, 0), (9, 64, 4096, 128, 0, 0, 24), (16, 31, 320, 64, 1, 1, 0),
    (17, 40, 256, 32, 0, 1, 0), (32, 129, 384, 128, 1, 1, 8), (33, 18, 128, 32, 1, 0, 0), (70, 20, 640, 128, 0, 1, 0), (1, 9600, 1024, 128, 1, 1, 0),
    (4, 9700, 544, 32, 1, 0, 0)])
def test_gemv_w4(dev, rng, xt, yt, m, n, k, group, zeros, bias, slack):
    ctx, groups = dev.ctx, k // group
    raw, val = store(rng.standard_normal((m, k + slack)) * np.where(rng.random(k + slack) < 0.02, 30, 1), xt)
    codes = rng.integers(0, 256, (n, k // 2)).astype(np.uint8)
    sraw, sval = store(rng.uniform(0.002, 0.03, (n, groups)), "bf16")
    z = rng.integers(0, 16, (n, groups)).astype(np.uint8) if zeros else None
    bv = rng.standard_normal(n).astype(np.float32) if bias else None
    y = dev.out((m, n + slack), RAW[yt])
    d = L.W4Desc(m=m, n=n, k=k, group=group, x_type=ET[xt], y_type=ET[yt], x_stride=k + slack, y_stride=n + slack)
    ctx.gemv_w4(d, dev.put(raw), dev.put(codes), dev.put(sraw), dev.put(z) if zeros else 0, dev.put(bv) if bias else 0, y)
    ctx.sync()
    q = np.stack([codes & 15, codes >> 4], -1).reshape(n, groups, group).astype(np.float64)
    w = ((q - (z[..., None] if zeros else 8)) * sval[..., None].astype(np.float64)).reshape(n, k)
    x = val[:, :k].astype(np.float64)
    want = x @ w.T + (bv if bias else 0)
    mag = abs(x) @ abs(w).T + (abs(bv) if bias else 0)
    tol = 2.0 ** -23 * (k / 16 + 16) * mag
    got = dev.floats(y, (m, n + slack), yt)
    lo, hi = want - tol, want + tol
    if yt == "bf16":
        lo, hi = (oref.round_bf16(v.astype(np.float32)) for v in (lo, hi))
    assert ((got[:, :n] >= lo) & (got[:, :n] <= hi)).all()
    if slack:   # between rows: untouched
        assert (ctx.download(y, (m, n + slack), RAW[yt])[:, n:].view(np.uint8) == 0xFF).all()


def test_gemv_w4_infinite_and_nan_inputs(dev):
    ctx, n, k = dev.ctx, 16, 128
    x = np.ones((3, k), np.float32)
    x[0, 5], x[1, 7], x[2, 3] = np.inf, np.nan, np.finfo(np.float32).max
    codes = np.full((n, k // 2), 0x99, np.uint8)
    s = dev.put(store(np.ones((n, 1)), "bf16")[0])
    y = dev.out((3, n), np.float32)
    ctx.gemv_w4(L.W4Desc(m=3, n=n, k=k, group=128, x_type=L.F32, y_type=L.F32, x_stride=k, y_stride=n), dev.put(x), dev.put(codes), s, 0, 0, y)
    ctx.sync()
    got = ctx.download(y, (3, n), np.float32)
    assert np.isposinf(got[0]).all() and np.isnan(got[1]).all()
    np.testing.assert_allclose(got[2], np.finfo(np.float32).max, rtol=1e-6)


def test_gemv_w4_refuses(ctx):
    ok = dict(m=1, n=16, k=128, group=128, x_type=L.BF16, y_type=L.BF16, x_stride=128, y_stride=16)
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(k=120), dict(group=16), dict(group=256, k=256), dict(x_type=L.S8), dict(y_type=L.U8),
                dict(x_stride=120), dict(x_stride=132), dict(y_stride=15)):
        with pytest.raises(L.MdlcError) as e:
            ctx.gemv_w4(L.W4Desc(**{**ok, **bad}), *[256] * 6)
        assert e.value.status == L.ERR_INVALID
    with pytest.raises(L.MdlcError) as e:
        ctx.gemv_w4(L.W4Desc(**{**ok, "m": 70000}), *[256] * 6)
    assert e.value.status == L.ERR_UNSUPPORTED
    for i in (0, 1, 2, 5):
        with pytest.raises(L.MdlcError):
            ctx.gemv_w4(L.W4Desc(**ok), *[0 if j == i else 256 for j in range(6)])
    for i in (0, 1):
        with pytest.raises(L.MdlcError):
            ctx.gemv_w4(L.W4Desc(**ok), *[264 if j == i else 256 for j in range(6)])


# ------------------------------------------------------------------ streams, capture
def test_bound_stream_orders_with_a_caller(ctx, rng):
    """Work issued on a bound stream sees what a caller's kernels on that stream wrote just before."""
    torch = pytest.importorskip("torch")
    s = torch.cuda.Stream()
    n, k = 256, 256
    codes = torch.full((n, k // 2), 0x99, dtype=torch.uint8, device="cuda")   # weight 1
    scales = torch.ones((n, k // 128), dtype=torch.bfloat16, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    d = L.W4Desc(m=1, n=n, k=k, group=128, x_type=L.F32, y_type=L.F32, x_stride=k, y_stride=n)
    for stream in (s, torch.cuda.default_stream()):
        ctx.bind_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            for i in range(1, 4):
                y = torch.zeros((1, n), device="cuda")
                x = (big @ big)[:1, :k] * 0 + i         # a slow producer
                x = x.contiguous()
                ctx.gemv_w4(d, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), 0, 0, y.data_ptr())
                z = y + 1                               # a consumer on the caller's stream
                assert (z == i * k + 1).all()
        ctx.unbind_stream()
    assert ctx.lib.mdlc_unbind_stream(ctx.h) == L.OK    # nothing bound: nothing to do


def test_capture_replays_with_new_lengths(dev, rng):
    """Plan and attention captured once replay with other lengths, tables and slots on the device."""
    ctx, d, page, kvh, h, b, stride = dev.ctx, 64, 16, 2, 4, 3, 8
    pages = b * stride
    kc, vc = (rng.standard_normal((pages, kvh, page, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((b, h, d)).astype(np.float32)
    table = np.full((b, stride), -1, np.int32)
    lens = dev.out(b, np.int32, 0)
    one, free = dev.put(np.ones(b, np.int32)), dev.put(np.arange(pages, dtype=np.int32))
    td, qs, kv, sl, ps, stt = dev.put(table), *(dev.out(n, np.int32) for n in (b + 1, b, b, b, 2))
    pd = L.PageDesc(batch=b, page=page, table_stride=stride, tokens=b, free_pages=pages)
    ad = L.AttnDesc(batch=b, tokens=b, heads=h, kv_heads=kvh, head_dim=d, page=page, pages=pages, table_stride=stride, max_q=1,
                    max_kv=stride * page, dtype=L.F32, scale=0.125, q_stride=h * d, out_stride=h * d)
    ws, out = dev.out(L.paged_attn_workspace(ad), np.uint8), dev.out((b, h, d), np.float32)
    args = (dev.put(q), dev.put(kc), dev.put(vc), td, qs, kv, out, 0, ws)
    ctx.graph_begin()
    ctx.page_plan(pd, lens, one, free, 0, td, qs, kv, sl, ps, stt)
    ctx.paged_attn(ad, *args)
    ctx.graph_end()
    for cached in ([0, 0, 0], [100, 3, 15], [16, 127, 40]):
        held = [-(-c // page) for c in cached]
        t0 = np.full((b, stride), -1, np.int32)
        ids = np.arange(pages)[::-1]
        for i in range(b):
            t0[i, :held[i]] = ids[i * stride:i * stride + held[i]]
        ctx.upload(td, t0)
        ctx.upload(lens, np.array(cached, np.int32))
        ctx.graph_launch()
        ctx.sync()
        t1 = ctx.download(td, t0.shape, np.int32)
        got = ctx.download(out, (b, h, d), np.float32)
        for i in range(b):
            n = cached[i] + 1
            k, v = (c[t1[i, :-(-n // page)]].transpose(0, 2, 1, 3).reshape(-1, kvh, d)[:n].astype(np.float64) for c in (kc, vc))
            want, _ = attn_definition(q[i:i + 1].astype(np.float64), k, v, n, 0, 0, 0.125)
            np.testing.assert_allclose(got[i], want[0], atol=2e-5)
    ctx.graph_reset()


def test_same_call_same_bits(dev, rng):
    """No result depends on the order in which blocks finish."""
    ctx, d = dev.ctx, 128
    kvh, h, page, kv = 2, 8, 16, 3000
    pages = -(-kv // page)
    desc = L.AttnDesc(batch=1, tokens=1, heads=h, kv_heads=kvh, head_dim=d, page=page, pages=pages, table_stride=pages, max_q=1, max_kv=kv,
                      dtype=L.F32, scale=0.1, q_stride=h * d, out_stride=h * d)
    ws, out = dev.out(L.paged_attn_workspace(desc), np.uint8), dev.out((h, d), np.float32)
    args = [dev.put(rng.standard_normal(s).astype(np.float32)) for s in ((h, d), (pages, kvh, page, d), (pages, kvh, page, d))]
    args += [dev.put(np.arange(pages, dtype=np.int32)), dev.put(np.array([0, 1], np.int32)), dev.put(np.array([kv], np.int32)), out, 0, ws]
    seen = set()
    for _ in range(20):
        ctx.paged_attn(desc, *args)
        ctx.sync()
        seen.add(ctx.download(out, (h, d), np.float32).tobytes())
    assert len(seen) == 1
