"""Page plans from tables and free lists that are not in order, and from lengths that do not fit the token rows."""

import numpy as np
import pytest

from mdlc_b200 import _lib as L
from test_paged_gpu import ctx, dev  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def plan(dev, cached, new, free, table, page, tokens, flagged=False):
    """(table, q_starts, kv_lens, slots, positions, status); `flagged`: the call has to record an error."""
    c, (b, stride) = dev.ctx, table.shape
    i32 = lambda a: dev.put(np.asarray(a, np.int32))  # noqa: E731
    td, outs = i32(table), [dev.out(n, np.int32) for n in (b + 1, b, tokens, tokens, 2)]
    c.page_plan(L.PageDesc(batch=b, page=page, table_stride=stride, tokens=tokens, free_pages=len(free)), i32(cached), i32(new),
                i32(free) if len(free) else 0, 0, td, *outs)
    if flagged:
        with pytest.raises(L.MdlcError) as e:
            c.sync()
        assert e.value.status == L.ERR_DEVICE
    else:
        c.sync()
    return (c.download(td, table.shape, np.int32), *(c.download(o, (n,), np.int32) for o, n in zip(outs, (b + 1, b, tokens, tokens, 2))))


@pytest.mark.parametrize("page", [16, 7])
def test_ids_whose_slots_pass_32_bits(dev, page):  # noqa: F811
    """No slot of such an id, held or taken; the largest one that fits is whole; the other requests are not touched."""
    top = (2 ** 31 - 1) // page                      # its first slots fit, the last ones do not unless the page ends there
    big = [2 ** 28 if page == 16 else 2 ** 29, 2 ** 31 - 1, -1, -2 ** 31]
    for bad in big:
        table = np.array([[bad, -1], [3, -1], [5, -1]], np.int32)
        got = plan(dev, [2, 1, 0], [2, 2, 3], [bad], table, page, 7, flagged=True)
        slots = got[3].tolist()
        assert slots[:2] == [-1, -1] and slots[2:4] == [3 * page + 1, 3 * page + 2] and slots[4:] == [-1] * 3
        assert got[4].tolist() == [2, 3, 1, 2, 0, 1, 2] and got[2].tolist() == [4, 3, 3]
    whole = (2 ** 31) // page - 1                    # whole page below 2^31
    got = plan(dev, [0], [page], [whole], np.array([[-1]], np.int32), page, page)
    assert got[3].tolist() == list(range(whole * page, whole * page + page))
    if top > whole:                                  # the page that the limit cuts
        got = plan(dev, [0], [page], [top], np.array([[-1]], np.int32), page, page, flagged=True)
        assert got[3].tolist() == [s if s < 2 ** 31 else -1 for s in range(top * page, top * page + page)]


# the tokens that have a row, when the rows are fewer than the new tokens
CUTS = [([4, 0, 8], [4, 4, 0], 5), ([4, 0, 8], [4, 4, 9], 2), ([0] * 4, [3, 3, 3, 3], 7), ([1, 2, 3], [1, 1, 1], 3), ([5, 6], [0, 40], 1)]


@pytest.mark.parametrize("cached,new,tokens", CUTS)
def test_cut_requests_count_as_if_they_brought_their_rows(dev, cached, new, tokens):  # noqa: F811
    """The same plan as from the lengths that fit the rows: pages, key lengths, slots, positions and refusals."""
    page, stride = 4, 4
    left, fit = tokens, []
    for n in new:
        fit.append(min(n, left))
        left -= fit[-1]
    table = np.full((len(cached), stride), -1, np.int32)
    for b, c in enumerate(cached):
        table[b, :-(-c // page)] = 20 + 4 * b + np.arange(-(-c // page))
    for free in ([40, 41, 42, 43, 44, 45, 46, 47, 48], [40], []):
        got, want = (plan(dev, cached, n, free, table, page, tokens) for n in (new, fit))
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g, w)
        lens = np.diff(got[1])
        for b in range(len(cached)):
            if (got[3][got[1][b]:got[1][b + 1]] >= 0).all():       # accepted: its rows are the last of its keys, as attention places them
                assert got[2][b] == cached[b] + lens[b]
                np.testing.assert_array_equal(got[4][got[1][b]:got[1][b + 1]], got[2][b] - lens[b] + np.arange(lens[b]))


def test_many_cut_requests(dev, rng):  # noqa: F811
    """More requests than threads scan at a time, cut in the middle, free pages for the first part of them only."""
    b, page = 1500, 8
    cached, new = rng.integers(0, 30, b), rng.integers(0, 20, b)
    tokens = int(new.sum()) // 2
    start = np.minimum(np.concatenate([[0], np.cumsum(new)]), tokens)
    table = np.full((b, 8), -1, np.int32)
    held = -(-cached // page)
    ids = rng.permutation(10 ** 6)
    for i in range(b):
        table[i, :held[i]] = ids[8 * i:8 * i + held[i]]
    free = ids[8 * b:8 * b + 700]
    got, want = (plan(dev, cached, n, free, table, page, tokens) for n in (new, np.diff(start)))
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    assert 0 < got[5][1] and got[5][0] <= 700


def test_attention_over_a_cut_request(dev, rng):  # noqa: F811
    """Plan, cache write and attention of requests of which the last has rows for 3 of its 9 tokens: each token sees the keys up
    to its own position, and no slot that nobody wrote."""
    c, d, page, cached, new, tokens = dev.ctx, 64, 4, [5, 2], [4, 9], 7
    table = np.array([[0, 1, -1, -1], [2, -1, -1, -1]], np.int32)
    pages = 8
    td, qs, kv, sl, ps, stt = dev.put(table), *(dev.out(n, np.int32) for n in (3, 2, tokens, tokens, 2))
    c.page_plan(L.PageDesc(batch=2, page=page, table_stride=4, tokens=tokens, free_pages=5), dev.put(np.array(cached, np.int32)),
                dev.put(np.array(new, np.int32)), dev.put(np.arange(3, 8, dtype=np.int32)), 0, td, qs, kv, sl, ps, stt)
    kc = np.full((pages, 1, page, d), np.nan, np.float32)          # slots that nobody writes hold NaN
    vc = kc.copy()
    keys = [rng.standard_normal((2, n, d)).astype(np.float32) for n in (9, 5)]
    for b in range(2):
        for j in range(cached[b]):
            kc[table[b, j // page], 0, j % page], vc[table[b, j // page], 0, j % page] = keys[b][:, j]
    x = rng.standard_normal((tokens, 3, d)).astype(np.float32)
    for t in range(tokens):
        b, j = (0, 5 + t) if t < 4 else (1, 2 + t - 4)
        x[t, 1:] = keys[b][:, j]
    p, kd, vd, q, out = dev.put(x), dev.put(kc), dev.put(vc), dev.out((tokens, d), np.float32), dev.out((tokens, d), np.float32)
    rd = L.RopeDesc(tokens=tokens, heads=1, kv_heads=1, head_dim=d, rot_dim=0, axes=1, max_pos=64, page=page, pages=pages, dtype=L.F32,
                    q_stride=3 * d, k_stride=3 * d, v_stride=3 * d, out_stride=d)
    c.rope_append(rd, p, p + 4 * d, p + 8 * d, ps, dev.put(np.zeros((64, 1, 2), np.float32)), sl, q, kd, vd)
    ad = L.AttnDesc(batch=2, tokens=tokens, heads=1, kv_heads=1, head_dim=d, page=page, pages=pages, table_stride=4, max_q=9, max_kv=16, dtype=L.F32,
                    scale=0.125, q_stride=d, out_stride=d)
    c.paged_attn(ad, q, kd, vd, td, qs, kv, out, 0, dev.out(L.paged_attn_workspace(ad), np.uint8))
    c.sync()
    got = c.download(out, (tokens, d), np.float32)
    for t in range(tokens):
        b, j = (0, 5 + t) if t < 4 else (1, 2 + t - 4)
        k, v = keys[b][:, :j + 1].astype(np.float64)
        s = 0.125 * (k @ x[t, 0].astype(np.float64))
        w = np.exp(s - s.max())
        np.testing.assert_allclose(got[t], (w / w.sum()) @ v, atol=2e-5)
