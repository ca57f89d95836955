"""The host side of a paged cache against a context that only keeps books (no GPU needed): what it allocates, gives back and
uploads, and what is left of it when a call fails."""

import numpy as np
import pytest

from mdlc_b200 import _lib as L
from mdlc_b200 import paged


class Books:
    """Stands in for a Context: addresses that are handed out once, and a page plan after its definition."""

    def __init__(self):
        self.next, self.live, self.fail, self.plans, self.uploads = 1 << 20, {}, None, [], {}

    def alloc(self, nbytes):
        if self.fail is not None and nbytes >= self.fail:
            raise L.MdlcError(L.ERR_NOMEM, "alloc")
        self.next += 1 << 12
        self.live[self.next] = nbytes
        return self.next

    def free(self, p):
        del self.live[p]          # KeyError: not an allocation, or freed twice

    def to_device(self, a):
        p = self.alloc(a.nbytes)
        self.uploads[p] = np.array(a)
        return p

    def upload(self, p, a):
        assert a.nbytes <= self.live[p]
        self.uploads[p] = np.array(a)

    def download(self, p, shape, dtype):
        raise AssertionError("nothing is read back")

    def sync(self):
        pass

    def page_plan(self, desc, cached, new, free, count, table, *outs):
        self.plans.append((self.uploads[cached].tolist(), self.uploads[new].tolist(),
                           self.uploads[free].tolist()[:desc.free_pages] if desc.free_pages else []))

    def rope_append(self, *a):
        pass

    def paged_attn(self, desc, q, k, v, table, q_starts, kv_lens, out, lse, workspace):
        assert workspace in self.live and self.live[workspace] >= L.paged_attn_workspace(desc)

    def gemv_w4(self, desc, x, codes, scales, zeros, bias, y):
        assert codes in self.live and scales in self.live


def cache(books, **kw):
    args = dict(layers=1, batch=2, pages=40, page=4, heads=2, kv_heads=1, head_dim=8, max_tokens=64, max_len=64, dtype=L.F32)
    return paged.PagedCache(books, **{**args, **kw})


def test_workspace_that_cannot_grow():
    """No memory for a larger workspace: the freed one is not used again, and lengths and pages are as before."""
    b = Books()
    c = cache(b, heads=8, kv_heads=1, head_dim=64, pages=600, max_tokens=300, max_len=2048)
    c.plan([1, 1])
    before = c._room
    grown = L.paged_attn_workspace(c._attn(201, 200))
    assert grown > before
    b.fail = grown
    lens, free = c.lens.copy(), list(c.free)
    with pytest.raises(L.MdlcError):
        c.plan([200, 1])
    assert (c.lens == lens).all() and c.free == free and len(b.plans) == 1
    b.fail = None
    c.plan([1, 1])                # needs no more than the one that is gone
    c.attend(0, 1, 2)             # checks that its workspace is allocated
    c.close()
    assert not b.live


@pytest.mark.parametrize("place", [-1, -2, 2, 100])
def test_release_of_no_such_place(place):
    """Refused: a negative place would read in front of the block table."""
    b = Books()
    c = cache(b)
    c.plan([5, 6])
    with pytest.raises(ValueError):
        c.release(place)
    assert list(c.lens) == [5, 6] and len(c.free) == 40 - 4


@pytest.mark.parametrize("window,sinks", [(0, 0), (8, 0), (7, 0), (9, 5), (1, 1), (30, 4), (5, 100)])
def test_pages_behind_the_window_are_given_back(rng, window, sinks):
    """At every step a place holds exactly the pages of the keys that its next token can see (and with no window all), each page
    belongs to one place or the free list, and the plan is given the pages that the host counts as taken."""
    b, page = Books(), 4
    c = cache(b, batch=3, pages=60, window=window, sinks=sinks)
    for step in range(60):
        new = rng.integers(0, 4, 3)
        if step % 9 == 8:
            place = int(rng.integers(0, 3))
            c.release(place)
            assert not c.held[place] and c.lens[place] == 0
        new = np.minimum(new, c.max_len - c.lens)
        if not new.sum():
            continue
        cached, before = c.lens.copy(), [dict(h) for h in c.held]
        c.plan(new)
        given = iter(b.plans[-1][2])
        for i in range(3):
            first = [j for j in range(-(-int(c.lens[i]) // page)) if j not in before[i]]
            taken = [j for j in range(-(-int(cached[i]) // page), -(-int(c.lens[i]) // page))]
            assert set(taken) <= set(first) and [c.held[i][j] for j in taken] == [next(given) for _ in taken]
            # what this step's first token (position `cached`) sees is held, nothing else but the new tokens' pages
            seen = {j for j in range(-(-int(cached[i]) // page)) if not window or (j + 1) * page > cached[i] - window + 1 or j * page < sinks}
            assert set(c.held[i]) == seen | set(taken)
        assert next(given, None) is None
        ids = c.free + [p for h in c.held for p in h.values()]
        assert sorted(ids) == list(range(60))
    if window and window < 20 and sinks < 20:
        assert max(len(h) for h in c.held) <= (window + sinks) // page + 4


def test_layers_and_caches_free_what_they_hold():
    b = Books()
    layers = [paged.W4Linear(b, np.ones((8, 64), np.float32), bias, group=32, zeros=z) for bias in (None, np.ones(8)) for z in (True, False)]
    c = cache(b)
    c.plan([3, 4])
    for layer in layers:
        layer(1, 1, 2, L.F32)
        layer.close()
        layer.close()
        with pytest.raises(AssertionError):
            layer(1, 1, 2, L.F32)
    c.close()
    c.close()
    assert not b.live


@pytest.mark.parametrize("zeros", [True, False])
def test_quantize_w4_of_tiny_and_large_weights(rng, zeros):
    """Weights too small for a bf16 scale become 0, the largest ones stay finite, others beside them keep their own scale."""
    with np.errstate(all="raise", under="ignore"):
        for size in (1e-41, 1e-39, 1e-30, 3e38):
            w = rng.uniform(-1, 1, (3, 96)).astype(np.float32)
            w[1, 32:64] = rng.uniform(-1, 1, 32) * size
            codes, bits, z = paged.quantize_w4(w, 32, zeros)
            scale = (bits.astype(np.uint32) << 16).view(np.float32)
            assert np.isfinite(scale).all() and (scale > 0).all()
            got = paged.dequantize_w4(codes, bits, z).reshape(3, 3, 32)
            err = abs(got.astype(np.float64) - w.reshape(3, 3, 32)).max(-1)
            # a step or, in the group that has no scale, the weights themselves
            assert (err <= np.where(scale == 1, size, 1.01 * scale)).all()
    for bad in (np.nan, np.inf, -np.inf):
        w = np.zeros((2, 64), np.float32)
        w[1, 40] = bad
        with pytest.raises(ValueError):
            paged.quantize_w4(w, 32, zeros)
