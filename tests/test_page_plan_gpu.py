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
