"""Streams of a context: transfers, fences and events by stream id while a caller's stream is bound; captures."""

import ctypes as C

import numpy as np
import pytest

from mdlc_b200 import _lib as L

pytestmark = pytest.mark.gpu

COMPUTE, COPY = 0, 1


@pytest.fixture
def ctx():
    c = L.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("bound", [None, "legacy", "own"])
def test_stream_ids_while_a_stream_is_bound(ctx, bound):
    """Upload, fences both ways, events and download by id do their work on whatever the compute stream is, the legacy default
    stream (a null handle) among them."""
    torch = pytest.importorskip("torch")
    own = torch.cuda.Stream()
    if bound:
        ctx.bind_stream(0 if bound == "legacy" else own.cuda_stream)
    n = 1 << 16
    src, dst = ctx.host_alloc(4 * n), ctx.host_alloc(4 * n)
    a, b = (np.ctypeslib.as_array(C.cast(p, C.POINTER(C.c_float)), (n,)) for p in (src, dst))
    a[:], b[:] = np.arange(n), 0
    dev, back = ctx.alloc(4 * n), ctx.alloc(4 * n)
    d = L.CopyDesc(dtype=L.F32, in_cs=64, out_cs=64, mode=0, pad_mode=0, value=0.0)
    d.in_dims[:], d.out_dims[:] = [n // 64, 64, 1, 1], [n // 64, 64, 1, 1]
    d.src_dim[:], d.offset[:] = [0, 1, 2, 3], [0, 0, 0, 0]
    ctx.event_record(0, COMPUTE)
    ctx.upload_on(COPY, dev, src, 4 * n)
    ctx.fence_record(0, COPY)
    ctx.fence_wait(0, COMPUTE)
    ctx.copy4d(d, dev, back)
    ctx.fence_record(1, COMPUTE)
    ctx.fence_wait(1, COPY)
    ctx.download_on(COPY, dst, back, 4 * n)
    ctx.fence_record(2, COPY)
    ctx.fence_sync(2)
    assert (a == b).all()
    b[:] = 0
    ctx.upload_on(COMPUTE, dev, src, 4 * n)
    ctx.download_on(COMPUTE, dst, dev, 4 * n)
    ctx.event_record(1, COMPUTE)
    ctx.sync()
    assert (a == b).all() and ctx.event_elapsed(0, 1) >= 0
    if bound:
        ctx.unbind_stream()
    for bad in (2, -1, 7):
        with pytest.raises(L.MdlcError) as e:
            ctx.fence_record(3, bad)
        assert e.value.status == L.ERR_INVALID


def test_a_second_begin_leaves_the_capture_open(ctx):
    dev = ctx.alloc(256)
    ctx.memset(dev, 0, 256)
    ctx.graph_begin()
    ctx.memset(dev, 7, 256)
    with pytest.raises(L.MdlcError) as e:
        ctx.graph_begin()
    assert e.value.status == L.ERR_INVALID
    ctx.graph_end()
    ctx.graph_launch()
    assert (ctx.download(dev, 256, np.uint8) == 7).all()
    ctx.graph_reset()
    with pytest.raises(L.MdlcError):
        ctx.graph_end()
