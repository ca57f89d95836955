"""Decodes and chunks in one attention call: the two run beside each other, behind the work that wrote their inputs and in front of
the work that reads their outputs or overwrites their inputs, on a plain stream and in a captured graph."""

import numpy as np
import pytest

from mdlc_b200 import _lib as L
from test_paged_gpu import ET, H, RAW, U, attn_definition, ctx, dev, store  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu

PAGE, KVH, G, STRIDE = 16, 2, 4, 160
CACHED, NEW = [2300, 40, 0, 900, 17], [1, 150, 70, 1, 1]


class Step:
    """Rotation (by angle 0) with cache write of fixed lengths, then attention, over buffers that `fill` changes."""

    def __init__(self, dev, dtype, d):
        self.dev, self.dtype, self.d, self.h = dev, dtype, d, KVH * G
        ctx, b, t = dev.ctx, len(NEW), sum(NEW)
        width, pages = (self.h + 2 * KVH) * d, b * STRIDE
        self.table = np.arange(pages, dtype=np.int32).reshape(b, STRIDE)
        slots = [self.table[i, p // PAGE] * PAGE + p % PAGE for i in range(b) for p in range(CACHED[i], CACHED[i] + NEW[i])]
        self.qkv, self.qo = dev.out((t, width), RAW[dtype]), dev.out((t, self.h * d), RAW[dtype])
        self.kc, self.vc = (dev.out((pages, KVH, PAGE, d), RAW[dtype]) for _ in range(2))
        self.out = dev.out((t, self.h, d), RAW[dtype])
        self.starts = np.concatenate([[0], np.cumsum(NEW)]).astype(np.int32)
        self.kv = np.array(CACHED, np.int32) + np.array(NEW, np.int32)
        cs = np.stack([np.ones((4, d // 2)), np.zeros((4, d // 2))], -1).astype(np.float32)
        esz = np.dtype(RAW[dtype]).itemsize
        rd = L.RopeDesc(tokens=t, heads=self.h, kv_heads=KVH, head_dim=d, rot_dim=d, axes=1, max_pos=4, page=PAGE, pages=pages, dtype=ET[dtype],
                        q_stride=width, k_stride=width, v_stride=width, out_stride=self.h * d)
        rd.section[0] = d // 2
        ad = L.AttnDesc(batch=b, tokens=t, heads=self.h, kv_heads=KVH, head_dim=d, page=PAGE, pages=pages, table_stride=STRIDE, max_q=max(NEW),
                        max_kv=int(self.kv.max()), dtype=ET[dtype], scale=0.125, q_stride=self.h * d, out_stride=self.h * d)
        rope = (rd, self.qkv, self.qkv + self.h * d * esz, self.qkv + (self.h + KVH) * d * esz, dev.put(np.zeros(t, np.int32)), dev.put(cs),
                dev.put(np.array(slots, np.int32)), self.qo, self.kc, self.vc)
        attn = (ad, self.qo, self.kc, self.vc, dev.put(self.table), dev.put(self.starts), dev.put(self.kv), self.out, 0,
                dev.out(L.paged_attn_workspace(ad), np.uint8))
        self.issue = lambda: (ctx.rope_append(*rope), ctx.paged_attn(*attn))
        self.width = width

    def values(self, rng):
        """(device copies of) new inputs, and the values that they stand for."""
        t, d = sum(NEW), self.d
        qkv, vq = store(rng.standard_normal((t, self.width)), self.dtype)
        caches = [store(rng.standard_normal((len(NEW) * STRIDE, KVH, PAGE, d)), self.dtype) for _ in range(2)]
        return (qkv, caches[0][0], caches[1][0]), (vq, caches[0][1], caches[1][1])

    def check(self, got, vals):
        vq, k, v = vals
        x = vq.reshape(-1, self.h + 2 * KVH, self.d).astype(np.float64)
        k, v = k.copy(), v.copy()
        for i in range(len(NEW)):
            rows = slice(self.starts[i], self.starts[i + 1])
            for r in range(NEW[i]):
                p = CACHED[i] + r
                at = self.table[i, p // PAGE], slice(None), p % PAGE
                k[at], v[at] = x[rows][r, self.h:self.h + KVH], x[rows][r, self.h + KVH:]
            ki, vi = (c[self.table[i]].transpose(0, 2, 1, 3).reshape(-1, KVH, self.d)[:self.kv[i]].astype(np.float64) for c in (k, v))
            want, _ = attn_definition(x[rows, :self.h], ki, vi, int(self.kv[i]), 0, 0, 0.125)
            # 64 roundings in fp32; in bf16 the weights' and the output's
            tol = (64 * U if self.dtype == "f32" else 2.5 * H) * abs(vi).max() + 1e-5
            assert abs(got[rows] - want).max() <= tol


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_mixed_calls_are_ordered(dev, rng, dtype, d, captured):  # noqa: F811
    ctx, s = dev.ctx, Step(dev, dtype, d)
    sets = [s.values(rng) for _ in range(3)]
    staged = [[dev.put(a) for a in raw] for raw, _ in sets]
    kept = [dev.out((sum(NEW), s.h, d), RAW[dtype]) for _ in sets]
    ident = []
    for dst, src in ((s.qkv, 0), (s.kc, 1), (s.vc, 2)):
        n = sets[0][0][src].size
        ident.append((dst, src, _copy(n, dtype)))
    back = _copy(sum(NEW) * s.h * d, dtype)
    if captured:
        ctx.graph_begin()
        s.issue()
        ctx.graph_end()
    for i in range(3):   # nothing waits on the host in between: inputs are overwritten right behind the call that reads them
        for dst, src, desc in ident:
            ctx.copy4d(desc, staged[i][src], dst)
        ctx.graph_launch() if captured else s.issue()
        ctx.copy4d(back, s.out, kept[i])
    ctx.sync()
    for (_, vals), out in zip(sets, kept):
        s.check(dev.floats(out, (sum(NEW), s.h, d), dtype), vals)
    if captured:
        ctx.graph_reset()


def _copy(n, dtype):
    rows = n // 64
    d = L.CopyDesc(dtype=ET[dtype], in_cs=64, out_cs=64, mode=0, pad_mode=0, value=0.0)
    d.in_dims[:] = [rows, 64, 1, 1]
    d.out_dims[:] = [rows, 64, 1, 1]
    d.src_dim[:] = [0, 1, 2, 3]
    d.offset[:] = [0, 0, 0, 0]
    return d


@pytest.mark.parametrize("bound", [False, True])
def test_mixed_call_in_a_capture_of_the_callers(dev, rng, bound):  # noqa: F811
    """The side stream joins a capture that the caller began on its own, bound stream, and leaves it again."""
    torch = pytest.importorskip("torch")
    ctx, s = dev.ctx, Step(dev, "bf16", 64)
    raw, vals = s.values(rng)
    for dst, a in zip((s.qkv, s.kc, s.vc), raw):
        ctx.upload(dst, a)
    if bound:
        stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        ctx.bind_stream(stream.cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            s.issue()
        g.replay()
        torch.cuda.synchronize()
        ctx.unbind_stream()
    else:
        s.issue()
    ctx.sync()
    s.check(dev.floats(s.out, (sum(NEW), s.h, s.d), "bf16"), vals)
