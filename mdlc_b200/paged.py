"""Host side of the paged decoder operators (``include/mdlc_b200.h``): the caches of a
decoder with their page bookkeeping, 4-bit weights, and rotation tables.

A step of a decoder is one :meth:`PagedCache.plan` (block tables, slots and positions
built on the GPU), then per layer :class:`W4Linear` projections, :meth:`PagedCache.append`
(rotation and cache write) and :meth:`PagedCache.attend`. The kernels are asynchronous on the
context's stream; ``plan`` uploads the step's lengths, which waits for it.
"""

from __future__ import annotations

import math

import numpy as np

from mdlc_b200 import _lib as L


def rope_table(max_pos: int, rot_dim: int, base: float = 10000.0) -> np.ndarray:
    """``[max_pos][rot_dim / 2][2]`` fp32 cosines and sines of ``pos * base^(-2 i / rot_dim)``, computed in fp64."""
    inv = base ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    angle = np.arange(max_pos, dtype=np.float64)[:, None] * inv[None]
    return np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)


def _bf16_bits(x: np.ndarray) -> np.ndarray:
    """fp32 -> bf16 bits, round to nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def quantize_w4(w: np.ndarray, group: int = 128, zeros: bool = True):
    """4-bit codes of ``w`` ([n, k]) with one bf16 scale per row and ``group`` columns.

    With ``zeros`` the codes span each group's [min, max] (0 included) around a zero point,
    else [-8, 7] times the scale around 8. Returns (codes [n, k / 2] uint8, scale bits
    [n, k / group] uint16, zero points [n, k / group] uint8 or None) as ``mdlc_gemv_w4`` reads them."""
    n, k = w.shape
    if k % group:
        raise ValueError(f"k = {k} is not a multiple of the group {group}")
    g = np.asarray(w, np.float32).reshape(n, k // group, group)
    if not np.isfinite(g).all():
        raise ValueError("weights that are not finite")
    if zeros:
        lo, hi = np.minimum(g.min(-1), 0), np.maximum(g.max(-1), 0)
        scale = hi / 15 - lo / 15
    else:
        scale = np.maximum(g.max(-1) / 7, -g.min(-1) / 8)
    bits = _bf16_bits(scale)
    bits = np.where(bits < 0x80, _bf16_bits(np.ones(1)), bits)   # all 0, or too small for a (normal) scale: every code stands for 0
    s = (bits.astype(np.uint32) << 16).view(np.float32)
    z = np.clip(np.rint(-lo / s), 0, 15) if zeros else np.full(s.shape, 8.0, np.float32)
    q = np.clip(np.rint(g / s[..., None]) + z[..., None], 0, 15).astype(np.uint8).reshape(n, k)
    return q[:, 0::2] | (q[:, 1::2] << 4), bits, z.astype(np.uint8) if zeros else None


def dequantize_w4(codes: np.ndarray, scale_bits: np.ndarray, zeros=None) -> np.ndarray:
    """The [n, k] fp32 weights that the codes stand for."""
    n, groups = scale_bits.shape
    q = np.stack([codes & 15, codes >> 4], -1).reshape(n, groups, -1).astype(np.float32)
    z = 8.0 if zeros is None else zeros[..., None].astype(np.float32)
    return ((q - z) * (scale_bits.astype(np.uint32) << 16).view(np.float32)[..., None]).reshape(n, -1)


class W4Linear:
    """``y = x W^T (+ bias)`` with 4-bit weights on the device."""

    def __init__(self, ctx: L.Context, w: np.ndarray, bias=None, *, group: int = 128, zeros: bool = True):
        self.ctx, (self.n, self.k), self.group = ctx, w.shape, group
        codes, scales, z = quantize_w4(w, group, zeros)
        self.weight = dequantize_w4(codes, scales, z)   # what the layer computes with
        self.codes, self.scales = ctx.to_device(codes), ctx.to_device(scales)
        self.zeros = 0 if z is None else ctx.to_device(z)
        self.bias = 0 if bias is None else ctx.to_device(np.asarray(bias, np.float32))

    def __call__(self, x: int, rows: int, y: int, dtype: int, *, x_stride: int = 0, y_stride: int = 0, out_dtype=None) -> None:
        desc = L.W4Desc(m=rows, n=self.n, k=self.k, group=self.group, x_type=dtype,
                        y_type=dtype if out_dtype is None else out_dtype, x_stride=x_stride or self.k, y_stride=y_stride or self.n)
        self.ctx.gemv_w4(desc, x, self.codes, self.scales, self.zeros, self.bias, y)

    def close(self) -> None:
        """Frees the weights on the device; the layer cannot be called again."""
        for p in filter(None, (self.codes, self.scales, self.zeros, self.bias)):
            self.ctx.free(p)
        self.codes = self.scales = self.zeros = self.bias = 0


class PagedCache:
    """Key / value caches of ``layers`` layers for ``batch`` request places, in pages of ``page`` tokens.

    ``plan(new_lens)`` gives every place its new tokens' pages and slots; the packed token
    rows of the step are the places' new tokens in order. The host keeps the lengths, each
    place's pages and the free list, so nothing is read back. With a window, pages that no later
    token sees go back to the free list."""

    def __init__(self, ctx: L.Context, *, layers: int, batch: int, pages: int, page: int, heads: int, kv_heads: int, head_dim: int,
                 max_tokens: int, max_len: int, dtype: int = L.BF16, window: int = 0, sinks: int = 0, rope_base: float = 10000.0):
        self.ctx, self.batch, self.pages, self.page, self.dtype = ctx, batch, pages, page, dtype
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.max_tokens, self.max_len, self.window, self.sinks = max_tokens, max_len, window, sinks
        self.stride = -(-max_len // page)
        nbytes = pages * kv_heads * page * head_dim * L.ELEM_BYTES[dtype]
        self.k = [ctx.alloc(nbytes) for _ in range(layers)]
        self.v = [ctx.alloc(nbytes) for _ in range(layers)]
        self.lens = np.zeros(batch, np.int64)
        self.free = list(range(pages))
        self.held = [{} for _ in range(batch)]   # place -> {index in its table row: page id}
        i32 = lambda n: ctx.alloc(4 * n)  # noqa: E731
        self.table = ctx.to_device(np.full((batch, self.stride), -1, np.int32))
        self.q_starts, self.kv_lens, self.slots, self.positions, self.status = (i32(n) for n in (batch + 1, batch, max_tokens, max_tokens, 2))
        self._cached, self._new, self._free = i32(batch), i32(batch), i32(pages)
        self.rope = ctx.to_device(rope_table(max_len, head_dim, rope_base))
        self.tokens = self.max_q = 0
        self.workspace, self._room = 0, 0   # grows with the steps that need more

    def _attn(self, tokens: int, max_q: int) -> L.AttnDesc:
        d = self.head_dim
        return L.AttnDesc(batch=self.batch, tokens=tokens, heads=self.heads, kv_heads=self.kv_heads, head_dim=d, page=self.page,
                          pages=self.pages, table_stride=self.stride, max_q=max_q, max_kv=self.max_len, window=self.window,
                          sinks=self.sinks, dtype=self.dtype, scale=1 / math.sqrt(d), q_stride=self.heads * d, out_stride=self.heads * d)

    def plan(self, new_lens) -> None:
        """Pages, slots and positions for ``new_lens[b]`` new tokens of each place."""
        new = np.asarray(new_lens, np.int64)
        total = int(new.sum())
        if new.shape != (self.batch,) or (new < 0).any() or not 0 < total <= self.max_tokens:
            raise ValueError(f"new lengths for {self.batch} places, 1 to {self.max_tokens} tokens in all")
        if (self.lens + new > self.max_len).any():
            raise ValueError(f"a request would pass {self.max_len} tokens")
        self._give_back()
        held = -(-self.lens // self.page)
        need = -(-(self.lens + new) // self.page) - held
        if need.sum() > len(self.free):
            raise L.MdlcError(L.ERR_NOMEM, f"{int(need.sum())} pages wanted, {len(self.free)} free")
        ctx, taken, max_q = self.ctx, int(need.sum()), int(new.max())
        # before anything is planned: a step that finds no memory leaves the cache as it was
        room = L.paged_attn_workspace(self._attn(total, max_q))
        if room > self._room:
            ctx.sync()
            old, self.workspace, self._room = self.workspace, 0, 0
            if old:
                ctx.free(old)
            self.workspace = ctx.alloc(room)
            self._room = room
        ctx.upload(self._cached, self.lens.astype(np.int32))
        ctx.upload(self._new, new.astype(np.int32))
        if taken:
            ctx.upload(self._free, np.array(self.free[:taken], np.int32))
        desc = L.PageDesc(batch=self.batch, page=self.page, table_stride=self.stride, tokens=total, free_pages=taken)
        ctx.page_plan(desc, self._cached, self._new, self._free, 0, self.table, self.q_starts, self.kv_lens, self.slots, self.positions, self.status)
        for b in range(self.batch):   # in the places' order, as the plan takes them
            n = int(need[b])
            self.held[b].update(zip(range(int(held[b]), int(held[b]) + n), self.free[:n]))
            del self.free[:n]
        self.lens += new
        self.tokens, self.max_q = total, max_q

    def _give_back(self) -> None:
        """Pages behind the window: the next token stands at ``lens`` and sees keys from ``lens - window + 1`` on, and the sinks."""
        if not self.window:
            return
        for b, held in enumerate(self.held):
            for i in [i for i in held if (i + 1) * self.page <= self.lens[b] - self.window + 1 and i * self.page >= self.sinks]:
                self.free.append(held.pop(i))

    def append(self, layer: int, qkv: int, q_out: int) -> None:
        """Rotate the queries of the packed [tokens][heads + 2 kv_heads][head_dim] projection into ``q_out`` and write its
        rotated keys and its values to the planned slots."""
        d, esz = self.head_dim, L.ELEM_BYTES[self.dtype]
        width = (self.heads + 2 * self.kv_heads) * d
        desc = L.RopeDesc(tokens=self.tokens, heads=self.heads, kv_heads=self.kv_heads, head_dim=d, rot_dim=d, axes=1, max_pos=self.max_len,
                          page=self.page, pages=self.pages, dtype=self.dtype, q_stride=width, k_stride=width, v_stride=width, out_stride=self.heads * d)
        desc.section[0] = d // 2
        self.ctx.rope_append(desc, qkv, qkv + self.heads * d * esz, qkv + (self.heads + self.kv_heads) * d * esz, self.positions, self.rope,
                             self.slots, q_out, self.k[layer], self.v[layer])

    def attend(self, layer: int, q: int, out: int) -> None:
        """Attention of the step's tokens ([tokens][heads][head_dim]) over their requests' pages."""
        self.ctx.paged_attn(self._attn(self.tokens, self.max_q), q, self.k[layer], self.v[layer], self.table, self.q_starts, self.kv_lens, out, 0,
                            self.workspace)

    def release(self, place: int) -> None:
        """End the request at ``place``: its pages go back to the free list."""
        if not 0 <= place < self.batch:
            raise ValueError(f"place {place} of {self.batch}")
        self.free.extend(self.held[place].values())
        self.held[place] = {}
        self.lens[place] = 0

    def close(self) -> None:
        """Frees the caches and the plan's buffers; a second call does nothing."""
        names = ("table", "q_starts", "kv_lens", "slots", "positions", "status", "_cached", "_new", "_free", "rope", "workspace")
        for p in filter(None, (*self.k, *self.v, *(getattr(self, n) for n in names))):
            self.ctx.free(p)
        self.k, self.v, self._room = [], [], 0
        for n in names:
            setattr(self, n, 0)
