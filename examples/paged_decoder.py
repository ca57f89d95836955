"""A small decoder that answers several requests from one paged cache.

Random weights in 4 bits; prompts enter in chunks of different lengths beside requests that are
already decoding, then every request continues greedily:

    python examples/paged_decoder.py [--steps 16] [--dtype bf16|fp32] [--check]

``--check`` compares every step's logits with a dense fp64 forward over the whole sequences.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mdlc_b200 import _lib as L  # noqa: E402
from mdlc_b200.paged import PagedCache, W4Linear, rope_table  # noqa: E402


class Decoder:
    """``layers`` blocks of x += W_o attn(W_qkv x), x += W_down (silu(W_gate x) * W_up x); logits = W_head x."""

    def __init__(self, ctx, *, layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, inner=512, vocab=1000, batch=4, page=16,
                 max_tokens=160, max_len=512, dtype=L.F32, window=0, sinks=0, seed=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.hidden, self.inner, self.vocab, self.dtype, self.layers = ctx, hidden, inner, vocab, dtype, layers
        self.heads, self.kv_heads, self.head_dim, self.window, self.sinks = heads, kv_heads, head_dim, window, sinks
        linear = lambda n, k, s: W4Linear(ctx, (s * rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32), group=64)  # noqa: E731
        self.embed = rng.standard_normal((vocab, hidden)).astype(np.float32)
        self.qkv = [linear((heads + 2 * kv_heads) * head_dim, hidden, 1.5) for _ in range(layers)]
        self.out = [linear(hidden, heads * head_dim, 0.5) for _ in range(layers)]
        self.up = [linear(2 * inner, hidden, 1.0) for _ in range(layers)]      # gate and up, one product
        self.down = [linear(hidden, inner, 0.5) for _ in range(layers)]
        self.head = linear(vocab, hidden, 1.0)
        self.cache = PagedCache(ctx, layers=layers, batch=batch, pages=batch * (max_len // page), page=page, heads=heads, kv_heads=kv_heads,
                                head_dim=head_dim, max_tokens=max_tokens, max_len=max_len, dtype=dtype, window=window, sinks=sinks)
        esz = L.ELEM_BYTES[dtype]
        widths = dict(x=hidden, qkv=(heads + 2 * kv_heads) * head_dim, q=heads * head_dim, attn=heads * head_dim, y=hidden, up=2 * inner, act=inner)
        self.buf = {k: ctx.alloc(max_tokens * w * esz) for k, w in widths.items()}
        self.gate, self.upper = ctx.alloc(max_tokens * inner * esz), ctx.alloc(max_tokens * inner * esz)
        self.logits = ctx.alloc(max_tokens * vocab * 4)

    def close(self):
        self.cache.close()
        for layer in (*self.qkv, *self.out, *self.up, *self.down, self.head):
            layer.close()
        for p in (*self.buf.values(), self.gate, self.upper, self.logits):
            self.ctx.free(p)

    def _program(self, rows, width, inputs, code):
        p = L.EwProg(n=rows, hw=1, c=width, c_stride=width, dtype=self.dtype, n_inputs=inputs, n_outputs=1, n_instr=len(code))
        for i in range(inputs):
            p.bcast[i] = L.BC_FULL
        for i, c in enumerate(code):
            p.code[i] = L.EwInstr(*c)
        p.out_reg[0] = code[-1][1]
        return p

    def step(self, tokens):
        """``tokens``: a list per place of its new token ids. Returns the fp32 logits of all new tokens, in order."""
        ctx, cache, b = self.ctx, self.cache, self.buf
        cache.plan([len(t) for t in tokens])
        n, f32 = cache.tokens, self.dtype == L.F32
        x = self.embed[np.concatenate([np.asarray(t, np.int64) for t in tokens if len(t)])]
        ctx.upload(b["x"], x if f32 else _bf16(x))
        add = self._program(n, self.hidden, 2, [(L.EW_ADD, 2, 0, 1, 0.0, 0.0)])
        silu = self._program(n, self.inner, 2, [(L.EW_SIGMOID, 2, 0, 0, 0.0, 0.0), (L.EW_MUL, 3, 0, 2, 0.0, 0.0), (L.EW_MUL, 4, 3, 1, 0.0, 0.0)])
        for i in range(self.layers):
            self.qkv[i](b["x"], n, b["qkv"], self.dtype)
            cache.append(i, b["qkv"], b["q"])
            cache.attend(i, b["q"], b["attn"])
            self.out[i](b["attn"], n, b["y"], self.dtype)
            ctx.eltwise(add, [b["x"], b["y"]], [b["x"]])
            self.up[i](b["x"], n, b["up"], self.dtype)
            for half, dst in ((0, self.gate), (1, self.upper)):
                self._columns(b["up"], n, half, dst)
            ctx.eltwise(silu, [self.gate, self.upper], [b["act"]])
            self.down[i](b["act"], n, b["y"], self.dtype)
            ctx.eltwise(add, [b["x"], b["y"]], [b["x"]])
        self.head(b["x"], n, self.logits, self.dtype, out_dtype=L.F32)
        return ctx.download(self.logits, (n, self.vocab), np.float32)

    def _columns(self, src, rows, half, dst):
        """Columns [half * inner, + inner) of a [rows][2 inner] buffer as a buffer of their own."""
        d = L.CopyDesc(dtype=self.dtype, in_cs=2 * self.inner, out_cs=self.inner, mode=0, pad_mode=0, value=0.0)
        d.in_dims[:] = [rows, 2 * self.inner, 1, 1]
        d.out_dims[:] = [rows, self.inner, 1, 1]
        d.src_dim[:] = [0, 1, 2, 3]
        d.offset[:] = [0, -half * self.inner, 0, 0]
        self.ctx.copy4d(d, src, dst)

    def dense(self, tokens):
        """fp64 forward over one whole sequence with the same weights: logits of every position."""
        h, kvh, d, n = self.heads, self.kv_heads, self.head_dim, len(tokens)
        x = self.embed[np.asarray(tokens)].astype(np.float64)
        cs = rope_table(n, d).astype(np.float64)[:, None]
        j, p = np.arange(n)[None], np.arange(n)[:, None]
        seen = (j <= p) & ((self.window == 0) | (j > p - self.window) | (j < self.sinks))

        def turn(a):
            u, w = a[..., :d // 2], a[..., d // 2:]
            return np.concatenate([u * cs[..., 0] - w * cs[..., 1], w * cs[..., 0] + u * cs[..., 1]], -1)
        for i in range(self.layers):
            qkv = (x @ self.qkv[i].weight.T.astype(np.float64)).reshape(n, h + 2 * kvh, d)
            q, k, v = turn(qkv[:, :h]), turn(qkv[:, h:h + kvh]), qkv[:, h + kvh:]
            o = np.empty((n, h, d))
            for e in range(h):
                s = np.where(seen, q[:, e] @ k[:, e // (h // kvh)].T / np.sqrt(d), -np.inf)
                w = np.exp(s - s.max(1, keepdims=True))
                o[:, e] = (w / w.sum(1, keepdims=True)) @ v[:, e // (h // kvh)]
            x = x + o.reshape(n, -1) @ self.out[i].weight.T.astype(np.float64)
            u = x @ self.up[i].weight.T.astype(np.float64)
            g = u[:, :self.inner]
            x = x + (g / (1 + np.exp(-g)) * u[:, self.inner:]) @ self.down[i].weight.T.astype(np.float64)
        return x @ self.head.weight.T.astype(np.float64)


def _bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def run(steps=16, dtype="fp32", check=False, seed=0, **kw):
    """Greedy answers to four prompts; returns (the sequences, the largest relative difference of the logits from the dense forward)."""
    ctx = L.Context(0)
    model = Decoder(ctx, dtype=L.F32 if dtype == "fp32" else L.BF16, seed=seed, **kw)
    rng = np.random.default_rng(seed + 1)
    prompts = [rng.integers(0, model.vocab, n).tolist() for n in (37, 1, 120, 64)]
    seqs, waiting, worst = [[] for _ in prompts], [list(p) for p in prompts], 0.0
    done = [0] * len(prompts)
    while min(done) < steps:
        # up to 48 tokens of a waiting prompt per step, one token of a request that decodes
        now = []
        for i, w in enumerate(waiting):
            now.append(w[:48])
            del w[:48]
        for s, t in zip(seqs, now):
            s.extend(t)
        logits = model.step(now)
        at = 0
        for i, t in enumerate(now):
            if not t:
                continue
            mine = logits[at:at + len(t)]
            at += len(t)
            if check:
                want = model.dense(seqs[i])[-len(t):]
                worst = max(worst, float(np.linalg.norm(mine - want) / np.linalg.norm(want)))
            if not waiting[i]:                       # the prompt is in: continue with the likeliest token
                if done[i] < steps:
                    waiting[i].append(int(mine[-1].argmax()))
                    done[i] += 1
                elif model.cache.lens[i]:
                    model.cache.release(i)           # answered: its pages serve the others
    ctx.sync()
    assert ctx.check_flag() == 0
    model.close()
    ctx.close()
    return seqs, worst


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--dtype", choices=("bf16", "fp32"), default="bf16")
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    seqs, worst = run(a.steps, a.dtype, a.check)
    for i, s in enumerate(seqs):
        print(f"request {i}: {len(s)} tokens, last {s[-a.steps:]}")
    if a.check:
        print(f"largest relative difference of the logits from the dense fp64 forward: {worst:.2e}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
