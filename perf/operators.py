"""The paged decoder operators as cases to time and compare: each in its plain form
(elementary torch operations in 32 bits) and through the library's entry points.

Four operators of one decoder step that answers requests from a paged key / value cache:

* ``plan``: block tables, slot maps and positions built on the GPU from request lengths;
* ``rope``: queries and keys rotated by one to four position axes, keys and values
  written to the cache slots of their tokens;
* ``attn``: attention of each request's new tokens over its pages, causal, with an
  optional sliding window and a few first tokens that stay visible;
* ``w4``: products of a few rows with 4-bit weights and group scales.

The caches are ``[pages][kv_heads][page][head_dim]``, a slot is ``page_id * page + offset``.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ELEM = {"bf16": 2, "f32": 4}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a small server: every request gets one token, a few cross into a new page
        dict(name="plan_step", op="plan", batch=64, new=1, cached=4000, page=16, spare=0, lens=1),
        # a packed prefill wave with chunks of very different lengths and some padding rows at its end
        dict(name="plan_wave", op="plan", batch=1000, new=160, cached=9000, page=32, spare=77, lens=2),
        # the rotation and cache write of one decode step of a few requests: latency
        dict(name="rope_step", op="rope", tokens=8, heads=32, kv_heads=8, head_dim=128, rot_dim=128, axes=1,
             interleaved=False, page=16, padded=0, dtype="bf16"),
        # an image or video prompt: time, height and width positions, an odd number of tokens, some of them padding
        dict(name="rope_video", op="rope", tokens=16001, heads=28, kv_heads=4, head_dim=128, rot_dim=128, axes=3,
             interleaved=False, page=32, padded=19, dtype="bf16"),
        # the next token of a single request: latency
        dict(name="attn_token", op="attn", batch=1, new=1, cached=1500, heads=32, kv_heads=8, head_dim=128, page=16,
             window=0, sinks=0, mixed=False, dtype="bf16", lens=3),
        # the decode step of a loaded server, contexts of all lengths: the cache's bytes
        dict(name="attn_tokens64", op="attn", batch=64, new=1, cached=8192, heads=32, kv_heads=8, head_dim=128,
             page=16, window=0, sinks=0, mixed=False, dtype="bf16", lens=4),
        # chunked prefill of long prompts: the matrix products
        dict(name="attn_chunks", op="attn", batch=3, new=2048, cached=8192, heads=32, kv_heads=8, head_dim=128,
             page=64, window=0, sinks=0, mixed=False, dtype="bf16", lens=5),
        # a continuous batch, decodes beside chunks, with a sliding window and four first tokens kept
        dict(name="attn_window", op="attn", batch=24, new=500, cached=12000, heads=16, kv_heads=2, head_dim=64,
             page=32, window=1024, sinks=4, mixed=True, dtype="bf16", lens=6),
        # the same operator at the reference precision, one head per key head
        dict(name="attn_f32", op="attn", batch=5, new=300, cached=1700, heads=12, kv_heads=12, head_dim=64, page=16,
             window=0, sinks=0, mixed=True, dtype="f32", lens=7),
        # a square projection for one token: latency
        dict(name="w4_square", op="w4", m=1, n=4096, k=4096, group=128, zeros=False, bias=False, dtype="bf16"),
        # an output projection over a large vocabulary for one token: the weights' bytes, more than the cache holds
        dict(name="w4_vocab", op="w4", m=1, n=65536, k=8192, group=128, zeros=False, bias=False, dtype="bf16"),
        # a few speculated tokens, odd sizes, small groups with zero points, 32-bit activations
        dict(name="w4_rows", op="w4", m=7, n=5003, k=2912, group=32, zeros=True, bias=True, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "rope", "attn", "attn", "w4"))
    lens = rng.randrange(1 << 20)
    if op == "plan":
        batch = _log(rng, 1, 2000)
        return dict(op=op, batch=batch, new=_log(rng, 1, max(1, min(4096, 160000 // batch))), cached=_log(rng, 1, 9000),
                    page=rng.choice((8, 16, 32, 64, 128)), spare=rng.randrange(100), lens=lens)
    dtype = rng.choice(("bf16", "bf16", "f32"))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 6, 7, 8))
    head_dim = rng.choice((64, 64, 80, 96, 128, 128))
    page = rng.choice((8, 16, 32, 64, 128))
    if op == "rope":
        return dict(op=op, tokens=_log(rng, 1, 16000 if heads <= 28 else 8000), heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, rot_dim=rng.choice((head_dim, head_dim, head_dim // 2)),
                    axes=rng.choice((1, 1, 2, 3, 4)), interleaved=rng.random() < 0.3, page=page,
                    padded=rng.choice((0, 0, 1, 19)), dtype=dtype)
    if op == "w4":
        group = rng.choice((32, 64, 128))
        k = group * _log(rng, max(1, 256 // group), 16384 // group)
        n = _log(rng, 64, min(65536, (65536 * 8192) // k))
        return dict(op=op, m=_log(rng, 1, 16), n=n, k=k, group=group, zeros=rng.random() < 0.5,
                    bias=rng.random() < 0.5, dtype=dtype)
    batch = _log(rng, 1, 64)
    new = rng.choice((1, 1, _log(rng, 1, 2048)))
    new = min(new, max(1, 6144 // batch))
    cached = _log(rng, 1, 16000 if new == 1 else 8192)
    if batch * cached > 64 * 8192:
        cached = 64 * 8192 // batch
    while batch * new * heads * (cached + new) > 6e8 * (1 if dtype == "bf16" else 0.25):
        new = max(1, new // 2)
        cached = max(1, cached * 3 // 4)
    window = rng.choice((0, 0, _log(rng, 16, 4096)))
    return dict(op=op, batch=batch, new=new, cached=cached, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, window=window, sinks=rng.choice((0, 4, 17)) if window else 0, mixed=rng.random() < 0.5,
                dtype=dtype, lens=lens)


def _lens(case):
    """(cached, new) lengths of the case's requests: the first has the case's own, the others spread below."""
    r = random.Random(case["lens"])
    cached = [case["cached"]] + [_log(r, max(1, case["cached"] // 64), case["cached"]) for _ in range(case["batch"] - 1)]
    new = [case["new"]] + [max(1, int(case["new"] * r.uniform(0.2, 1.0))) for _ in range(case["batch"] - 1)]
    if case.get("mixed"):
        new = [n if i % 3 == 0 else 1 for i, n in enumerate(new)]
    return cached, new


def _sections(case):
    """Frequency pairs of each position axis: an even split, the first axis smallest."""
    pairs, axes = case["rot_dim"] // 2, case["axes"]
    return [pairs // axes + (1 if a >= axes - pairs % axes else 0) for a in range(axes)]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn, "w4": _prepare_w4}[case["op"]](case, g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _randn(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(DTYPES[dtype])


def _table(lens, page, g, spare):
    """(block table of `lens` tokens per request with -1 past their pages, ids left over): a random order of page ids."""
    need = (lens + page - 1) // page
    stride = int(need.max())
    total = int(need.sum())
    ids = torch.randperm(total + spare, device="cuda", generator=g).int()
    col = torch.arange(stride, device="cuda", dtype=torch.int32)
    first = (torch.cumsum(need, 0) - need).int()
    at = (first[:, None] + col[None]).clamp(max=total - 1).long()
    return torch.where(col[None] < need[:, None], ids[at], -1).int(), ids[total:].contiguous()


def _prepare_plan(case, g):
    cached, new = (_ints(v) for v in _lens(case))
    page, tokens = case["page"], int(new.sum()) + case["spare"]
    spare = int(((cached + new + page - 1) // page - (cached + page - 1) // page).sum()) + 5
    held, free = _table(cached, page, g, spare)
    stride = int(((cached + new + page - 1) // page).max())
    table = torch.full((case["batch"], stride), -1, dtype=torch.int32, device="cuda")
    table[:, :held.shape[1]] = held
    out = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(case=case, cached=cached, new=new, free=free, free_count=_ints([free.numel()]), table=table,
                q_starts=out(case["batch"] + 1), kv_lens=out(case["batch"]), slots=out(tokens), positions=out(tokens),
                status=out(2))


def _rope_table(max_pos, rot_dim):
    inv = 10000.0 ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    a = np.arange(max_pos, dtype=np.float64)[:, None] * inv[None]
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).cuda()


def _prepare_rope(case, g):
    t, h, kvh, d, page = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "page"))
    qkv = _randn((t, (h + 2 * kvh) * d), case["dtype"], g)
    max_pos = 4096
    pages = (t + page - 1) // page + 3
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:t].int()
    if case["padded"] and t > case["padded"]:
        slots[t - case["padded"]:] = -1
    cache = lambda: torch.zeros((pages, kvh, page, d), dtype=DTYPES[case["dtype"]], device="cuda")  # noqa: E731
    return dict(case=case, qkv=qkv, table=_rope_table(max_pos, case["rot_dim"]), slots=slots,
                positions=torch.randint(0, max_pos, (case["axes"], t), device="cuda", generator=g, dtype=torch.int32),
                q_out=torch.zeros((t, h, d), dtype=DTYPES[case["dtype"]], device="cuda"), k_cache=cache(), v_cache=cache())


def _prepare_attn(case, g):
    cached, new = (_ints(v) for v in _lens(case))
    kv = cached + new
    h, kvh, d, page = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    table, rest = _table(kv, page, g, 3)
    pages = int(((kv + page - 1) // page).sum()) + 3
    tokens = int(new.sum())
    cache = lambda scale: _randn((pages, kvh, page, d), case["dtype"], g, scale)  # noqa: E731
    return dict(case=case, q=_randn((tokens, h, d), case["dtype"], g, 1.5), k_cache=cache(1.0), v_cache=cache(1.0),
                table=table, kv_lens=kv, q_starts=torch.cat([_ints([0]), torch.cumsum(new, 0).int()]),
                max_q=int(new.max()), max_kv=int(kv.max()),
                out=torch.zeros((tokens, h, d), dtype=DTYPES[case["dtype"]], device="cuda"),
                lse=torch.zeros((tokens, h), dtype=torch.float32, device="cuda"))


def _prepare_w4(case, g):
    m, n, k, groups = case["m"], case["n"], case["k"], case["k"] // case["group"]
    x = torch.randn((m, k), device="cuda", generator=g)
    x = (x * (1.0 + 9.0 * (torch.rand((1, k), device="cuda", generator=g) < 0.01))).to(DTYPES[case["dtype"]])  # a few large channels
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = (0.01 * (0.5 + torch.rand((n, groups), device="cuda", generator=g))).bfloat16()
    zeros = torch.randint(5, 11, (n, groups), device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
    bias = torch.randn((n,), device="cuda", generator=g) if case["bias"] else None
    return dict(case=case, x=x, codes=codes, scales=scales, zeros=zeros, bias=bias,
                y=torch.zeros((m, n), dtype=DTYPES[case["dtype"]], device="cuda"))


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn, "w4": _plain_w4}[state["case"]["op"]](state)


def _plain_plan(s):
    page, stride, tokens, n_free = s["case"]["page"], s["table"].shape[1], s["slots"].numel(), s["free"].numel()
    cached, new = s["cached"], s["new"]
    held, need = (cached + page - 1) // page, (cached + new + page - 1) // page
    fits = need <= stride
    take = torch.where(fits, need - held, 0)
    end = torch.cumsum(take, 0)
    ok = fits & ((take == 0) | (end <= s["free_count"]))
    col = torch.arange(stride, device="cuda", dtype=torch.int32)[None]
    at = ((end - take)[:, None] + col - held[:, None]).clamp(0, n_free - 1).long()
    fresh = ok[:, None] & (col >= held[:, None]) & (col < need[:, None])
    table = torch.where(fresh, s["free"][at], s["table"])
    q_starts = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0).int()]).clamp(max=tokens)
    t = torch.arange(tokens, device="cuda", dtype=torch.int32)
    req = torch.searchsorted(q_starts[1:].contiguous(), t, right=True)
    real = req < new.numel()
    req = req.clamp(max=new.numel() - 1)
    pos = cached[req] + t - q_starts[req]
    slot = table[req, (pos // page).clamp(max=stride - 1).long()] * page + pos % page
    status = torch.stack([torch.where(ok & (take > 0), end, 0).max(), (~ok).sum()]).int()
    return dict(table=table, q_starts=q_starts, kv_lens=cached + torch.where(ok, new, 0),
                slots=torch.where(real & ok[req], slot, -1), positions=torch.where(real, pos, 0), status=status)


def _rotate(x, cs, rot_dim, interleaved):
    """x [tokens, heads, head_dim] in 32 bits, cs [tokens, rot_dim / 2, 2]."""
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    r, rest = x[..., :rot_dim], x[..., rot_dim:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = r[..., :rot_dim // 2], r[..., rot_dim // 2:]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([r, rest], -1)


def _split_qkv(s):
    c = s["case"]
    h, kvh, d = c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = s["qkv"].view(c["tokens"], h + 2 * kvh, d).split([h, kvh, kvh], 1)
    return q, k, v


def _plain_rope(s):
    c = s["case"]
    q, k, v = _split_qkv(s)
    axis = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(_sections(c))).cuda()
    pair = torch.arange(c["rot_dim"] // 2, device="cuda")
    cs = s["table"][s["positions"].long()[axis].t(), pair[None]]
    dtype = q.dtype
    s["q_out"].copy_(_rotate(q.float(), cs, c["rot_dim"], c["interleaved"]).to(dtype))
    k = _rotate(k.float(), cs, c["rot_dim"], c["interleaved"]).to(dtype)
    real = s["slots"] >= 0
    at = s["slots"][real].long()
    s["k_cache"][at // c["page"], :, at % c["page"]] = k[real]
    s["v_cache"][at // c["page"], :, at % c["page"]] = v[real]
    return dict(q=s["q_out"], k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attn(s):
    c = s["case"]
    h, kvh, d = c["heads"], c["kv_heads"], c["head_dim"]
    b, nq, nk = c["batch"], s["max_q"], s["table"].shape[1] * c["page"]
    lens = (s["q_starts"][1:] - s["q_starts"][:-1])[:, None]
    row = torch.arange(nq, device="cuda")[None]
    at = (s["q_starts"][:-1, None] + row).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().view(b, nq, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, h // kvh * nq, d)
    pages = s["table"].clamp(min=0).long()
    k = s["k_cache"][pages].permute(0, 2, 1, 3, 4).reshape(b, kvh, nk, d).float()
    v = s["v_cache"][pages].permute(0, 2, 1, 3, 4).reshape(b, kvh, nk, d).float()
    key = torch.arange(nk, device="cuda")[None, None]
    pos = (s["kv_lens"][:, None] - lens + row)[:, :, None]
    seen = key <= pos
    if c["window"]:
        seen = seen & ((key > pos - c["window"]) | (key < c["sinks"]))
    w = (q @ k.transpose(-1, -2)).view(b, kvh, h // kvh, nq, nk)
    w *= 1.0 / math.sqrt(d)
    w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    w = w.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    o = w.view(b, kvh, h // kvh * nq, nk) @ torch.where((key[0] < s["kv_lens"][:, None])[:, None, :, None], v, 0.0)
    o = o.view(b, kvh, h // kvh, nq, d) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log())[..., 0]
    req = torch.searchsorted(s["q_starts"][1:].contiguous(), torch.arange(s["q"].shape[0], device="cuda").int(), right=True)
    i = torch.arange(s["q"].shape[0], device="cuda") - s["q_starts"][req]
    out = o.permute(0, 3, 1, 2, 4).reshape(b, nq, h, d)[req, i].to(s["q"].dtype)
    return dict(out=out, lse=lse.permute(0, 3, 1, 2).reshape(b, nq, h)[req, i])


def _plain_w4(s):
    c = s["case"]
    n, k, groups = c["n"], c["k"], c["k"] // c["group"]
    w = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(n, groups, c["group"]).float()
    w = (w - (s["zeros"][..., None].float() if c["zeros"] else 8.0)) * s["scales"][..., None].float()
    y = s["x"].float() @ w.view(n, k).t()
    if c["bias"]:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------ the library's entry points
_context = None


def _ctx():
    global _context
    from mdlc_b200 import _lib
    if _context is None:
        _context = _lib.Context(torch.cuda.current_device())
        _context.bind_stream(torch.cuda.current_stream().cuda_stream)
    return _lib, _context


def _run_own(s):
    if "call" not in s:  # the descriptor and the pointers, as a program sets them up once for its buffers
        s["call"] = {"plan": _own_plan, "rope": _own_rope, "attn": _own_attn, "w4": _own_w4}[s["case"]["op"]](s)
    call, args, out = s["call"]
    call(*args)
    return out


def _own_plan(s):
    lib, ctx = _ctx()
    desc = lib.PageDesc(batch=s["case"]["batch"], page=s["case"]["page"], table_stride=s["table"].shape[1],
                        tokens=s["slots"].numel(), free_pages=s["free"].numel())
    out = {k: s[k] for k in ("table", "q_starts", "kv_lens", "slots", "positions", "status")}
    return ctx.page_plan, (desc, *(s[k].data_ptr() for k in ("cached", "new", "free", "free_count")),
                           *(v.data_ptr() for v in out.values())), out


def _own_rope(s):
    lib, ctx = _ctx()
    c = s["case"]
    q, k, v = _split_qkv(s)
    desc = lib.RopeDesc(tokens=c["tokens"], heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["head_dim"],
                        rot_dim=c["rot_dim"], interleaved=int(c["interleaved"]), axes=c["axes"], max_pos=s["table"].shape[0],
                        page=c["page"], pages=s["k_cache"].shape[0], dtype=lib.BF16 if c["dtype"] == "bf16" else lib.F32,
                        q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0), out_stride=s["q_out"].stride(0))
    desc.section[:c["axes"]] = _sections(c)
    out = dict(q=s["q_out"], k_cache=s["k_cache"], v_cache=s["v_cache"])
    return ctx.rope_append, (desc, *(t.data_ptr() for t in (q, k, v, s["positions"], s["table"], s["slots"])),
                             *(t.data_ptr() for t in out.values())), out


def _own_attn(s):
    lib, ctx = _ctx()
    c = s["case"]
    desc = lib.AttnDesc(batch=c["batch"], tokens=s["q"].shape[0], heads=c["heads"], kv_heads=c["kv_heads"],
                        head_dim=c["head_dim"], page=c["page"], pages=s["k_cache"].shape[0], table_stride=s["table"].shape[1],
                        max_q=s["max_q"], max_kv=s["max_kv"], window=c["window"], sinks=c["sinks"],
                        dtype=lib.BF16 if c["dtype"] == "bf16" else lib.F32, scale=1.0 / math.sqrt(c["head_dim"]),
                        q_stride=s["q"].stride(0), out_stride=s["out"].stride(0))
    s["workspace"] = torch.empty(max(16, lib.paged_attn_workspace(desc)), dtype=torch.uint8, device="cuda")
    ins = ("q", "k_cache", "v_cache", "table", "q_starts", "kv_lens", "out", "lse", "workspace")
    return ctx.paged_attn, (desc, *(s[k].data_ptr() for k in ins)), dict(out=s["out"], lse=s["lse"])


def _own_w4(s):
    lib, ctx = _ctx()
    c = s["case"]
    dtype = lib.BF16 if c["dtype"] == "bf16" else lib.F32
    desc = lib.W4Desc(m=c["m"], n=c["n"], k=c["k"], group=c["group"], x_type=dtype, y_type=dtype,
                      x_stride=s["x"].stride(0), y_stride=s["y"].stride(0))
    zeros, bias = (0 if t is None else t.data_ptr() for t in (s["zeros"], s["bias"]))
    return ctx.gemv_w4, (desc, s["x"].data_ptr(), s["codes"].data_ptr(), s["scales"].data_ptr(), zeros, bias,
                         s["y"].data_ptr()), s["y"]


# ------------------------------------------------------------------ what a pass cannot do without
def _seen(case, cached, new):
    """(visible pairs, keys that some row sees) of one request and head."""
    w, sinks = case["window"], case["sinks"]
    p = np.arange(cached, cached + new, dtype=np.int64)
    if not w:
        return int((p + 1).sum()), cached + new
    first = np.maximum(p - w + 1, 0)
    pairs = p + 1 - first + np.minimum(first, sinks)
    return int(pairs.sum()), int(cached + new - first[0] + min(first[0], sinks))


def work(case):
    op = case["op"]
    if op == "plan":
        cached, new = _lens(case)
        page, tokens = case["page"], sum(new) + case["spare"]
        fresh = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
        return dict(bytes=4 * (4 * case["batch"] + 2 * fresh + 2 * tokens), flops=0)
    e = ELEM[case["dtype"]]
    if op == "rope":
        t, h, kvh, d, r = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "rot_dim"))
        rows = min(t * case["axes"], 4096)
        return dict(bytes=2 * e * t * (h + 2 * kvh) * d + 4 * t * (case["axes"] + 1) + rows * r * 4,
                    flops=3 * t * (h + kvh) * r)
    if op == "w4":
        m, n, k, groups = case["m"], case["n"], case["k"], case["k"] // case["group"]
        return dict(bytes=n * k // 2 + n * groups * (3 if case["zeros"] else 2) + e * m * (n + k) + (4 * n if case["bias"] else 0),
                    flops=2 * m * n * k)
    cached, new = _lens(case)
    seen = [_seen(case, c, n) for c, n in zip(cached, new)]
    h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    return dict(bytes=e * d * (2 * h * sum(new) + 2 * kvh * sum(s[1] for s in seen)) + 4 * h * sum(new),
                flops=4 * d * h * sum(s[0] for s in seen))


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "attn": _exact_attn, "w4": _exact_w4}[case["op"]](s)


def _exact_plan(s):
    page = s["case"]["page"]
    cached, new, free = (s[k].tolist() for k in ("cached", "new", "free"))
    table = s["table"].cpu().numpy().copy()
    tokens, left, asked, taken, refused = s["slots"].numel(), s["free_count"].item(), 0, 0, 0
    slots, positions = np.full(tokens, -1, np.int32), np.zeros(tokens, np.int32)
    starts, kv = [0], []
    for b, (c, n) in enumerate(zip(cached, new)):
        held, need = -(-c // page), -(-(c + n) // page)
        asked += need - held if need <= table.shape[1] else 0
        good = need <= table.shape[1] and (need == held or asked <= left)
        for j in range(held, need if good else held):
            table[b, j] = free[taken]
            taken += 1
        refused += not good
        for i in range(n):
            t = starts[-1] + i
            if t < tokens:
                positions[t] = c + i
                if good:
                    slots[t] = table[b, (c + i) // page] * page + (c + i) % page
        starts.append(min(starts[-1] + n, tokens))
        kv.append(c + n if good else c)
    return dict(table=table, q_starts=np.array(starts, np.int32), kv_lens=np.array(kv, np.int32), slots=slots,
                positions=positions, status=np.array([taken, refused], np.int32))


def _exact_rope(s):
    c = s["case"]
    h, kvh, d, page, rot = (c[k] for k in ("heads", "kv_heads", "head_dim", "page", "rot_dim"))
    x = s["qkv"].double().view(c["tokens"], h + 2 * kvh, d)
    y = x.clone()
    pair = 0
    for axis, count in enumerate(_sections(c)):
        angle = s["table"].double()[s["positions"][axis].long()]
        for i in range(pair, pair + count):
            u, w = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)
            cos, sin = angle[:, i, 0, None], angle[:, i, 1, None]
            y[:, :h + kvh, u] = x[:, :h + kvh, u] * cos - x[:, :h + kvh, w] * sin
            y[:, :h + kvh, w] = x[:, :h + kvh, u] * sin + x[:, :h + kvh, w] * cos
        pair += count
    caches = []
    for cache, lo in ((s["k_cache"], h), (s["v_cache"], h + kvh)):
        flat = cache.double().transpose(1, 2).reshape(-1, kvh, d).clone()
        real = torch.nonzero(s["slots"] >= 0)[:, 0]
        flat[s["slots"][real].long()] = y[real, lo:lo + kvh]
        caches.append(flat.view(-1, page, kvh, d).transpose(1, 2).contiguous())
    return dict(q=y[:, :h].contiguous(), k_cache=caches[0], v_cache=caches[1])


def _exact_attn(s):
    c = s["case"]
    h, kvh, d, page = (c[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    cached, new = _lens(c)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (nc, n) in enumerate(zip(cached, new)):
        ids = s["table"][b, :-(-(nc + n) // page)].long()
        k, v = (x[ids].transpose(0, 1).reshape(kvh, -1, d)[:, :nc + n].double() for x in (s["k_cache"], s["v_cache"]))
        q = s["q"][first:first + n].double()
        j = torch.arange(nc + n, device="cuda")[None]
        p = torch.arange(nc, nc + n, device="cuda")[:, None]
        hidden = j > p
        if c["window"]:
            hidden |= (j <= p - c["window"]) & (j >= c["sinks"])
        for i in range(h):
            e = i // (h // kvh)
            score = (q[:, i] @ k[e].t()) / math.sqrt(d)
            score[hidden] = -math.inf
            lse[first:first + n, i] = torch.logsumexp(score, -1)
            out[first:first + n, i] = torch.exp(score - lse[first:first + n, i, None]) @ v[e]
        first += n
    return dict(out=out, lse=lse)


def _exact_w4(s):
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    zero = s["zeros"].double() if c["zeros"] else torch.full((n, k // group), 8.0, dtype=torch.float64, device="cuda")
    y = torch.zeros((c["m"], n), dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for g in range(k // group):
        codes = s["codes"][:, g * group // 2:(g + 1) * group // 2]
        part = x[:, g * group:(g + 1) * group]
        acc = part[:, 0::2] @ (codes % 16).double().t() + part[:, 1::2] @ (codes // 16).double().t()
        y += (acc - part.sum(1, keepdim=True) * zero[:, g]) * s["scales"][:, g].double()
    return y + s["bias"].double() if c["bias"] else y
