"""The transformer operators of the library at the sizes they are used at.

Four operators: rotary positions with several axes, appending keys and values
to a paged cache (16 bits, or e4m3 with a scale for each page and head), the
attention that reads that cache, and the norms around a block with its gate
and residual scale.  ``run`` computes an operator in its plain form, in
elementary torch operations, or, where ``own`` is true, through the library.
"""
import math
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F8 = torch.float8_e4m3fn


def listed():
    return [
        # one control step of one vehicle with a short history: latency is all of it
        dict(name="attention one token", op="attention", sequences=1, new=1, length=37, prefix=0, heads=3, kv_heads=3,
             dim=64, page=16, dtype="bf16", storage="same", window=0, sinks=0, frame=1),
        # the image planner's 1024 candidates: a shared history and each candidate's own last steps
        dict(name="attention candidates", op="attention", sequences=1024, new=1, length=34, prefix=24, heads=16,
             kv_heads=16, dim=64, page=16, dtype="bf16", storage="same", window=0, sinks=0, frame=1),
        # a few long sessions, one token each, grouped heads: the cache is read once
        dict(name="attention long sessions", op="attention", sequences=4, new=1, length=65536, prefix=0, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16", storage="same", window=0, sinks=0, frame=1),
        # a served fleet on an 8-bit cache: a window of the newest tokens and the first ones
        dict(name="attention window 8 bit", op="attention", sequences=48, new=1, length=30000, prefix=0, heads=16,
             kv_heads=4, dim=128, page=32, dtype="f16", storage="e4m3", window=4096, sinks=4, frame=1),
        # reading in whole histories: causal, grouped heads, the most arithmetic
        dict(name="attention history", op="attention", sequences=2, new=8192, length=8192, prefix=0, heads=16,
             kv_heads=4, dim=128, page=64, dtype="bf16", storage="same", window=0, sinks=0, frame=1),
        # two new ViT frames (197 tokens each) for eight vehicles: tokens of a frame see each other, a window of
        # eight frames and the first frame
        dict(name="attention frames 8 bit", op="attention", sequences=8, new=394, length=7880, prefix=0, heads=12,
             kv_heads=12, dim=64, page=64, dtype="f16", storage="e4m3", window=8, sinks=197, frame=197),
        # every candidate's next token into an 8-bit cache: pages that hold earlier tokens
        dict(name="append candidates 8 bit", op="append", sequences=1024, new=1, length=40, heads=16, kv_heads=16,
             dim=64, page=16, dtype="bf16", storage="e4m3", axes=1, interleaved=False),
        # eight video frames of 14 x 14 patches for sixteen vehicles, rotated by time, height and width
        dict(name="append video", op="append", sequences=16, new=1568, length=3136, heads=16, kv_heads=16, dim=64,
             page=64, dtype="bf16", storage="same", axes=3, interleaved=False),
        # an image encoder's queries: 64 frames of 14 x 14 patches, the ViT's 3 heads, rows and columns
        dict(name="rotary images", op="rotary", tokens=12544, heads=3, dim=64, dtype="f32", axes=2, interleaved=True,
             inverse=False),
        # a long video's keys turned back (the transpose)
        dict(name="rotary video back", op="rotary", tokens=131072, heads=16, dim=64, dtype="bf16", axes=3,
             interleaved=False, inverse=True),
        # the predictor's block over 1024 candidates: each its own action's modulation, AdaLN's two norms
        dict(name="norm predictor", op="norm", rows=1024, width=192, residual="f32", dtype="f32", cond="f32",
             per_cond=1, post="none", pre="layer", gate=True, modulate=True, residual_scale=False, out_norm=True),
        # a video model's block: norms on both sides, residual in 32 bits, one modulation for a clip
        dict(name="norm video", op="norm", rows=50176, width=1024, residual="f32", dtype="bf16", cond="bf16",
             per_cond=1568, post="rms", pre="rms", gate=True, modulate=True, residual_scale=True, out_norm=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "rotary", "norm"])
    if op == "attention":
        kv, group = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 8])
        dim, page = rng.choice([32, 64, 64, 128, 128]), rng.choice([16, 32, 64, 128])
        while True:
            sequences, length = _log(rng, 1, 1024), _log(rng, 1, 65536)
            if sequences * length * kv * dim <= 200_000_000:
                break
        new = 1
        if rng.random() < 0.6:
            most = min(length, 8192, 1_500_000_000 // max(1, sequences * length * kv * group))
            new = _log(rng, 1, max(1, most))
        frame = rng.choice([1, 1, 1, 49, 197])
        window = 0 if rng.random() < 0.5 else _log(rng, 1, 8192) if frame == 1 else rng.randint(1, 16)
        return dict(op=op, sequences=sequences, new=new, length=length, prefix=0, heads=kv * group, kv_heads=kv,
                    dim=dim, page=page, dtype=rng.choice(["bf16", "f16"]), storage=rng.choice(["same", "e4m3"]),
                    window=window, sinks=rng.choice([0, 1, 4, 130]) if window else 0, frame=frame)
    if op == "append":
        kv, group = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 2, 4])
        dim = rng.choice([32, 64, 128])
        sequences = _log(rng, 1, 1024)
        new = _log(rng, 1, max(1, min(4096, 25000 // sequences)))
        held = _log(rng, 1, max(1, min(4000, 50_000 // sequences)))  # tokens that are in the cache already
        return dict(op=op, sequences=sequences, new=new, length=new + held,
                    heads=kv * group, kv_heads=kv, dim=dim, page=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["bf16", "f16"]), storage=rng.choice(["same", "e4m3"]),
                    axes=rng.choice([1, 2, 3] if dim > 32 else [1, 2]), interleaved=rng.random() < 0.5)
    if op == "rotary":
        return dict(op=op, tokens=_log(rng, 1, 100_000), heads=rng.choice([1, 3, 8, 16]), dim=rng.choice([64, 128, 64]),
                    dtype=rng.choice(["f32", "bf16", "f16"]), axes=rng.choice([1, 2, 3]),
                    interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3)
    rows = _log(rng, 1, 50000)
    width = rng.choice([64, 192, 193, 384, 768, 1000, 1024, 2048, 4096])
    rows = min(rows, 50_000_000 // width)
    dtype = rng.choice(["f32", "bf16", "f16"])
    pre = rng.choice(["layer", "rms"])
    return dict(op=op, rows=rows, width=width, residual=rng.choice(["f32", dtype]), dtype=dtype,
                cond=rng.choice(["f32", dtype]), per_cond=rng.choice([1, 1, 7, 197, 1568]),
                post=rng.choice(["none", "layer", "rms"]), pre=pre, gate=rng.random() < 0.8,
                modulate=rng.random() < 0.8, residual_scale=rng.random() < 0.5,
                out_norm=pre == "layer" and rng.random() < 0.4)


# --------------------------------------------------------------- inputs

def _axis_dims(dim, axes):
    """Channels of each axis (multiples of 16): time first, the rest shared."""
    units = dim // 16
    share = [units // axes] * axes
    share[0] += units - sum(share)
    return [16 * u for u in share]


def _bases(axes):
    return [10000.0] * axes if axes == 1 else [10000.0] + [100.0] * (axes - 1)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _positions(case, count, rng):
    """Token positions on each axis: a running index, or (time, row, column) of 14 x 14 patches."""
    base = rng.integers(0, 100_000)
    i = np.arange(count, dtype=np.int64) + base * (case["axes"] == 1)
    if case["axes"] == 1:
        cols = [i]
    else:
        cols = [i // 14 % 14, i % 14] if case["axes"] == 2 else [base // 196 + i // 196, i // 14 % 14, i % 14]
    return torch.from_numpy(np.stack(cols, 1).astype(np.int32)).to(DEV)


def _batch(case):
    """Host plan of a ragged batch: new tokens, lengths and page table; every seventh sequence of a large batch rests.
    It goes by the case alone, so that other values come in the same shapes."""
    rng = np.random.default_rng([case["sequences"], case["new"], case["length"], case["page"]])
    s, new, length = case["sequences"], case["new"], case["length"]
    lens = rng.integers((length + 1) // 2, length + 1, s)
    news = rng.integers((new + 1) // 2, new + 1, s)
    lens[0], news[0] = length, new
    prefix = case.get("prefix", 0)
    if prefix:
        lens = rng.integers(prefix + 1, length + 1, s)
        lens[0] = length
    news = np.minimum(news, lens)
    if s >= 14:
        news[6::7] = 0
    page = case["page"]
    per = -(-length // page)
    shared = prefix // page
    pages = shared + s * (per - shared)
    order = rng.permutation(pages + 3)[:pages]  # pages lie anywhere in the pool
    table = np.zeros((s, per), np.int32)
    table[:, :shared] = order[:shared]
    table[:, shared:] = order[shared:].reshape(s, per - shared)
    starts = np.zeros(s + 1, np.int32)
    starts[1:] = np.cumsum(news)
    return lens.astype(np.int32), news.astype(np.int32), starts, table, pages + 3


def _page_scale(amax):
    """The least power of two with amax <= 448 times it."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -120)).clamp(-120, 120)
    return torch.ldexp(torch.ones_like(amax), e)


def _pools(case, pages, g):
    """Cached keys and values: 16 bits, or e4m3 codes with the scale of each page and head."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    out = {}
    for name in ("k", "v"):
        x = _normal(g, *shape)
        if name == "v":
            x *= torch.exp(0.5 * _normal(g, pages, case["kv_heads"], 1, 1))  # pages differ in size
        if case["storage"] == "e4m3":
            scale = _page_scale(x.abs().amax((2, 3)))
            out[name] = (x / scale[:, :, None, None]).to(F8)
            out[name + "_scale"] = scale
        else:
            out[name] = x.to(DTYPES[case["dtype"]])
        del x
    return out


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    g = torch.Generator(DEV).manual_seed(seed)
    st = dict(case=case)
    if case["op"] in ("rotary", "append"):
        dims, bases = _axis_dims(case["dim"], case["axes"]), _bases(case["axes"])
        first, second, freq, axis, off = [], [], [], [], 0
        for a, n in enumerate(dims):
            i = np.arange(n // 2)
            first.append(off + (2 * i if case["interleaved"] else i))
            second.append(off + (2 * i + 1 if case["interleaved"] else i + n // 2))
            freq.append(bases[a] ** (-2.0 * i / n))
            axis.append(np.full(n // 2, a))
            off += n
        st.update(dims=dims, bases=bases, first=_dev(np.concatenate(first)), second=_dev(np.concatenate(second)),
                  freq=_dev(np.concatenate(freq)), axis=_dev(np.concatenate(axis)))
    if case["op"] == "rotary":
        dt = DTYPES[case["dtype"]]
        st["x"] = _normal(g, case["tokens"], case["heads"], case["dim"]).to(dt)
        st["out"] = torch.empty_like(st["x"])
        st["positions"] = _positions(case, case["tokens"], rng)
        return st
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        dt, rt, ct = DTYPES[case["dtype"]], DTYPES[case["residual"]], DTYPES[case["cond"]]
        st["x"] = (2.0 * _normal(g, rows, width) + _normal(g, width)).to(rt)
        st["y"] = _normal(g, rows, width).to(dt)
        conds = -(-rows // case["per_cond"])
        table = 0.3 * _normal(g, conds, 3 * width)  # gate, shift and scale of a block: one modulation table
        st["table"] = table.to(ct)
        for n in ("post_w", "pre_w", "out_w"):
            st[n] = 1.0 + 0.1 * _normal(g, width)
        for n in ("post_b", "pre_b", "out_b"):
            st[n] = 0.1 * _normal(g, width)
        st["rs"] = 0.5 + 0.1 * _normal(g, width)
        st["x_out"], st["h"] = torch.empty_like(st["x"]), torch.empty_like(st["y"])
        return st
    lens, news, starts, table, pages = _batch(case)
    st.update(lens=lens, news=news, tokens=int(starts[-1]), table=_dev(table), starts=_dev(starts),
              lengths=_dev(lens))
    st.update(_pools(case, pages, g))
    dt, tokens, d = DTYPES[case["dtype"]], st["tokens"], case["dim"]
    if case["op"] == "attention":
        st["q"] = _normal(g, tokens, case["heads"], d).to(dt)
        st["out"] = torch.empty_like(st["q"])
        return st
    # a fused projection's output: queries, keys and values of a token side by side
    heads, kv = case["heads"], case["kv_heads"]
    st["qkv"] = _normal(g, tokens, heads + 2 * kv, d).to(dt)
    st["q_out"] = torch.empty((tokens, heads, d), device=DEV, dtype=dt)
    st["positions"] = _positions(case, tokens, rng)
    # what is read back: the new tokens and up to a page of older ones, which a grown scale has rounded again
    back = np.where(news > 0, np.minimum(lens, news + case["page"]), 0).astype(np.int32)
    bs = np.zeros(len(back) + 1, np.int32)
    bs[1:] = np.cumsum(back)
    st.update(back=back, back_tokens=int(bs[-1]), back_starts=_dev(bs), back_max=int(back.max()))
    st["k_back"] = torch.empty((int(bs[-1]), kv, d), device=DEV, dtype=dt)
    st["v_back"] = torch.empty_like(st["k_back"])
    return st


# ----------------------------------------------------------- plain forms

def _rotate(st, x, positions, inverse=False):
    angle = positions.double()[:, st["axis"]] * st["freq"]
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    s = -s if inverse else s
    x = x.float()
    a, b = x[..., st["first"]], x[..., st["second"]]
    out = x.clone()
    out[..., st["first"]] = a * c - b * s
    out[..., st["second"]] = a * s + b * c
    return out


def _owners(starts, lengths, count):
    """Sequence and cache index of each packed token."""
    t = torch.arange(count, device=DEV)
    seq = torch.searchsorted(starts[1:].long(), t, right=True)
    return seq, lengths[seq].long() - (starts[seq + 1].long() - t)


def _plain_append(st):
    case = st["case"]
    heads, kv, page = case["heads"], case["kv_heads"], case["page"]
    qkv = st["qkv"]
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    seq, index = _owners(st["starts"], st["lengths"], st["tokens"])
    at, slot = st["table"][seq, index // page].long(), index % page
    q = _rotate(st, q, st["positions"]).to(q.dtype)
    new = {"k": _rotate(st, k, st["positions"]), "v": v.float()}
    if case["storage"] == "e4m3":
        fresh = index - slot >= (st["lengths"] - (st["starts"][1:] - st["starts"][:-1]))[seq]
        for n, x in new.items():
            pool, scale = st[n], st[n + "_scale"]
            amax = torch.zeros_like(scale).index_reduce_(
                0, at, torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2), "amax")
            old = scale.clone()
            scale[at] = torch.maximum(_page_scale(amax[at]), torch.where(fresh[:, None], 0.0, old[at]))
            # earlier tokens of the pages that are written to, at their pages' new scales
            again = torch.ones_like(scale)
            again[at] = torch.where(fresh[:, None], 1.0, old[at] / scale[at])
            pool.copy_((pool.float() * again[:, :, None, None]).to(F8))
            pool.view(torch.uint8)[at, :, slot] = (x / scale[at][:, :, None]).to(F8).view(torch.uint8)
    else:
        for n, x in new.items():
            st[n][at, :, slot] = x.to(st[n].dtype)
    seq, index = _owners(st["back_starts"], st["lengths"], st["back_tokens"])
    at, slot = st["table"][seq, index // page].long(), index % page
    back = []
    for n in ("k", "v"):
        if case["storage"] == "e4m3":
            x = st[n].view(torch.uint8)[at, :, slot].view(F8).float() * st[n + "_scale"][at][:, :, None]
            back.append(x.to(qkv.dtype))
        else:
            back.append(st[n][at, :, slot])
    return {"q": q, "k": back[0], "v": back[1]}


def _plain_attention(st):
    case = st["case"]
    heads, kv, d, f = case["heads"], case["kv_heads"], case["dim"], case["frame"]
    s, n, length = case["sequences"], int(st["news"].max()), case["length"]
    group = heads // kv

    def cached(name):
        x = st[name][st["table"].long()].float()  # [s, pages, kv, page, d]
        if case["storage"] == "e4m3":
            x = x * st[name + "_scale"][st["table"].long()][..., None, None]
        return x.transpose(1, 2).reshape(s, kv, -1, d)[:, :, :length]

    i = torch.arange(n, device=DEV)
    starts, lens = st["starts"].long(), st["lengths"].long()
    count = starts[1:] - starts[:-1]
    live = i < count[:, None]
    token = torch.where(live, starts[:-1, None] + i, 0)
    q = st["q"][token].float().reshape(s, n, kv, group, d).permute(0, 2, 3, 1, 4).reshape(s, kv, group * n, d)
    p = lens[:, None] - count[:, None] + i
    after = (torch.div(p, f, rounding_mode="floor") + 1) * f
    hi = torch.minimum(after, lens[:, None])
    lo = after - case["window"] * f if case["window"] else torch.zeros_like(hi)
    j = torch.arange(length, device=DEV)
    seen = (j < hi[..., None]) & ((j >= lo[..., None]) | (j < case["sinks"])) & live[..., None]
    w = torch.matmul(q, cached("k").transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(s, kv, group, n, length)
    w.masked_fill_(~seen[:, None, None], float("-inf"))
    w = torch.where(live[:, None, None, :, None], w, 0.0)
    w -= w.amax(-1, keepdim=True)
    w.exp_()
    total = w.sum(-1, keepdim=True)
    # keys that no row of a sequence sees hold whatever their pages held: their weights are exact zeros
    o = torch.matmul(w.view(s, kv, group * n, length), cached("v")).view(s, kv, group, n, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(s, n, heads, d)
    return o[live].to(st["q"].dtype)


def _norm(x, kind, w, b, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    return x + b if kind == "layer" else x


def _plain_norm(st):
    case, width = st["case"], st["case"]["width"]
    x, y = st["x"].float(), st["y"].float()
    table = st["table"].float()[torch.arange(case["rows"], device=DEV) // case["per_cond"]]
    gate, shift, scale = table[:, :width], table[:, width:2 * width], table[:, 2 * width:]
    y = _norm(y, case["post"], st["post_w"], st["post_b"], 1e-6)
    if case["residual_scale"]:
        y = y * st["rs"]
    x = x + (gate * y if case["gate"] else y)
    h = _norm(x, case["pre"], st["pre_w"], st["pre_b"], 1e-6)
    if case["modulate"]:
        h = h * (1.0 + scale) + shift
    if case["out_norm"]:
        h = _norm(h, "layer", st["out_w"], st["out_b"], 1e-5)
    return {"x": x.to(st["x"].dtype), "h": h.to(st["y"].dtype)}


# ----------------------------------------------------------- the library

_context = None


def _lib():
    global _context
    if _context is None:
        if "le-wm-nv_b200" not in sys.path:
            sys.path.insert(0, "le-wm-nv_b200")
        import lewm_b200
        ctx = lewm_b200.Context(0)
        # The calls run on the context's own stream.  A program that uses them works on it throughout, as a callback
        # scorer does, and waits once for what it had in hand before.
        stream = ctx.torch_stream()
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
        _context = (lewm_b200, ctx, stream, torch.accelerator.current_stream(), torch.cuda.Event(), torch.cuda.Event())
    return _context


def _own(st):
    L, ctx, stream, usual, ready, done = _lib()
    case, op = st["case"], st["case"]["op"]
    plan = st.get("plan")
    if plan is None:  # what a program lays out once for a model and a batch
        plan = st["plan"] = {}
        if op in ("rotary", "append"):
            plan["rotary"] = L.Rotary.make(st["dims"], st["bases"], case["interleaved"])
        if op in ("append", "attention"):
            plan["cache"] = L.PagedCache(st["k"], st["v"], st.get("k_scale"), st.get("v_scale"),
                                         dtype=DTYPES[case["dtype"]])
            plan["batch"] = L.CacheBatch(st["table"], st["starts"], st["lengths"], st["tokens"],
                                         max_new=int(st["news"].max()), max_length=case["length"])
        if op == "append":
            plan["back"] = L.CacheBatch(st["table"], st["back_starts"], st["lengths"], st["back_tokens"],
                                        max_new=st["back_max"], max_length=case["length"])
            heads, kv = case["heads"], case["kv_heads"]
            plan["q"], plan["k"], plan["v"] = (st["qkv"][:, :heads], st["qkv"][:, heads:heads + kv],
                                               st["qkv"][:, heads + kv:])
        if op == "norm":
            layer = case["pre"] == "layer"
            plan["norm"] = L.GatedNorm(
                post=case["post"], post_weight=st["post_w"], post_bias=st["post_b"] if case["post"] == "layer" else None,
                post_eps=1e-6, residual_scale=st["rs"] if case["residual_scale"] else None, pre=case["pre"],
                pre_weight=st["pre_w"], pre_bias=st["pre_b"] if layer else None, pre_eps=1e-6,
                out_weight=st["out_w"] if case["out_norm"] else None,
                out_bias=st["out_b"] if case["out_norm"] else None, out_eps=1e-5)
            w = case["width"]
            t = st["table"]
            plan["gate"] = t[:, :w] if case["gate"] else None
            plan["shift"] = t[:, w:2 * w] if case["modulate"] else None
            plan["scale"] = t[:, 2 * w:] if case["modulate"] else None
    if torch.accelerator.current_stream() == usual:
        return _call(L, ctx, st, plan)
    # on any other stream: after what it has in hand, and before what it does next
    here = torch.cuda.current_stream()
    ready.record(here)
    stream.wait_event(ready)
    out = _call(L, ctx, st, plan)
    done.record(stream)
    here.wait_event(done)
    return out


def _call(L, ctx, st, plan):
    case, op = st["case"], st["case"]["op"]
    if op == "rotary":
        L.rotary_device(ctx, plan["rotary"], st["x"], st["out"], st["positions"], inverse=case["inverse"])
        return st["out"]
    if op == "norm":
        L.gated_norm_device(ctx, plan["norm"], st["x"], st["y"], st["x_out"], st["h"], gate=plan["gate"],
                            shift=plan["shift"], scale=plan["scale"], rows_per_cond=case["per_cond"])
        return {"x": st["x_out"], "h": st["h"]}
    if op == "attention":
        L.cache_attention_device(ctx, plan["cache"], plan["batch"], st["q"], st["out"], window=case["window"],
                                 sinks=case["sinks"], frame_tokens=case["frame"])
        return st["out"]
    L.cache_append_device(ctx, plan["cache"], plan["batch"], plan["k"], plan["v"], rotary=plan["rotary"],
                          positions=st["positions"], q=plan["q"], q_out=st["q_out"])
    L.cache_gather_device(ctx, plan["cache"], plan["back"], st["k_back"], st["v_back"])
    return {"q": st["q_out"], "k": st["k_back"], "v": st["v_back"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "rotary":
        return _rotate(state, state["x"], state["positions"], state["case"]["inverse"]).to(state["x"].dtype)
    if op == "norm":
        return _plain_norm(state)
    return _plain_attention(state) if op == "attention" else _plain_append(state)


# ------------------------------------------------------------------ work

def _ranges(case, lens, news):
    """Per sequence: keys that some row sees, and (row, key) pairs seen, summed over rows."""
    keys, pairs = 0, 0
    for length, n in zip(lens.tolist(), news.tolist()):
        if n == 0:
            continue
        p = np.arange(length - n, length, dtype=np.int64)
        after = (p // case["frame"] + 1) * case["frame"]
        hi = np.minimum(after, length)
        lo = np.maximum(after - case["window"] * case["frame"], 0) if case["window"] else np.zeros_like(hi)
        first = np.minimum(case["sinks"], np.minimum(lo, hi))
        pairs += int((np.maximum(hi - lo, 0) + first).sum())
        keys += int(hi.max() - min(lo.min(), hi.max())) + int(first.min() if len(first) else 0)
    return keys, pairs


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    e = size[case["dtype"]]
    if case["op"] == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * e + 4 * case["tokens"] * case["axes"], "flops": 3 * n}
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        cond = -(-case["rows"] // case["per_cond"]) * case["width"] * size[case["cond"]]
        return {"bytes": n * 2 * (e + size[case["residual"]]) + cond * (case["gate"] + 2 * case["modulate"]),
                "flops": 20 * n}
    lens, news, starts, table, _ = _batch(case)
    tokens, d, kv = int(starts[-1]), case["dim"], case["kv_heads"]
    store = 1 if case["storage"] == "e4m3" else 2
    if case["op"] == "append":
        back = int(np.where(news > 0, np.minimum(lens, news + case["page"]), 0).sum())
        moved = tokens * d * ((2 * case["heads"] + 2 * kv) * e + 2 * kv * store) + back * d * 2 * kv * (store + e)
        return {"bytes": moved + 4 * tokens * case["axes"], "flops": 3 * tokens * d * (case["heads"] + kv)}
    keys, pairs = _ranges(case, lens, news)
    shared = case["prefix"] // case["page"] * case["page"]
    if shared:
        keys -= shared * (int((news > 0).sum()) - 1)
    return {"bytes": keys * kv * d * 2 * store + 2 * tokens * case["heads"] * d * e,
            "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------- 64-bit results

def _turned(x, positions, dims, bases, interleaved, sign):
    """x [tokens, heads, dim] in 64 bits, each axis' channels as complex numbers times exp(i angle)."""
    parts, off = [], 0
    for a, n in enumerate(dims):
        sec = x[..., off:off + n].double()
        z = torch.complex(sec[..., 0::2], sec[..., 1::2]) if interleaved else torch.complex(sec[..., :n // 2],
                                                                                            sec[..., n // 2:])
        i = torch.arange(n // 2, device=DEV, dtype=torch.float64)
        t = positions[:, a].double()[:, None] * torch.exp(-math.log(bases[a]) * 2.0 * i / n) * sign
        z = z * torch.polar(torch.ones_like(t), t)[:, None]
        parts.append(torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1))
        off += n
    return torch.cat(parts + [x[..., off:].double()], -1)


def _exact_attention(st):
    case = st["case"]
    page, group, f = case["page"], case["heads"] // case["kv_heads"], case["frame"]
    starts, out = st["starts"].tolist(), torch.zeros(st["q"].shape, device=DEV, dtype=torch.float64)
    for s, (length, n) in enumerate(zip(st["lens"].tolist(), st["news"].tolist())):
        if n == 0:
            continue
        rows = st["table"][s, :-(-length // page)].long()
        p = torch.arange(length - n, length, device=DEV)
        block = p // f
        j = torch.arange(length, device=DEV)
        jb = j // f
        seen = jb[None] <= block[:, None]
        if case["window"]:
            seen &= (jb[None] > (block - case["window"])[:, None]) | (j < case["sinks"])[None]
        kv = []
        for name in ("k", "v"):
            x = st[name][rows].double()
            if case["storage"] == "e4m3":
                x = x * st[name + "_scale"][rows].double()[:, :, None, None]
            kv.append(x.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["dim"])[:, :length])
        q = st["q"][starts[s]:starts[s + 1]].double()
        if n == 1:
            qg = q[0].reshape(case["kv_heads"], group, case["dim"])
            w = torch.einsum("hgd,hld->hgl", qg, kv[0]) * case["dim"] ** -0.5
            w = torch.softmax(w.masked_fill(~seen[0], -math.inf), -1)
            out[starts[s]] = torch.einsum("hgl,hld->hgd", w, kv[1]).reshape(case["heads"], case["dim"])
            continue
        for h in range(case["heads"]):
            w = (q[:, h] @ kv[0][h // group].T) * case["dim"] ** -0.5
            w = torch.softmax(w.masked_fill(~seen, -math.inf), -1)
            out[starts[s]:starts[s + 1], h] = w @ kv[1][h // group]
    return out


def _exact_append(st):
    case = st["case"]
    heads, kv, page, quant = case["heads"], case["kv_heads"], case["page"], case["storage"] == "e4m3"
    q = _turned(st["qkv"][:, :heads], st["positions"], st["dims"], st["bases"], case["interleaved"], 1.0)
    k = _turned(st["qkv"][:, heads:heads + kv], st["positions"], st["dims"], st["bases"], case["interleaved"], 1.0)
    new = {"k": k, "v": st["qkv"][:, heads + kv:].double()}
    starts, got = st["starts"].tolist(), {"k": [], "v": []}
    for s, (length, n, b) in enumerate(zip(st["lens"].tolist(), st["news"].tolist(), st["back"].tolist())):
        if n == 0:
            continue
        low = (length - b) // page  # whole pages from here on
        rows = st["table"][s, low:-(-length // page)].long()
        for name, x in new.items():
            old = st[name][rows].double()  # [pages, kv, page, dim]
            if quant:
                old = old * st[name + "_scale"][rows].double()[:, :, None, None]
            line = old.transpose(1, 2).reshape(-1, kv, case["dim"]).clone()
            first = length - n - low * page
            line[first:first + n] = x[starts[s]:starts[s + 1]]
            if quant:
                cut = line.view(len(rows), page, kv, case["dim"])
                at = torch.arange(len(rows), device=DEV) * page
                place = torch.arange(page, device=DEV)
                added = ((at[:, None] + place >= first) & (at[:, None] + place < first + n))
                top = (cut.abs() * added[:, :, None, None]).amax((1, 3))
                need = torch.exp2(torch.ceil(torch.log2(top.clamp_min(1e-30) / 448.0)))
                had = st[name + "_scale"][rows].double()
                scale = torch.where((at >= first)[:, None], need, torch.maximum(need, had))
                scale = torch.where(added.any(1)[:, None], scale, had)[:, None, :, None]
                cut = (cut / scale).to(F8).double() * scale
                line = cut.reshape(-1, kv, case["dim"])
            end = length - low * page
            got[name].append(line[end - b:end])
    return {"q": q, "k": torch.cat(got["k"]), "v": torch.cat(got["v"])}


def _exact_norm(st):
    case = st["case"]
    width, eps = case["width"], 1e-6
    cond = torch.repeat_interleave(st["table"].double(), case["per_cond"], 0)[:case["rows"]].split(width, 1)

    def whole(t, kind, w, b, e):
        if kind == "layer":
            return (t - t.mean(1, True)) * torch.rsqrt((t.square().mean(1, True) - t.mean(1, True).square()) + e) * w.double() + b.double()
        return t * torch.rsqrt(t.square().mean(1, True) + e) * w.double() if kind == "rms" else t

    y = whole(st["y"].double(), case["post"], st["post_w"], st["post_b"], eps)
    if case["gate"]:
        y = y * cond[0]
    if case["residual_scale"]:
        y = y * st["rs"].double()
    x = st["x"].double() + y
    h = whole(x, case["pre"], st["pre_w"], st["pre_b"], eps)
    if case["modulate"]:
        h = h + h * cond[2] + cond[1]
    if case["out_norm"]:
        h = whole(h, "layer", st["out_w"], st["out_b"], 1e-5)
    return {"x": x, "h": h}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        return _turned(st["x"], st["positions"], st["dims"], st["bases"], case["interleaved"],
                       -1.0 if case["inverse"] else 1.0)
    if case["op"] == "norm":
        return _exact_norm(st)
    return _exact_attention(st) if case["op"] == "attention" else _exact_append(st)
