"""More transformer operators of the library at the sizes they are used at.

Three operators of a world model whose candidates continue one history:
attention over a paged cache whose sequences share a long prefix, linear
attention with a decay for each head (a whole history, or a token a sequence)
and drawing tokens from logits with given random numbers.  ``run`` computes an
operator in its plain form, in elementary torch operations, or, where ``own``
is true, through the library.
"""
import math
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F8 = torch.float8_e4m3fn


def listed():
    return [
        # one vehicle, a handful of candidates after one image of history: latency is all of it
        dict(name="shared few", op="shared", groups=1, candidates=8, prefix=197, tail=5, new=1, heads=3, kv_heads=3,
             dim=64, page=16, dtype="bf16", storage="same", window=0, sinks=0, frame=1),
        # the image planner's 1024 candidates after eight frames of 14 x 14 patches
        dict(name="shared candidates", op="shared", groups=1, candidates=1024, prefix=1568, tail=16, new=1, heads=16,
             kv_heads=16, dim=64, page=16, dtype="bf16", storage="same", window=0, sinks=0, frame=1),
        # a fleet on an 8-bit cache: each vehicle's candidates see a window of its history and the first tokens
        dict(name="shared fleet 8 bit", op="shared", groups=16, candidates=64, prefix=8000, tail=40, new=1, heads=16,
             kv_heads=4, dim=128, page=32, dtype="f16", storage="e4m3", window=4096, sinks=4, frame=1),
        # candidates of several tokens each after a very long session, grouped heads: the most arithmetic
        dict(name="shared long session", op="shared", groups=1, candidates=64, prefix=65536, tail=64, new=4, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16", storage="same", window=0, sinks=0, frame=1),
        # one control step of a few vehicles: latency
        dict(name="linear few tokens", op="linear", sequences=8, new=1, heads=3, kv_heads=3, dim=64, dtype="bf16",
             fork=False),
        # a rollout's step of 1024 candidates, each its own state: the states are read and written
        dict(name="linear candidates", op="linear", sequences=1024, new=1, heads=16, kv_heads=16, dim=64, dtype="bf16",
             fork=False),
        # the first step of a rollout: all candidates from the history's one state, grouped heads
        dict(name="linear fork", op="linear", sequences=256, new=1, heads=16, kv_heads=4, dim=128, dtype="f16",
             fork=True),
        # histories of eight frames of 14 x 14 patches for sixteen vehicles
        dict(name="linear video", op="linear", sequences=16, new=1568, heads=16, kv_heads=16, dim=64, dtype="bf16",
             fork=False),
        # one very long session read in: few heads, so the time axis is what there is to share
        dict(name="linear long session", op="linear", sequences=1, new=65536, heads=16, kv_heads=16, dim=128,
             dtype="bf16", fork=False),
        # every candidate's next token of a small codebook
        dict(name="draw codebook", op="draw", rows=1024, vocab=1024, dtype="bf16", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0),
        # a served batch over a text-like vocabulary: a nucleus, and nothing much less likely than the best
        dict(name="draw nucleus", op="draw", rows=256, vocab=32000, dtype="f32", temperature=0.8, top_k=0, top_p=0.95,
             min_p=0.002),
        # few sessions over a large vocabulary: the 50 best of it
        dict(name="draw best of many", op="draw", rows=16, vocab=131072, dtype="bf16", temperature=1.3, top_k=50,
             top_p=0.9, min_p=0.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["shared", "linear", "draw"])
    if op == "shared":
        kv, group = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 4, 8])
        dim = rng.choice([32, 64, 64, 128])
        while True:
            groups, candidates = _log(rng, 1, 32), _log(rng, 2, 1024)
            prefix, tail, new = _log(rng, 1, 65536), _log(rng, 1, 200), rng.choice([1, 1, 1, 2, 5, 16])
            tail = max(tail, new)
            rows = groups * candidates * new * kv * group
            if rows * (prefix + tail) <= 200_000_000 and groups * prefix * kv * dim <= 100_000_000 and \
                    groups * candidates * tail * kv * dim <= 200_000_000:
                break
        frame = rng.choice([1, 1, 1, 49])
        window = 0 if rng.random() < 0.6 else _log(rng, 16, 8192) if frame == 1 else rng.randint(1, 64)
        return dict(op=op, groups=groups, candidates=candidates, prefix=prefix, tail=tail, new=new, heads=kv * group,
                    kv_heads=kv, dim=dim, page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "f16"]),
                    storage=rng.choice(["same", "e4m3"]), window=window,
                    sinks=rng.choice([0, 1, 4, 130]) if window else 0, frame=frame)
    if op == "linear":
        kv, group, dim = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 4]), rng.choice([32, 64, 64, 128])
        heads = kv * group
        while True:
            sequences, new = _log(rng, 1, 1024), 1 if rng.random() < 0.4 else _log(rng, 1, 65536)
            if sequences * heads * dim * dim <= 70_000_000 and sequences * new * heads * dim <= 130_000_000:
                break
        return dict(op=op, sequences=sequences, new=new, heads=heads, kv_heads=kv, dim=dim,
                    dtype=rng.choice(["bf16", "f16"]), fork=rng.random() < 0.4)
    rows, vocab = _log(rng, 1, 2048), _log(rng, 2, 200_000)
    rows = min(rows, max(1, 20_000_000 // vocab))
    return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "f16"]),
                temperature=round(rng.uniform(0.3, 2.0), 2), top_k=rng.choice([0, 0, 1, 20, 50, 1000]),
                top_p=rng.choice([1.0, 0.5, 0.9, 0.95]), min_p=rng.choice([0.0, 0.0, 0.001, 0.1]))


# --------------------------------------------------------------- inputs

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _batch(case):
    """Host plan of candidates in groups that share a prefix: it goes by the case alone, so that other values come in
    the same shapes.  Groups and tails are ragged, every seventh candidate of a large batch rests; only whole pages of
    a prefix are shared, its last page is each candidate's own copy."""
    rng = np.random.default_rng([case["groups"], case["candidates"], case["prefix"], case["tail"], case["page"]])
    n, page = case["groups"], case["page"]
    sizes = rng.integers((case["candidates"] + 1) // 2, case["candidates"] + 1, n)
    shared = rng.integers((case["prefix"] + 1) // 2, case["prefix"] + 1, n)
    sizes[0], shared[0] = case["candidates"], case["prefix"]
    groups = np.zeros(n + 1, np.int32)
    groups[1:] = np.cumsum(sizes)
    s = int(groups[-1])
    of = np.repeat(np.arange(n), sizes)
    tails = rng.integers((case["tail"] + 1) // 2, case["tail"] + 1, s)
    news = rng.integers((case["new"] + 1) // 2, case["new"] + 1, s)
    tails[0], news[0] = case["tail"], case["new"]
    news = np.minimum(news, tails)
    if s >= 14:
        news[6::7] = 0
    lens = shared[of] + tails
    whole = shared // page
    per = -(-lens // page) - whole[of]  # pages of each sequence's own
    total = int(whole.sum() + per.sum())
    order = rng.permutation(total + 3)[:total]  # pages lie anywhere in the pool
    table = np.zeros((s, int((-(-lens // page)).max())), np.int32)
    first = np.concatenate([[0], np.cumsum(whole)])
    at = int(whole.sum())
    for i in range(s):
        w, p = int(whole[of[i]]), int(per[i])
        table[i, :w] = order[first[of[i]]:first[of[i]] + w]
        table[i, w:w + p] = order[at:at + p]
        at += p
    starts = np.zeros(s + 1, np.int32)
    starts[1:] = np.cumsum(news)
    return dict(groups=groups, shared=shared.astype(np.int32), of=of, lens=lens.astype(np.int32),
                news=news.astype(np.int32), starts=starts, table=table, pages=total + 3)


def _page_scale(amax):
    """The least power of two with amax <= 448 times it."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, -120)).clamp(-120, 120))


def _pools(case, b, g):
    """Cached keys and values: 16 bits, or e4m3 codes with the scale of each page and head; the page that a prefix
    ends in holds the same tokens in every candidate's copy."""
    page, shape = case["page"], (b["pages"], case["kv_heads"], case["page"], case["dim"])
    out = {}
    for name in ("k", "v"):
        x = _normal(g, *shape)
        if name == "v":
            x *= torch.exp(0.5 * _normal(g, b["pages"], case["kv_heads"], 1, 1))  # pages differ in size
        codes = case["storage"] == "e4m3"
        if codes:
            scale = _page_scale(x.abs().amax((2, 3)))
            x = (x / scale[:, :, None, None]).to(F8).view(torch.uint8)
        else:
            x = x.to(DTYPES[case["dtype"]])
        slots = torch.arange(page, device=DEV)
        rest, leader = b["shared"] % page, b["groups"][:-1]
        mine = _dev(b["table"][np.arange(len(b["of"])), (b["shared"] // page)[b["of"]]]).long()
        theirs = _dev(b["table"][leader, b["shared"] // page][b["of"]]).long()
        same = (slots < _dev(rest[b["of"]])[:, None])[:, None, :, None]
        x[mine] = torch.where(same, x[theirs], x[mine])
        out[name] = x.view(F8) if codes else x
        if codes:
            scale[mine] = torch.where(_dev(rest[b["of"]] > 0)[:, None], scale[theirs], scale[mine])
            out[name + "_scale"] = scale
    return out


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    st = dict(case=case)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "draw":
        rows, vocab = case["rows"], case["vocab"]
        # most tokens unlikely, a few peaks, and each row with a spread of its own
        x = _normal(g, rows, vocab) * (1.0 + 2.0 * torch.rand(rows, 1, generator=g, device=DEV))
        x += 6.0 * (torch.rand(rows, vocab, generator=g, device=DEV) < min(0.2, 30.0 / vocab))
        st["logits"] = x.to(dt)
        st["uniform"] = torch.rand(rows, generator=g, device=DEV)
        st["tokens"] = torch.empty(rows, device=DEV, dtype=torch.int32)
        st["log_probs"] = torch.empty(rows, device=DEV)
        return st
    if case["op"] == "shared":
        b = st["batch"] = _batch(case)
        st.update(table=_dev(b["table"]), starts=_dev(b["starts"]), lengths=_dev(b["lens"]), groups=_dev(b["groups"]),
                  shared=_dev(b["shared"]), tokens=int(b["starts"][-1]))
        st.update(_pools(case, b, g))
        st["q"] = _normal(g, st["tokens"], case["heads"], case["dim"]).to(dt)
        st["out"] = torch.empty_like(st["q"])
        return st
    rng = np.random.default_rng([case["sequences"], case["new"], case["heads"]])
    s, h, d = case["sequences"], case["heads"], case["dim"]
    news = rng.integers((case["new"] + 1) // 2, case["new"] + 1, s)
    news[0] = case["new"]
    if s >= 14:
        news[6::7] = 0
    starts = np.zeros(s + 1, np.int32)
    starts[1:] = np.cumsum(news)
    tokens = int(starts[-1])
    # states before the call, then the slots for the states after it, in any order
    held = 1 if case["fork"] else s
    source = np.zeros(s, np.int32) if case["fork"] else rng.permutation(s).astype(np.int32)
    target = (held + rng.permutation(s)).astype(np.int32)
    st.update(news=news, tokens=tokens, starts=_dev(starts), source=_dev(source), target=_dev(target), held=held)
    st["states"] = torch.zeros(held + s, h, d, d, device=DEV)
    st["states"][:held] = 3.0 * _normal(g, held, h, d, d)
    # a fused projection's output: queries, keys and values of a token side by side
    kv = case["kv_heads"]
    st["qkv"] = _normal(g, tokens, h + 2 * kv, d).to(dt)
    # heads forget at rates from 1 / 32 to 1 / 4096 a token
    st["log_decay"] = torch.log1p(-torch.exp2(-5.0 - 7.0 * torch.arange(h, device=DEV, dtype=torch.float64)
                                              / max(1, h - 1))).float()
    st["out"] = torch.empty(tokens, h, d, device=DEV, dtype=dt)
    return st


# ----------------------------------------------------------- plain forms

def _plain_shared(st):
    case, b = st["case"], st["batch"]
    heads, kv, d, f, page = case["heads"], case["kv_heads"], case["dim"], case["frame"], case["page"]
    group, n_groups, tokens = heads // kv, case["groups"], st["tokens"]
    starts, lens, groups, shared = (st[n].long() for n in ("starts", "lengths", "groups", "shared"))
    t = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(starts[1:], t, right=True)
    grp = torch.searchsorted(groups[1:], seq, right=True)
    p = lens[seq] - (starts[seq + 1] - t)  # cache index of each token
    after = (torch.div(p, f, rounding_mode="floor") + 1) * f
    hi = torch.minimum(after, lens[seq])
    lo = after - case["window"] * f if case["window"] else torch.zeros_like(hi)

    def cached(name, rows, index):  # [b, n] pages and slots to [b, kv, n, d]
        pages = rows.gather(1, index // page).long()
        x = st[name].view(torch.uint8) if case["storage"] == "e4m3" else st[name]
        x = x[pages, :, index % page]
        if case["storage"] == "e4m3":
            x = x.view(F8).float() * st[name + "_scale"][pages][..., None]
        return x.float().transpose(1, 2)

    # rows in blocks: of a group for the prefix, of a sequence for what follows it
    row0 = starts[groups[:-1]]
    per_group, per_seq = int((b["starts"][b["groups"][1:]] - b["starts"][b["groups"][:-1]]).max()), int(b["news"].max())
    in_group, in_seq = t - row0[grp], t - starts[seq]
    q = st["q"].float().view(tokens, kv, group, d)
    n_seq, n_key, n_tail = len(b["lens"]), int(b["shared"].max()), int((b["lens"] - b["shared"][b["of"]]).max())
    qg = torch.zeros(n_groups, per_group, kv, group, d, device=DEV)
    qs = torch.zeros(n_seq, per_seq, kv, group, d, device=DEV)
    qg[grp, in_group], qs[seq, in_seq] = q, q
    j = torch.arange(n_key, device=DEV)
    jg = torch.minimum(j, shared[:, None] - 1).clamp_min(0)
    js = torch.arange(n_tail, device=DEV) + shared[torch.searchsorted(groups[1:], torch.arange(n_seq, device=DEV),
                                                                       right=True)][:, None]
    jc = torch.minimum(js, lens[:, None] - 1)
    scale = 1.0 / math.sqrt(d)

    def scores(rows, keys):  # [b, n, kv, group, d] and [b, kv, m, d] to [b, n, kv, group, m]
        w = torch.matmul(rows.permute(0, 2, 3, 1, 4).flatten(2, 3), keys.transpose(2, 3)).mul_(scale)
        return w.view(w.shape[0], kv, group, -1, w.shape[-1]).permute(0, 3, 1, 2, 4)

    def weighted(w, values):
        o = torch.matmul(w.permute(0, 2, 3, 1, 4).flatten(2, 3), values)
        return o.view(o.shape[0], kv, group, -1, d).permute(0, 3, 1, 2, 4)

    kept = (j >= lo[:, None]) | (j < case["sinks"])
    wp = scores(qg, cached("k", st["table"][groups[:-1]], jg))[grp, in_group]
    wp.masked_fill_(~(kept & (j < shared[grp][:, None]))[:, None, None], float("-inf"))
    at = js[seq]
    wt = scores(qs, cached("k", st["table"], jc))[seq, in_seq]
    wt.masked_fill_(~((at < hi[:, None]) & ((at >= lo[:, None]) | (at < case["sinks"])))[:, None, None], float("-inf"))
    top = torch.maximum(wp.amax(-1, keepdim=True), wt.amax(-1, keepdim=True))
    wp, wt = wp.sub_(top).exp_(), wt.sub_(top).exp_()
    total = wp.sum(-1, keepdim=True) + wt.sum(-1, keepdim=True)
    back = torch.zeros(n_groups, per_group, kv, group, n_key, device=DEV)
    back[grp, in_group] = wp
    o = weighted(back, cached("v", st["table"][groups[:-1]], jg))[grp, in_group]
    back = torch.zeros(n_seq, per_seq, kv, group, n_tail, device=DEV)
    back[seq, in_seq] = wt
    o = (o + weighted(back, cached("v", st["table"], jc))[seq, in_seq]) / total
    return o.reshape(tokens, heads, d).to(st["q"].dtype)


def _split(st):
    h, kv = st["case"]["heads"], st["case"]["kv_heads"]
    return st["qkv"][:, :h], st["qkv"][:, h:h + kv], st["qkv"][:, h + kv:]


def _plain_linear(st):
    case = st["case"]
    s, h, kv, d = case["sequences"], case["heads"], case["kv_heads"], case["dim"]
    n = int(st["news"].max())
    c = min(128, n)  # tokens of a chunk
    chunks = -(-n // c)
    starts, a = st["starts"].long(), st["log_decay"].double()
    t = torch.arange(st["tokens"], device=DEV)
    seq = torch.searchsorted(starts[1:], t, right=True)
    place = t - starts[seq]
    count = (starts[1:] - starts[:-1])

    def padded(x):  # [tokens, heads, d] to [s, heads, chunks, c, d]
        out = torch.zeros(s, chunks * c, x.shape[1], d, device=DEV)
        out[seq, place] = x.float()
        out = out.repeat_interleave(h // x.shape[1], 2) if x.shape[1] < h else out
        return out.view(s, chunks, c, h, d).permute(0, 3, 1, 2, 4)

    q, k, v = (padded(x) for x in _split(st))
    before = st["states"][st["source"].long()]
    i = torch.arange(c, device=DEV)
    apart = i[:, None] - i
    near = torch.where(apart >= 0, torch.exp(a[:, None, None] * apart.clamp_min(0)), 0.0).float()
    w = torch.matmul(q, k.transpose(-1, -2)) * near[None, :, None]
    o = torch.matmul(w, v)
    # states before each chunk: what each chunk adds, and the decay from its end to there
    to_end = torch.exp(a[:, None] * (c - 1 - i)).float()
    added = torch.matmul((k * to_end[None, :, None, :, None]).transpose(-1, -2), v).flatten(3)
    m = torch.arange(chunks, device=DEV)
    far = m[:, None] - 1 - m
    weigh = torch.where(far >= 0, torch.exp(a[:, None, None] * c * far.clamp_min(0)), 0.0).float()
    held = torch.matmul(weigh, added).view(s, h, chunks, d, d)
    held = held + torch.exp(a[:, None] * c * m).float()[None, :, :, None, None] * before[:, :, None]
    o = o + torch.matmul(q, held) * torch.exp(a[:, None] * (i + 1)).float()[None, :, None, :, None]
    o = o.permute(0, 2, 3, 1, 4).reshape(s, chunks * c, h, d)[seq, place] * d ** -0.5
    # the states after the last tokens
    left = count[:, None, None] - 1 - (m[:, None] * c + i).view(1, chunks, c)
    w = torch.where(left[:, None] >= 0, torch.exp(a[None, :, None, None] * left.clamp_min(0)[:, None]), 0.0).float()
    state = torch.matmul((k * w[..., None]).flatten(2, 3).transpose(-1, -2), v.flatten(2, 3))
    state = state + torch.exp(a * count[:, None]).float()[..., None, None] * before
    st["states"][st["target"].long()] = state
    return {"out": o.to(st["qkv"].dtype), "states": st["states"][st["held"]:]}


def _plain_draw(st):
    case = st["case"]
    x = st["logits"].double()
    rank = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((rank.values - rank.values[:, :1]) / case["temperature"])
    if case["top_k"]:
        w[:, case["top_k"]:] = 0.0
    total = w.sum(1, keepdim=True)
    kept = w >= case["min_p"]
    if case["top_p"] < 1.0:
        before = torch.cat([torch.zeros_like(total), w.cumsum(1)[:, :-1]], 1)
        kept &= before < case["top_p"] * total
    w = torch.where(kept, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, rank.indices, w)
    upto = w.cumsum(1)
    total = w.sum(1, keepdim=True)
    token = (upto <= st["uniform"].double()[:, None] * total).sum(1, keepdim=True)
    last = case["vocab"] - 1 - (w.flip(1) > 0).int().argmax(1, keepdim=True)
    token = torch.minimum(token, last)
    log_prob = torch.log(w.gather(1, token) / total)
    return {"tokens": token[:, 0].int(), "log_probs": log_prob[:, 0].float()}


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
    case = st["case"]
    plan = st.get("plan")
    if plan is None:  # what a program lays out once for a model and a batch
        plan = st["plan"] = {}
        if case["op"] == "shared":
            b = st["batch"]
            plan["cache"] = L.PagedCache(st["k"], st["v"], st.get("k_scale"), st.get("v_scale"),
                                         dtype=DTYPES[case["dtype"]])
            plan["batch"] = L.CacheBatch(st["table"], st["starts"], st["lengths"], st["tokens"],
                                         max_new=int(b["news"].max()), max_length=int(b["lens"].max()))
            rows = b["starts"][b["groups"]]
            plan["prefix"] = L.SharedPrefix(st["groups"], st["shared"], max_tokens=int((rows[1:] - rows[:-1]).max()),
                                            max_length=int(b["shared"].max()),
                                            max_tail=int((b["lens"] - b["shared"][b["of"]]).max()))
            size = L.shared_attention_workspace(plan["cache"], plan["batch"], plan["prefix"], case["heads"],
                                                window=case["window"], sinks=case["sinks"], frame_tokens=case["frame"])
            plan["workspace"] = torch.empty(size, device=DEV, dtype=torch.uint8)
        if case["op"] == "linear":
            plan["states"] = L.StateBatch(st["states"], st["starts"], st["tokens"], int(st["news"].max()),
                                          source=st["source"], target=st["target"])
            plan["qkv"] = _split(st)
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
    case = st["case"]
    if case["op"] == "shared":
        L.cache_attention_shared_device(ctx, plan["cache"], plan["batch"], plan["prefix"], st["q"], st["out"],
                                        plan["workspace"], window=case["window"], sinks=case["sinks"],
                                        frame_tokens=case["frame"])
        return st["out"]
    if case["op"] == "linear":
        q, k, v = plan["qkv"]
        L.linear_attention_device(ctx, plan["states"], q, k, v, st["out"], st["log_decay"])
        return {"out": st["out"], "states": st["states"][st["held"]:]}
    L.sample_tokens_device(ctx, st["logits"], st["uniform"], st["tokens"], st["log_probs"],
                           temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"],
                           min_p=case["min_p"])
    return {"tokens": st["tokens"], "log_probs": st["log_probs"]}


def run(state):
    if own:
        return _own(state)
    return {"shared": _plain_shared, "linear": _plain_linear, "draw": _plain_draw}[state["case"]["op"]](state)


# ------------------------------------------------------------------ work

def work(case):
    e = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] == "draw":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + 12 * case["rows"], "flops": 10 * n}
    d, kv, heads = case["dim"], case["kv_heads"], case["heads"]
    if case["op"] == "linear":
        rng = np.random.default_rng([case["sequences"], case["new"], case["heads"]])
        s = case["sequences"]
        news = rng.integers((case["new"] + 1) // 2, case["new"] + 1, s)
        news[0] = case["new"]
        if s >= 14:
            news[6::7] = 0
        tokens, held = int(news.sum()), 1 if case["fork"] else s
        return {"bytes": tokens * d * (2 * heads + 2 * kv) * e + (held + s) * heads * d * d * 4,
                "flops": 4 * tokens * heads * d * d}
    b, f = _batch(case), case["frame"]
    # per row, the keys of the prefix and of its tail that it sees; per group, those that any of its rows sees
    seq = np.repeat(np.arange(len(b["news"])), b["news"])
    tokens, of = len(seq), b["of"][seq]
    p = b["lens"][seq].astype(np.int64) - (b["starts"][seq + 1] - np.arange(tokens))
    after = (p // f + 1) * f
    lo = np.maximum(after - case["window"] * f, 0) if case["window"] else np.zeros_like(after)
    hi, cut, sinks = np.minimum(after, b["lens"][seq]), b["shared"][of].astype(np.int64), case["sinks"]

    def seen(a, z):  # keys of [a, z) that a row sees
        first = np.clip(np.minimum(sinks, lo), a, z) - a
        return np.maximum(z - np.clip(lo, a, z), 0) + first
    zero = np.zeros_like(cut)
    pairs = int((seen(zero, cut) + seen(cut, np.maximum(hi, cut))).sum())
    keys = 0
    for i in range(case["groups"]):
        mine = of == i
        if mine.any():
            low = min(int(lo[mine].min()), int(b["shared"][i]))
            keys += int(b["shared"][i]) - low + min(sinks, low)
    own_lo = np.full(len(b["news"]), np.iinfo(np.int64).max)
    np.minimum.at(own_lo, seq, lo)
    live = b["news"] > 0
    keys += int((b["lens"] - np.clip(own_lo, b["shared"][b["of"]], b["lens"]))[live].sum())
    store = 1 if case["storage"] == "e4m3" else 2
    return {"bytes": keys * kv * d * 2 * store + 2 * tokens * heads * d * e, "flops": 4 * pairs * heads * d}


# ------------------------------------------------------- 64-bit results

def _exact_shared(st):
    case, b = st["case"], st["batch"]
    page, group, f = case["page"], case["heads"] // case["kv_heads"], case["frame"]
    out = torch.zeros(st["q"].shape, device=DEV, dtype=torch.float64)
    for s, (length, n) in enumerate(zip(b["lens"].tolist(), b["news"].tolist())):
        if n == 0:
            continue
        rows = st["table"][s, :-(-length // page)].long()
        kv = []
        for name in ("k", "v"):
            x = st[name][rows].double()
            if case["storage"] == "e4m3":
                x = x * st[name + "_scale"][rows].double()[:, :, None, None]
            kv.append(x.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["dim"])[:, :length])
        p = torch.arange(length - n, length, device=DEV)
        jb, block, j = torch.arange(length, device=DEV) // f, p // f, torch.arange(length, device=DEV)
        seen = jb[None] <= block[:, None]
        if case["window"]:
            seen &= (jb[None] > (block - case["window"])[:, None]) | (j < case["sinks"])[None]
        first = int(b["starts"][s])
        q = st["q"][first:first + n].double().view(n, case["kv_heads"], group, case["dim"])
        w = torch.einsum("nhgd,hld->hgnl", q, kv[0]) * case["dim"] ** -0.5
        w = torch.softmax(w.masked_fill(~seen, -math.inf), -1)
        out[first:first + n] = torch.einsum("hgnl,hld->nhgd", w, kv[1]).reshape(n, case["heads"], case["dim"])
    return out


def _exact_linear(st):
    """The recurrence in steps of at most 32 tokens, all sequences at once."""
    case = st["case"]
    s, h, d = case["sequences"], case["heads"], case["dim"]
    count = torch.from_numpy(st["news"]).to(DEV)
    starts, lam = st["starts"].long()[:-1], torch.exp(st["log_decay"].double())
    q, k, v = _split(st)
    share = h // case["kv_heads"]
    state = st["states"][st["source"].long()].double()
    out = torch.zeros(st["tokens"], h, d, device=DEV, dtype=torch.float64)
    step = 32
    power = lam[:, None] ** torch.arange(step + 1, device=DEV)
    i = torch.arange(step, device=DEV)
    near = torch.tril(lam[:, None, None] ** (i[:, None] - i).clamp_min(0))
    for first in range(0, int(st["news"].max()), step):
        live = (first + i)[None] < count[:, None]
        at = torch.where(live, starts[:, None] + first + i, 0)
        part = [torch.where(live[..., None, None], x[at].double(), 0.0).transpose(1, 2) for x in (q, k, v)]
        qq, kk, vv = part[0], *(x.repeat_interleave(share, 1) for x in part[1:])
        o = torch.einsum("shid,shde->shie", qq * power[:, 1:, None], state)
        o = o + torch.einsum("shij,hij,shje->shie", qq @ kk.transpose(-1, -2), near, vv)
        out[at[live]] = o.transpose(1, 2)[live] * d ** -0.5
        n = (count - first).clamp(0, step)
        left = n[:, None] - 1 - i
        w = torch.where(left[:, None] >= 0, lam[None, :, None] ** left.clamp_min(0)[:, None], 0.0)
        state = state * (lam ** n[:, None])[..., None, None] + torch.einsum("shi,shid,shie->shde", w, kk, vv)
    states = st["states"].double()
    states[st["target"].long()] = state
    return {"out": out, "states": states[st["held"]:]}


def _exact_draw(st):
    case = st["case"]
    x, u = st["logits"].double().cpu().numpy(), st["uniform"].double().cpu().numpy()
    tokens, logs = [], []
    for row, point in zip(x, u):
        w = np.exp((row - row.max()) / case["temperature"])
        best = np.lexsort((np.arange(len(row)), -row))[:case["top_k"] or None]
        total = math.fsum(w[best])
        n = len(best)
        if case["top_p"] < 1.0:
            n = 1 + int(np.searchsorted(np.cumsum(w[best]), case["top_p"] * total, side="left"))
        kept = np.sort(best[:n][w[best[:n]] >= case["min_p"]])
        sums = np.cumsum(w[kept])
        i = min(int(np.searchsorted(sums, point * sums[-1], side="right")), len(kept) - 1)
        tokens.append(int(kept[i]))
        logs.append(math.log(w[kept[i]]) - math.log(sums[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=DEV),
            "log_probs": torch.tensor(logs, dtype=torch.float64, device=DEV)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"shared": _exact_shared, "linear": _exact_linear, "draw": _exact_draw}[case["op"]](st)
