"""Attention of sequences that share a prefix against 64 bits, with the
reference, tolerances and pools of the plain cache attention: every type and
width, prefixes that end in pages or not, ragged groups, rows of one token and
many, masks inside the prefix and behind it, keys split and not, what is not
seen, and what the call skips and reports.

The join adds to a row's error: the logarithms of the parts' sums (2^-22 and
half a step of a number up to 2^8 each, 2^-16 in the exponent) scale whole
parts, which is 2^-15 of the mass at most; everything else is as in the plain
attention."""
import numpy as np
import pytest

import lewm_b200 as L
from test_gpu_blocks import Paged, attention_64, attention_tolerance, close, gen, ints, mask_of, randn

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
POOLS = [(BF16, False), (F16, False), (BF16, True), (F16, True)]
# What makes the groups the cheaper way by the library's costs, whatever the sizes: a bound of the lengths, or, with a
# window, many sequences that have no rows (by themselves they would cost a window each, here a tail).
LONG, RESTING = 1 << 22, 30000


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


class Groups:
    """Groups (prefix, tails) in a pool: whole pages of a prefix are the first sequence's, the page it ends in is a
    copy in each."""

    def __init__(self, seed, groups, page, kv, d, dtype=BF16, codes=False, alone=()):
        self.prefix = [p for p, tails in groups for _ in tails] + [0] * len(alone)
        lengths = [p + t for p, tails in groups for t in tails] + list(alone)
        self.c = c = Paged(seed, lengths, page, kv, d, dtype, codes)
        c.fill_random(seed)
        s = 0
        self.starts = [0]
        for p, tails in groups:
            lead, w, rest = s, p // page, p % page
            for s in range(lead, lead + len(tails)):
                c.table[s, :w] = c.table[lead, :w]
                if rest and s > lead:
                    a, b = int(c.table[lead, w]), int(c.table[s, w])
                    for pool, scale in ((c.k, c.ks), (c.v, c.vs)):
                        pool = pool.view(torch.uint8) if codes else pool
                        pool[b, :, :rest] = pool[a, :, :rest]
                        if codes:
                            scale[b] = scale[a]
            s = lead + len(tails)
            self.starts.append(s)
        self.lengths = [p for p, _ in groups]

    def call(self, ctx, news, heads, seed=1, causal=True, window=0, sinks=0, frame=1, scale=None, behind=3, q=None,
             max_length=0, max_tail=0, max_tokens=None, split=None):
        c = self.c
        tokens = sum(news) + behind
        q = randn(gen(seed), tokens, heads, c.d, dtype=c.dtype) if q is None else q
        out = torch.full((tokens, heads, c.d), 5.0, device="cuda", dtype=c.dtype)
        b = self.batch(news, tokens, window)
        max_tail = max_tail or (1 if window else max(n - p for n, p in zip(c.lengths, self.prefix)))
        p = L.SharedPrefix(ints(self.starts), ints(self.lengths), max_tokens, max_length or max(self.lengths + [1]), max_tail)
        mask = dict(causal=causal, window=window, sinks=sinks, frame_tokens=frame)
        size = L.shared_attention_workspace(c.cache, b, p, heads, **mask)
        assert size > 0  # the kernels of this operator run
        if split is not None:
            assert (size // (tokens * heads * (c.d + 1) * 4) > 1) == split
        work = torch.full((size + 64,), 0x7f, device="cuda", dtype=torch.uint8)
        L.cache_attention_shared_device(ctx, c.cache, b, p, q, out, work[:size], scale=scale, **mask)
        ctx.synchronize()
        assert (work[size:] == 0x7f).all()
        self.check(q, out, news, causal, window, sinks, frame, scale)
        return q, out

    def batch(self, news, tokens, window):
        c, rest = self.c, RESTING if window else 0
        table = np.concatenate([c.table, np.full((rest, c.table.shape[1]), -1)])
        starts = np.concatenate([[0], np.cumsum(list(news) + [0] * rest)])
        return L.CacheBatch(ints(table), ints(starts), ints(c.lengths + [0] * rest), tokens, max(news), LONG)

    def check(self, q, out, news, causal=True, window=0, sinks=0, frame=1, scale=None):
        c, t = self.c, 0
        for s, (length, n) in enumerate(zip(c.lengths, news)):
            if n:
                parts = attention_64(q[t:t + n].double(), c.dense("k", s), c.dense("v", s),
                                     mask_of(length, n, causal, window, sinks, frame), c.d ** -0.5 if scale is None else scale)
                vs = float(c.vs[c.table[s, :-(-length // c.page)]].nan_to_num(0).max()) if c.codes else 0.0
                close(out[t:t + n], parts[0], attention_tolerance(*parts, c.d, c.dtype, c.codes, vs) + parts[1] * 2.0 ** -15)
            t += n
        assert (out[t:] == 5.0).all()


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 128])
def test_single_tokens(ctx, dtype, codes, d, page):
    g = Groups(1, [(200, [1, 5, 40, 17]), (1, [3, 1]), (128, [1] * 5)], page, 2, d, dtype, codes)
    g.call(ctx, [1] * 11, 4)
    g.call(ctx, [1, 0, 1, 1, 0, 0, 1, 0, 1, 1, 0], 2)


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("window,sinks,frame", [(0, 0, 1), (0, 0, 7), (60, 0, 1), (60, 4, 1), (150, 130, 1), (3, 49, 49),
                                                (1, 0, 30), (9, 300, 1), (250, 0, 1)])
def test_masks_inside_the_prefix_and_behind_it(ctx, dtype, codes, window, sinks, frame):
    g = Groups(2, [(290, [30, 2, 11, 150]), (77, [9, 20])], 32, 2, 64, dtype, codes)
    g.call(ctx, [3, 2, 11, 20, 1, 20], 4, window=window, sinks=sinks, frame=frame)
    g.call(ctx, [3, 2, 1, 20, 9, 2], 2, window=window, sinks=sinks, frame=frame, causal=False)


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("kv,heads,d", [(1, 1, 64), (3, 3, 64), (2, 8, 128), (1, 5, 32)])
def test_heads_and_many_rows(ctx, dtype, codes, kv, heads, d):
    """More rows than one block takes, and a group of one sequence."""
    g = Groups(3, [(333, [4] * 90), (64, [2])], 64, kv, d, dtype, codes)
    g.call(ctx, [4] * 90 + [1], heads)


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [64, 128])
def test_long_prefixes_are_split_and_joined(ctx, dtype, codes, d):
    g = Groups(4, [(5000, [1, 9, 30])], 64, 1, d, dtype, codes)
    g.call(ctx, [1, 2, 1], 2, split=True)
    g.call(ctx, [1, 2, 1], 2, window=3000, sinks=700, split=True)  # parts that begin and end among the sinks
    g.call(ctx, [1, 2, 1], 2, window=100, sinks=4, split=False)  # (one tile of keys has no parts)


def test_parts_without_a_key(ctx):
    """A group's prefix of one tile beside one that is cut into many parts."""
    g = Groups(5, [(6000, [3, 5]), (20, [4, 1]), (1, [1])], 64, 1, 64)
    g.call(ctx, [1] * 5, 1, split=True)


@pytest.mark.parametrize("dtype,codes", POOLS)
def test_long_tails(ctx, dtype, codes):
    """Few jobs: four warps and a cluster share a tail."""
    g = Groups(6, [(100, [3000, 1200, 1])], 64, 2, 64, dtype, codes)
    g.call(ctx, [1, 3, 1], 4, max_tail=3000)
    g.call(ctx, [1, 3, 1], 4, max_tail=300, window=500, sinks=160)  # (a bound that is too low costs time only)


def test_many_candidates_take_a_warp_each(ctx):
    g = Groups(7, [(150, [1 + i % 20 for i in range(300)]), (40, [3] * 50)], 16, 4, 64)
    g.call(ctx, [1] * 350, 4, max_tail=20)
    g.call(ctx, [1 - (i % 7 == 6) for i in range(350)], 4, max_tail=20, window=30, sinks=3)
    g = Groups(8, [(150, [1 + i % 20 for i in range(300)])], 16, 4, 128, F16, True)
    g.call(ctx, [1] * 300, 8, max_tail=20)


def test_sequences_of_no_group_and_empty_groups(ctx):
    g = Groups(9, [(50, [3, 4]), (0, [2, 7])], 16, 2, 64, alone=[70, 5])
    g.starts.insert(1, g.starts[1])  # nothing in it
    g.lengths.insert(1, 0)
    g.call(ctx, [1, 2, 1, 1, 3, 1], 2)
    # groups that begin late
    g.starts, g.lengths = [2, 4], [0]
    g.call(ctx, [1, 2, 1, 1, 3, 1], 2, max_length=50)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.2])
def test_scale(ctx, scale):
    Groups(10, [(140, [3, 9])], 16, 1, 64).call(ctx, [2, 1], 2, scale=scale)


def test_one_side_far_above_the_other(ctx):
    """Scores of the prefix hundreds above the tail's, and the other way round: weights that vanish, no NaN."""
    for high in ("prefix", "tail"):
        g = Groups(11, [(100, [20, 20])], 32, 1, 64)
        c = g.c
        q = torch.ones(5, 1, 64, device="cuda", dtype=BF16)
        for s in range(2):
            for j in range(-(-c.lengths[s] // 32)):
                at = torch.arange(j * 32, j * 32 + 32, device="cuda")
                up = (at < 100) if high == "prefix" else (at >= 100)
                c.k[int(c.table[s, j])] = torch.where(up, 30.0, -30.0).to(BF16)[None, :, None]
        g.call(ctx, [1, 1], 1, q=q)


@pytest.mark.parametrize("dtype,codes", POOLS)
def test_rows_are_not_reached_by_what_they_do_not_see(ctx, dtype, codes):
    """NaN in a token of the prefix and in one candidate's tail, inside the window and outside."""
    g = Groups(12, [(200, [60, 2, 2])], 32, 1, 64, dtype, codes)
    c = g.c
    clean_q, clean = g.call(ctx, [1, 1, 1], 1, window=150, sinks=0)
    page = int(c.table[1, 3])  # tokens 96 .. 127 of the prefix
    other = int(c.table[0, 7])  # tokens 224 .. of the first candidate's tail
    for pool in (c.k, c.v):
        pool = pool.view(torch.uint8) if codes else pool
        pool[page, :, 110 - 96] = 0x7f if codes else float("nan")
        pool[other, :, 3] = 0x7f if codes else float("nan")
    b = g.batch([1, 1, 1], 6, 150)
    p = L.SharedPrefix(ints(g.starts), ints(g.lengths), None, 200, 1)
    size = L.shared_attention_workspace(c.cache, b, p, 1, window=150)
    out = torch.zeros_like(clean)
    L.cache_attention_shared_device(ctx, c.cache, b, p, clean_q, out, torch.empty(size, device="cuda", dtype=torch.uint8), window=150)
    ctx.synchronize()
    assert torch.isnan(out[:3]).all()  # 110 .. 259 and 52 .. 201
    # a shorter window leaves token 110 out for all of them, and 227 for the first
    out.zero_()
    L.cache_attention_shared_device(ctx, c.cache, b, p, clean_q, out, torch.empty(size, device="cuda", dtype=torch.uint8), window=20)
    ctx.synchronize()
    assert not torch.isnan(out[:3]).any()  # 240 .. 259 and 182 .. 201


def test_in_place_strides_and_repeats(ctx):
    g = Groups(13, [(500, [8, 3, 20]), (30, [5])], 32, 2, 64)
    c, news = g.c, [2, 1, 3, 1]
    big = randn(gen(3), 7, 9, 80, dtype=BF16)
    q = big[:, 1:8:2, 8:72]
    b = c.batch(news, max_length=LONG)
    p = L.SharedPrefix(ints(g.starts), ints(g.lengths), None, 500, 20)
    work = torch.empty(L.shared_attention_workspace(c.cache, b, p, 4), device="cuda", dtype=torch.uint8)
    outs = []
    for _ in range(3):
        out = torch.full((7, 4, 64), 5.0, device="cuda", dtype=BF16)
        L.cache_attention_shared_device(ctx, c.cache, b, p, q, out, work)
        outs.append(out)
    g.check(q, outs[0], news)
    before = big.clone()
    L.cache_attention_shared_device(ctx, c.cache, b, p, q, q, work)
    ctx.synchronize()
    assert torch.equal(q, outs[0]) and torch.equal(outs[1], outs[0]) and torch.equal(outs[2], outs[0])
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[:, 1:8:2, 8:72] = False
    assert torch.equal(big[mask], before[mask])


def test_few_sequences_run_by_themselves(ctx):
    """The rule's other side: no workspace, the plain attention's results."""
    g = Groups(14, [(37, [3, 2])], 16, 3, 64)
    c = g.c
    b, p = c.batch([1, 1], max_length=40), L.SharedPrefix(ints(g.starts), ints(g.lengths), None, 37, 3)
    assert L.shared_attention_workspace(c.cache, b, p, 3) == 0
    q = randn(gen(1), 2, 3, 64, dtype=BF16)
    out, plain = torch.empty_like(q), torch.empty_like(q)
    L.cache_attention_shared_device(ctx, c.cache, b, p, q, out)
    L.cache_attention_device(ctx, c.cache, b, q, plain)
    ctx.synchronize()
    assert torch.equal(out, plain)


def test_captured_calls_replay_on_new_lengths(ctx):
    g = Groups(15, [(400, [10, 20]), (90, [30])], 32, 2, 64)
    c, news = g.c, [1, 1, 1]
    q = randn(gen(4), 3, 2, 64, dtype=BF16)
    out = torch.empty_like(q)
    lengths, shared = ints([405, 402, 95]), ints([390, 80])
    b = L.CacheBatch(ints(c.table), ints([0, 1, 2, 3]), lengths, 3, 1, LONG)
    p = L.SharedPrefix(ints(g.starts), shared, 2, 400, 30)
    work = torch.empty(L.shared_attention_workspace(c.cache, b, p, 2), device="cuda", dtype=torch.uint8)
    L.cache_attention_shared_device(ctx, c.cache, b, p, q, out, work)
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        L.cache_attention_shared_device(ctx, c.cache, b, p, q, out, work)
    for ls, sh in (([405, 402, 95], [390, 80]), (c.lengths, g.lengths), ([401, 401, 91], [400, 0])):
        lengths.copy_(ints(ls))
        shared.copy_(ints(sh))
        work.fill_(0x7f)
        graph.replay()
        ctx.synchronize()
        kept, c.lengths = c.lengths, list(ls)
        g.check(q, out, news)
        c.lengths = kept
    del graph


@pytest.mark.parametrize("window", [0, 30])
def test_what_does_not_fit_is_skipped_and_reported(ctx, window):
    g = Groups(16, [(60, [9, 3]), (40, [2, 5])], 16, 1, 64)
    c, news = g.c, [1, 1, 1, 1]
    q = randn(gen(5), 4, 2, 64, dtype=BF16)
    reach = c.table.shape[1] * 16
    for groups, lengths, seq, message, bad in (
            ([0, 2, 4], [60, reach + 1], c.lengths, "group 1: ", [2, 3]),
            ([0, 2, 4], [-1, 40], c.lengths, "group 0: ", [0, 1]),
            ([0, 2, -4], [60, 40], c.lengths, "group 1: ", []),
            ([0, 2, 4], [60, 40], [69, 60, 42, 45], "sequence 1: new tokens reach into the shared prefix", [1]),
            ([0, 2, 4], [60, 40], [69, -1, 42, 45], "sequence 1: length -1", [1])):
        out = torch.full_like(q, 5.0)
        kept, c.lengths = c.lengths, list(seq)
        b = g.batch(news, 4, window)
        c.lengths = kept
        p = L.SharedPrefix(ints(groups), ints(lengths), 2, 60, 1)
        work = torch.zeros(L.shared_attention_workspace(c.cache, b, p, 2, window=window), device="cuda", dtype=torch.uint8)
        L.cache_attention_shared_device(ctx, c.cache, b, p, q, out, work, window=window)
        with pytest.raises(L.LwmError, match=message):
            ctx.synchronize()
        ctx.synchronize()
        assert (out[bad] == 5.0).all()
        for s in range(4):
            if s not in bad:
                parts = attention_64(q[s:s + 1].double(), c.dense("k", s), c.dense("v", s), mask_of(c.lengths[s], 1, True, window, 0, 1), 0.125)  # (the lengths of those are as they were)
                close(out[s:s + 1], parts[0], attention_tolerance(*parts, 64, BF16, False, 0.0) + parts[1] * 2.0 ** -15)
    # more rows than max_tokens
    out = torch.full_like(q, 5.0)
    p = L.SharedPrefix(ints([0, 2, 4]), ints([60, 40]), 1, 60, 9)
    b = c.batch(news, max_length=LONG)
    work = torch.zeros(L.shared_attention_workspace(c.cache, b, p, 2), device="cuda", dtype=torch.uint8)
    L.cache_attention_shared_device(ctx, c.cache, b, p, q, out, work)
    with pytest.raises(L.LwmError, match="group [01]: "):
        ctx.synchronize()
    assert (out == 5.0).all()
