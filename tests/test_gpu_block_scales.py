"""Attention over 8-bit caches whose pages have value scales far apart, as far
as an append writes them: the page that a row attends to keeps its precision
whatever the scales of the others, in both attention kernels, whether the
large page has no weight, a weight that its scale makes up for, or is not
seen at all.  The tolerance counts roundings relative to a row's own largest
weighted scale."""
import math

import pytest

import lewm_b200 as L
from test_gpu_blocks import (BF16, E32, F16, MANY, U, Paged, attention_64, close, gen, mask_of, on_context_stream,  # noqa: F401
                             randn, rounded)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def set_scales(c, s, exponents, frac=1.0):
    """Value scales 2^exponents[j] frac for page j of sequence s, codes as they are."""
    for j in range(-(-c.lengths[s] // c.page)):
        c.vs[int(c.table[s, j])] = 2.0 ** exponents[j % len(exponents)] * frac


def token_scales(c, s):
    """The value scale of each cached token, [length, kv] in 64 bits."""
    pages = torch.tensor(c.table[s, :-(-c.lengths[s] // c.page)], device="cuda", dtype=torch.int64)
    return c.vs[pages].double().repeat_interleave(c.page, 0)[:c.lengths[s]]


def tolerance(parts, q, k, vs, seen, scale, dtype):
    """Each weight (with its scale) is rounded to a half: 2^-11 of itself, and 2^-25 of the row's unit, which is at
    most twice its largest weighted scale; codes are at most 448.  Exponents: scores' products and sums, (d + 6)
    roundings, and 6 of differences as large as the scales' own spread; the exponential 2^-21.  Sums over the keys
    in 32 bits."""
    out, mass, reach, keys = parts
    d, group = q.shape[2], q.shape[1] // k.shape[1]
    spread = float(torch.log2(vs.max() / vs.min()))
    each = E32 * ((d + 6) * reach * 1.5 + 6 * (spread + 1)) + 2.0 ** -21
    score = torch.einsum("nhd,lhd->nhl", q, k.repeat_interleave(group, 1)) * scale
    w = torch.softmax(torch.where(seen[:, None], score, -math.inf), -1)
    w = torch.where(seen[:, None], w, 0.0) * vs.repeat_interleave(group, 1).T
    top = w.amax(-1, keepdim=True)
    return mass * (U(F16) + 2 * each + 2 * (keys + 16) * E32) + keys * 2.0 ** -24 * 448 * top + rounded(dtype, out)


def check(ctx, c, news, heads, seed, offsets, many=False, window=0, sinks=0, max_length=0):
    """Rows that weigh the keys by 2^(offset * k[0]), every row another offset."""
    g, tokens = gen(seed), MANY if many else sum(news)
    q = 0.3 * randn(g, tokens, heads, c.d)
    pick = torch.randint(0, len(offsets), (tokens, heads), generator=g, device="cuda")
    q[..., 0] = torch.tensor(offsets, device="cuda", dtype=torch.float32)[pick] * math.log(2) * c.d ** 0.5
    q = q.to(c.dtype)
    out = torch.full_like(q, 5.0)
    b = c.batch(news, tokens=tokens, max_length=max_length, **(dict(max_new=MANY) if many else {}))
    L.cache_attention_device(ctx, c.cache, b, q, out, window=window, sinks=sinks)
    t, scale = 0, c.d ** -0.5
    for s, n in enumerate(news):
        if n:
            seen, rows, k = mask_of(c.lengths[s], n, True, window, sinks, 1), q[t:t + n].double(), c.dense("k", s)
            parts = attention_64(rows, k, c.dense("v", s), seen, scale)
            close(out[t:t + n], parts[0], tolerance(parts, rows, k, token_scales(c, s), seen, scale, c.dtype))
        t += n
    return out


def filled(seed, lengths, page, kv, d, dtype, exponents, marked, frac=1.0):
    """Random codes; keys of the pages in `marked` (of the exponents' period) have -1 in channel 0, others 0."""
    c = Paged(seed, lengths, page, kv, d, dtype, True)
    g = gen(seed + 1)
    for s, n in enumerate(lengths):
        k = 0.2 * randn(g, n, kv, d)
        j = torch.arange(n, device="cuda") // page % len(exponents)
        k[..., 0] = -torch.isin(j, torch.tensor(marked, device="cuda")).float()[:, None]
        c.set("k", s, k)
        c.set("v", s, randn(g, n, kv, d))
        set_scales(c, s, exponents, frac)
    return c


# exponents of the pages' scales in turn, and the pages whose keys a row can weigh down
SPREADS = [([7, -13], [0]), ([-15, 7], [1]), ([-17, -17, 7], [2]), ([0, -10, -3, 5], [0, 3])]
FAR = [([40, -40], [0]), ([-100, 100], [1]), ([-120, 0, 119], [1, 2]), ([0, -90, -90, -90], [0]), ([-59, 2], [1])]


def offsets_of(exponents):
    """The large page as it is, made up for by its weight, and of no weight."""
    far = max(exponents) - min(exponents)
    return [0.0, far - 6.0, far + 3.0, far + 12.0, 2.0 * far + 20.0]


def check_far_apart(ctx, exponents, marked, dtype, d, news, many):
    c = filled(200, [130, 70, 300], 16, 2, d, dtype, exponents, marked, frac=1.0 if d == 64 else 1.37)
    for heads in (2, 6):
        check(ctx, c, news, heads, 201, offsets_of(exponents), many)


@pytest.mark.parametrize("exponents,marked,dtype", [(*x, t) for x in SPREADS for t in (BF16, F16)] +
                         [(*x, BF16) for x in FAR])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("news", [[1, 1, 1], [5, 0, 3]])
def test_scales_far_apart(ctx, exponents, marked, dtype, d, news):
    check_far_apart(ctx, exponents, marked, dtype, d, news, False)


@pytest.mark.parametrize("exponents,marked,dtype", [(*x, t) for x in SPREADS for t in (BF16, F16)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_scales_apart_on_many_rows(ctx, exponents, marked, dtype, d):
    check_far_apart(ctx, exponents, marked, dtype, d, [60, 1, 130], True)


@pytest.mark.parametrize("exponents,marked", FAR)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_scales_far_apart_on_many_rows(ctx, exponents, marked, d):
    """Pages more than 2^60 below the block's largest: their weights vanish from its products, not from its sums."""
    check_far_apart(ctx, exponents, marked, BF16, d, [60, 1, 130], True)


def check_outside_the_window(ctx, exponents, marked, many):
    """Rows of one tile, some of which see the large pages and some not: each row as if it were alone."""
    c = filled(203, [400, 333], 32, 1, 64, BF16, exponents, marked)
    for window, sinks in ((160, 0), (180, 3), (160, 40)) if many else ((20, 0), (40, 3), (33, 40), (1, 0)):
        check(ctx, c, [150, 90] if many else [12, 7], 2, 204, offsets_of(exponents), many, window, sinks)


@pytest.mark.parametrize("exponents,marked", [SPREADS[0], SPREADS[3], *FAR])
def test_large_scales_outside_the_window(ctx, exponents, marked):
    check_outside_the_window(ctx, exponents, marked, False)


@pytest.mark.parametrize("exponents,marked", [SPREADS[0], SPREADS[3]])
def test_large_scales_outside_the_window_on_many_rows(ctx, exponents, marked):
    check_outside_the_window(ctx, exponents, marked, True)


@pytest.mark.parametrize("exponents,marked", FAR)
def test_far_scales_outside_the_window_on_many_rows(ctx, exponents, marked):
    check_outside_the_window(ctx, exponents, marked, True)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_far_scales_come_and_go(ctx, d):
    """Large pages before, after and between small ones over several key tiles, rows that begin with either."""
    for exponents, marked in (([-100] * 5 + [60], [5]), ([60] + [-100] * 8, [0]), ([-110, -110, 0, 100], [2, 3]),
                              ([-120] * 9 + [119], [9])):
        c = filled(218, [700, 257], 64, 1, d, BF16, exponents, marked)
        check(ctx, c, [400, 257], 2, 219, offsets_of(exponents), True)
        check(ctx, c, [300, 130], 2, 220, offsets_of(exponents), True, window=150, sinks=30)


@pytest.mark.parametrize("exponents,marked", [SPREADS[1], FAR[0], FAR[2]])
@pytest.mark.parametrize("d,kv", [(64, 1), (128, 2)])
def test_scales_far_apart_in_long_contexts(ctx, exponents, marked, d, kv):
    """Warps and blocks of a cluster that hold parts of different scales are joined."""
    c = filled(206, [5000, 3000], 64, kv, d, BF16, exponents, marked)
    check(ctx, c, [1, 1], 4 * kv, 207, offsets_of(exponents))
    check(ctx, c, [3, 1], 4 * kv, 208, offsets_of(exponents), window=2000, sinks=100)
    # the large scale on one page alone, which no row weighs
    for s in range(2):
        set_scales(c, s, [-20])
        c.vs[int(c.table[s, 7])] = 2.0 ** 60
        c.k.view(torch.uint8)[int(c.table[s, 7]), ..., 0] = 0xb8  # -1
        c.ks[int(c.table[s, 7])] = 1.0
    check(ctx, c, [1, 1], 4 * kv, 209, [200.0])


def test_scales_far_apart_in_many_short_sequences(ctx):
    """A warp alone walks a short context."""
    lengths = [1 + (7 * i) % 60 for i in range(640)]
    for exponents, marked in (SPREADS[1], FAR[1]):
        c = filled(210, lengths, 16, 1, 64, BF16, exponents, marked)
        check(ctx, c, [1] * 640, 3, 211, offsets_of(exponents), max_length=60)


@pytest.mark.parametrize("many", [False, True])
def test_a_row_does_not_depend_on_scales_it_does_not_see(ctx, many):
    """The same rows over a window of small pages, with and without large pages before it: equal to one rounding."""
    n, large = (140, 100) if many else (3, 100)
    c = filled(212, [600], 32, 1, 64, BF16, [-30], [0])
    want = check(ctx, c, [n], 2, 213, [0.0], many, window=160 if many else 100)[:n].double()
    for j in range((600 - n - (160 if many else 100)) // 32):
        c.vs[int(c.table[0, j])] = 2.0 ** large
    got = check(ctx, c, [n], 2, 213, [0.0], many, window=160 if many else 100)[:n].double()
    # what one rounding of each side allows: the pages seen are the same, so are their scales
    assert ((got - want).abs() <= 2 * rounded(BF16, want)).all()


@pytest.mark.parametrize("exponents,marked", [([-127], [0]), ([-133], [0]), ([-140, -149], [0]), ([-128, -60], [1]),
                                              ([-149, 30], [1])])
@pytest.mark.parametrize("news,many", [([1, 5, 3], False), ([60, 1, 130], True)])
def test_scales_below_the_smallest_normal(ctx, exponents, marked, news, many):
    """Positive and finite is all that a scale has to be."""
    c = filled(221, [130, 70, 300], 16, 2, 64, BF16, exponents, marked)
    check(ctx, c, news, 6, 222, offsets_of(exponents), many)


@pytest.mark.parametrize("many", [False, True])
def test_zero_and_broken_scales(ctx, many):
    """A scale of zero is a page of zeros; of infinity or NaN, NaN for the rows that see it and for no other."""
    n, window = (200, 160) if many else (12, 5)
    c = filled(214, [512], 32, 1, 64, BF16, [0, -40], [0])
    p = [int(x) for x in c.table[0]]
    c.vs[p[15]] = 0.0
    check(ctx, c, [n], 2, 215, [0.0, 60.0], many, window=160 if many else 20)
    c.vs[p[15]] = 2.0 ** -40
    for bad in (float("inf"), float("nan")):
        c.vs[p[(512 - n) // 32]] = bad
        q = randn(gen(216), MANY if many else n, 2, 64, dtype=BF16)
        out = torch.empty_like(q)
        L.cache_attention_device(ctx, c.cache, c.batch([n], tokens=q.shape[0], max_new=q.shape[0]), q, out, window=window)
        index = torch.arange(512 - n, 512, device="cuda")
        j = (512 - n) // 32
        hit = (index >= 32 * j) & (index - window + 1 < 32 * (j + 1))
        assert torch.isnan(out[:n][hit]).all() and torch.isfinite(out[:n][~hit]).all()


@pytest.mark.parametrize("dtype,codes", [(F16, False), (BF16, True), (F16, True), (BF16, False)])
@pytest.mark.parametrize("length,n,power", [(50000, 1, 25.5), (50000, 1, 27.0), (700, 1, 24.5), (16000, 60, 25.2),
                                            (30000, 20, 26.0)])
def test_small_weights_add_up(ctx, dtype, codes, length, n, power):
    """One key outweighs each of the others by 2^power and has small values: the others, each less than the halves'
    last step beside it, still count.  Lost: 2^-29 of the largest weight for each key at most, beside the weights' own
    rounding."""
    many = n > 1
    c = Paged(223, [length], 64, 1, 64, dtype, codes)
    g = gen(224)
    k, v = torch.zeros(length, 1, 64, device="cuda"), randn(g, length, 1, 64).abs()
    k[..., 1], k[1, 0, 0], v[1] = 1.0, 1.0, 2.0 ** -6  # (channel 1, which no query has, gives each page a scale)
    c.set("k", 0, k)
    c.set("v", 0, v)
    if codes:
        c.vs[:] = 2.0 ** -7
    q = torch.zeros(MANY if many else n, 2, 64, device="cuda", dtype=dtype)
    keys, values = c.dense("k", 0), c.dense("v", 0)
    q[..., 0] = power * math.log(2) * 8 / float(keys[1, 0, 0])
    out = torch.empty_like(q)
    b = c.batch([n], tokens=q.shape[0], max_new=q.shape[0])
    L.cache_attention_device(ctx, c.cache, b, q, out)
    assert torch.isfinite(keys).all() and torch.isfinite(values).all()
    seen = mask_of(length, n, True, 0, 0, 1)
    want, mass, reach, count = attention_64(q[:n].double(), keys, values, seen, 0.125)
    each = E32 * 70 * reach * 1.5 + 2.0 ** -21
    top = 1 / (1 + length * 2.0 ** -power)
    tol = mass * (U(F16 if codes else dtype) + 2 * each + 2 * (count + 16) * E32) + rounded(dtype, want)
    close(out[:n], want, tol + count * 2.0 ** -29 * float(values.max()) * top)
