"""The transformer blocks against plain 64-bit implementations: rotary
positions, the paged cache (16 and 8 bits), its attention and the gated norms,
at the sizes, masks and layouts where they can go wrong, and all of them
together under a planner.

Tolerances count roundings.  u is half a step of the output's type (2^-8 bf16,
2^-11 fp16, 2^-24 f32); every product and sum in 32 bits costs 2^-24 of the
magnitudes that enter it."""
import itertools
import math

import numpy as np
import pytest

import lewm_b200 as L

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn
E32 = 2.0 ** -24


def U(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(dtype, out):
    """What rounding `out` to its type costs: half a step of the value, and of the subnormals (tiny eps apart)."""
    return U(dtype) * (out.abs() * 1.001 + torch.finfo(dtype).tiny)


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    """Torch works on the context's stream, as a callback scorer does."""
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


def close(got, want, tol):
    got = got.double()
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(got == want)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        t = tol if isinstance(tol, float) else float(tol.expand_as(want)[i])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {i}: {float(got[i])} for "
                             f"{float(want[i])}, tolerance {t}")


# ------------------------------------------------------------------- rotary

def turned(x, positions, dims, bases, interleaved, inverse=False):
    """(x turned, |x| of each pair) in 64 bits."""
    out, mag = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    off = 0
    for a, n in enumerate(dims):
        for i in range(n // 2):
            c0, c1 = (off + 2 * i, off + 2 * i + 1) if interleaved else (off + i, off + i + n // 2)
            angle = positions[:, a].double() * bases[a] ** (-2.0 * i / n) * (-1 if inverse else 1)
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            x0, x1 = x[..., c0].double(), x[..., c1].double()
            out[..., c0], out[..., c1] = x0 * c - x1 * s, x0 * s + x1 * c
            mag[..., c0] = mag[..., c1] = x0.abs() + x1.abs()
        off += n
    return out, mag


def turn_tolerance(out, mag, dtype, positions=None):
    # cosine and sine: the angle as a 24-bit fraction of a half turn (pi 2^-25) and sincospif (2 ulp), under
    # 2^-21 together; two products and a sum in 32 bits; the rounding of the output.  The reference's own angle
    # in 64 bits is off by |position| 2^-52.
    far = 0.0 if positions is None else float(positions.abs().max()) * 2.0 ** -51
    return mag * (2.0 ** -21 + 3 * E32 + far) + rounded(dtype, out)


ROTARY = [([64], 64, False), ([32, 32], 64, True), ([32, 16, 16], 64, False), ([16, 16], 40, False),
          ([8, 16, 8, 8], 48, True), ([64, 32, 32], 128, False), ([128], 256, False), ([16], 16, False)]


@pytest.mark.parametrize("dims,d,interleaved", ROTARY)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (7, 3), (400, 5)])
def test_rotary(ctx, dims, d, interleaved, dtype, tokens, heads):
    g = gen(1)
    bases = [10000.0, 100.0, 37.5, 2.0][: len(dims)]
    x = randn(g, tokens, heads, d, dtype=dtype)
    pos = torch.randint(-50, 5000, (tokens, len(dims)), generator=g, device="cuda", dtype=torch.int32)
    r = L.Rotary.make(dims, bases, interleaved)
    out = torch.full_like(x, float("nan"))
    L.rotary_device(ctx, r, x, out, pos)
    want, mag = turned(x, pos, dims, bases, interleaved)
    close(out, want, turn_tolerance(want, mag, dtype, pos))
    back = torch.empty_like(x)
    L.rotary_device(ctx, r, out, back, pos, inverse=True)
    want, mag = turned(out, pos, dims, bases, interleaved, inverse=True)
    close(back, want, turn_tolerance(want, mag, dtype, pos))


def test_rotary_far_positions_strides_and_in_place(ctx):
    g = gen(2)
    pos = ints([[2 ** 31 - 1], [-2 ** 31], [10 ** 9 + 7], [-1], [0]])
    r = L.Rotary.make([64], [10000.0])
    big = randn(g, 5, 9, 80, dtype=BF16)
    x = big[:, 1:8:2, 8:72]  # token stride 720, head stride 160
    before = big.clone()
    want, mag = turned(x, pos, [64], [10000.0], False)
    tol = turn_tolerance(want, mag, BF16, pos)
    heads_first = torch.empty(4, 5, 64, device="cuda", dtype=BF16).transpose(0, 1)
    L.rotary_device(ctx, r, x, heads_first, pos)
    close(heads_first, want, tol)
    L.rotary_device(ctx, r, x, x, pos)
    close(x, want, tol)
    before[:, 1:8:2, 8:72] = x
    assert torch.equal(big, before)


def test_rotary_inverse_is_the_gradient(ctx):
    g = gen(3)
    pos = torch.randint(0, 300, (6, 2), generator=g, device="cuda", dtype=torch.int32)
    r = L.Rotary.make([32, 32], [1e4, 1e2], True)
    x, up = randn(g, 6, 2, 64), randn(g, 6, 2, 64)
    grad = torch.empty_like(x)
    L.rotary_device(ctx, r, up, grad, pos, inverse=True)
    leaf = x.double().requires_grad_()
    with torch.enable_grad():
        (turned_graph(leaf, pos, [32, 32], [1e4, 1e2]) * up.double()).sum().backward()
    _, mag = turned(up, pos, [32, 32], [1e4, 1e2], True)
    close(grad, leaf.grad, turn_tolerance(leaf.grad, mag, F32, pos))
    # and against differences of the operator itself, which is linear
    step, out0, out1 = 0.25, torch.empty_like(x), torch.empty_like(x)
    for c in (0, 5, 63):
        moved = x.clone()
        moved[2, 1, c] += step
        L.rotary_device(ctx, r, x, out0, pos)
        L.rotary_device(ctx, r, moved, out1, pos)
        got = float(((out1.double() - out0.double()) * up.double()).sum()) / step
        bound = 64 * E32 * float((out0.abs() * up.abs()).sum()) / step + 2.0 ** -20 * float(mag[2, 1, c])
        assert abs(got - float(grad[2, 1, c])) <= bound


def turned_graph(x, positions, dims, bases):
    parts, off = [], 0
    for a, n in enumerate(dims):
        i = torch.arange(n // 2, device="cuda", dtype=torch.float64)
        t = positions[:, a].double()[:, None] * bases[a] ** (-2.0 * i / n)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        x0, x1 = x[..., off:off + n:2], x[..., off + 1:off + n:2]
        parts.append(torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], -1).flatten(-2))
        off += n
    return torch.cat(parts, -1)


# -------------------------------------------------------------- paged cache

class Paged:
    """A cache with random pages, and the same tokens kept dense."""

    def __init__(self, seed, lengths, page, kv, d, dtype=BF16, codes=False, fill=float("nan"), spare=3):
        rng = np.random.default_rng(seed)
        self.lengths, self.page, self.kv, self.d, self.dtype, self.codes = list(lengths), page, kv, d, dtype, codes
        per = max(1, max(-(-n // page) for n in lengths))
        n = len(lengths)
        pages = sum(-(-x // page) for x in lengths) + spare
        order = rng.permutation(pages)
        self.table = np.full((n, per), -1, np.int64)  # entries behind a sequence are not in the pool
        at = 0
        for s, length in enumerate(lengths):
            m = -(-length // page)
            self.table[s, :m] = order[at:at + m]
            at += m
        shape = (pages, kv, page, d)
        if codes:
            self.k = torch.full(shape, 0x7f, device="cuda", dtype=torch.uint8).view(F8)
            self.v = self.k.clone()
            self.ks = torch.full((pages, kv), fill, device="cuda")
            self.vs = torch.full((pages, kv), fill, device="cuda")
        else:
            self.k = torch.full(shape, fill, device="cuda", dtype=dtype)
            self.v = self.k.clone()
            self.ks = self.vs = None
        self.cache = L.PagedCache(self.k, self.v, self.ks, self.vs, dtype=dtype)

    def set(self, which, s, values):
        """Puts values [length, kv, d] into sequence s."""
        pool, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        for j in range(-(-len(values) // self.page)):
            part = values[j * self.page:(j + 1) * self.page].transpose(0, 1)  # [kv, tokens, d]
            p = int(self.table[s, j])
            if self.codes:
                sc = part.float().abs().amax((1, 2)) / 448 * (1 + 3 * torch.rand(self.kv, device="cuda"))
                scale[p] = sc
                pool.view(torch.uint8)[p, :, :part.shape[1]] = (part.float() / sc[:, None, None]).to(F8).view(torch.uint8)
            else:
                pool[p, :, :part.shape[1]] = part.to(self.dtype)

    def dense(self, which, s):
        """Sequence s as [length, kv, d] in 64 bits."""
        if self.lengths[s] == 0:
            return torch.zeros(0, self.kv, self.d, device="cuda", dtype=torch.float64)
        pool, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        rows = torch.tensor(self.table[s, :-(-self.lengths[s] // self.page)], device="cuda", dtype=torch.int64)
        x = (pool.view(torch.uint8)[rows].view(F8) if self.codes else pool[rows]).double()
        if self.codes:
            x = x * scale[rows].double()[:, :, None, None]
        return x.transpose(1, 2).reshape(-1, self.kv, self.d)[:self.lengths[s]]

    def fill_random(self, seed):
        torch.cuda.manual_seed(seed)  # the scales of set()
        g = gen(seed)
        for s, n in enumerate(self.lengths):
            for w in ("k", "v"):
                self.set(w, s, randn(g, n, self.kv, self.d))

    def batch(self, news, lengths=None, tokens=None, table=None, **kw):
        starts = np.concatenate([[0], np.cumsum(news)])
        t = int(starts[-1]) if tokens is None else tokens
        kw.setdefault("max_new", min(t, max(list(news) + [0])))
        return L.CacheBatch(ints(self.table if table is None else table), ints(starts),
                            ints(self.lengths if lengths is None else lengths), t, **kw)


def need_scale(amax):
    """The least power of two with amax <= 448 times it, as the header says."""
    if amax == 0:
        return 2.0 ** -120
    e = math.ceil(math.log2(amax / 448.0))
    while 448.0 * 2.0 ** (e - 1) >= amax:
        e -= 1
    while 448.0 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** max(-120, min(120, e))


@pytest.mark.parametrize("page,kv,d", [(16, 1, 32), (16, 3, 64), (32, 2, 128), (64, 4, 64), (128, 2, 32)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rotate", [None, "index", "axes"])
def test_append_16_bit_and_gather(ctx, page, kv, d, dtype, rotate):
    g = gen(4)
    lengths, news = [5, 1, 0, 40, page + 1, 2 * page, 133], [5, 1, 0, 7, page + 1, 1, 130]
    c = Paged(5, lengths, page, kv, d, dtype, fill=7.0)
    tokens, heads = sum(news) + 4, 2 * kv  # four packed rows behind the last sequence
    qkv = randn(g, tokens, heads + 2 * kv, d, dtype=dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    q_out = torch.full((heads, tokens, d), 9.0, device="cuda", dtype=dtype).transpose(0, 1)
    index = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, news)] + [np.zeros(4, int)])
    dims, bases = ([16, 16], [1e4, 50.0]) if rotate == "axes" else ([d], [1e4])
    pos = None
    if rotate == "axes":
        pos = torch.randint(-9, 3000, (tokens, 2), generator=g, device="cuda", dtype=torch.int32)
    r = None if rotate is None else L.Rotary.make(dims, bases, rotate == "axes")
    kpool, vpool = c.k.clone(), c.v.clone()
    b = c.batch(news, tokens=tokens)
    L.cache_append_device(ctx, c.cache, b, k, v, rotary=r, positions=pos, q=q, q_out=q_out)
    if rotate is None:
        wq, wk, tq, tk = q.double(), k.double(), 0.0, 0.0
    else:
        at = pos if pos is not None else ints(index)[:, None]
        wq, mq = turned(q, at, dims, bases, rotate == "axes")
        wk, mk = turned(k, at, dims, bases, rotate == "axes")
        tq, tk = turn_tolerance(wq, mq, dtype, at)[: sum(news)], turn_tolerance(wk, mk, dtype, at)
    close(q_out[: sum(news)], wq[: sum(news)], tq)
    assert (q_out[sum(news):] == 9.0).all()
    t = 0
    for s, (n, m) in enumerate(zip(lengths, news)):
        for i in range(n - m, n):
            p, slot = int(c.table[s, i // page]), i % page
            close(c.k[p, :, slot], wk[t], tk if rotate is None else tk[t])
            assert torch.equal(c.v[p, :, slot], v[t])
            kpool[p, :, slot], vpool[p, :, slot] = c.k[p, :, slot], v[t]
            t += 1
    assert torch.equal(c.k, kpool) and torch.equal(c.v, vpool)  # nothing else was touched
    ko = torch.full((tokens, kv, d), 9.0, device="cuda", dtype=dtype)
    vo = torch.full((kv, tokens, d), 9.0, device="cuda", dtype=dtype).transpose(0, 1)
    L.cache_gather_device(ctx, c.cache, b, ko, vo)
    assert torch.equal(vo[: sum(news)], v[: sum(news)]) and (ko[sum(news):] == 9.0).all() and (vo[sum(news):] == 9).all()
    for s, (n, m) in enumerate(zip(lengths, news)):
        o = sum(news[:s])
        assert torch.equal(ko[o:o + m].double(), c.dense("k", s)[n - m:])


def test_append_in_place_queries_and_none(ctx):
    g = gen(6)
    c = Paged(7, [3], 16, 2, 64, fill=0.0)
    q, k, v = randn(g, 3, 4, 64, dtype=BF16), randn(g, 3, 2, 64, dtype=BF16), randn(g, 3, 2, 64, dtype=BF16)
    want, mag = turned(q, ints([[0], [1], [2]]), [64], [1e4], False)
    r = L.Rotary.make([64], [1e4])
    L.cache_append_device(ctx, c.cache, c.batch([3]), k, v, rotary=r, q=q, q_out=q)
    close(q, want, turn_tolerance(want, mag, BF16))
    first = c.k.clone()
    c.k.zero_()
    L.cache_append_device(ctx, c.cache, c.batch([3]), k, v, rotary=r)
    assert torch.equal(first, c.k)


@pytest.mark.parametrize("page,kv,d", [(16, 2, 32), (16, 3, 64), (32, 1, 128), (128, 2, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_8_bit_step_by_step(ctx, page, kv, d, dtype):
    """Chunks of several sizes whose values grow and shrink, so that pages keep, raise and restart their scales."""
    rng, g = np.random.default_rng(8), gen(9)
    total = [3 * page + 5, 2 * page, 1]
    c = Paged(10, total, page, kv, d, dtype, codes=True, fill=2.0 ** 60)  # stale scales of a reused pool
    r = L.Rotary.make([d], [1e4])
    kept = {}  # (which, page) -> (scale [kv], codes as values / scale, [kv, slots, d])
    have = [0] * len(total)
    while have != total:
        news = [min(n - h, int(rng.choice([0, 1, 3, page // 2, page, 2 * page]))) for n, h in zip(total, have)]
        if not sum(news):
            continue
        lens = [h + m for h, m in zip(have, news)]
        size = float(np.exp2(rng.integers(-14, 7)))
        k, v = randn(g, sum(news), kv, d), randn(g, sum(news), kv, d)
        k, v = (k * size).to(dtype), (v * size * 3).to(dtype)
        v[0, 0, :] = 0
        index = np.concatenate([np.arange(h, h + m) for h, m in zip(have, news)])
        wk, mk = turned(k, ints(index)[:, None], [d], [1e4], False)
        L.cache_append_device(ctx, c.cache, c.batch(news, lengths=lens), k, v, rotary=r)
        ctx.synchronize()
        t = 0
        for s, (h, m) in enumerate(zip(have, news)):
            i = h
            while i < h + m:
                j, slot = i // page, i % page
                count = min(page - slot, h + m - i)
                p = int(c.table[s, j])
                for which, new, pool, scale in (("k", wk, c.k, c.ks), ("v", v.double(), c.v, c.vs)):
                    part = new[t:t + count].transpose(0, 1)  # [kv, count, d]
                    old = kept.get((which, p))
                    for hd in range(kv):
                        amax = float(part[hd].abs().max())
                        need = need_scale(amax)
                        got = float(scale[p, hd])
                        low = 0.0 if slot == 0 else float(old[0][hd])
                        want = max(need, low)
                        if got != want:  # keys are turned in 32 bits: next to a border either power is right
                            assert which == "k" and got == max(need_scale(amax * (1 + 2.0 ** -20)), low) or \
                                got == max(need_scale(amax * (1 - 2.0 ** -20)), low), (which, got, want, amax)
                        codes = pool[p, hd].double()
                        x = part[hd] / got
                        # half a step of e4m3: 2^-4 of the value, 2^-10 below its smallest normal; keys: a little more
                        tol = (x.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * 1.001 + (
                            mk[t:t + count, hd] / got * 2.0 ** -20 if which == "k" else 0.0)
                        close(codes[slot:slot + count], x, tol)
                        if slot:
                            before = old[1][hd, :slot] * (float(old[0][hd]) / got)
                            assert torch.equal(codes[:slot], before.float().to(F8).double())
                    kept[(which, p)] = (scale[p].clone(), pool[p].double().clone())
                t += count
                i += count
        have = lens


@pytest.mark.parametrize("page,kv,d", [(128, 2, 64), (64, 8, 32), (16, 3, 64), (32, 1, 128), (128, 2, 128)])
@pytest.mark.parametrize("news", [[300, 0, 65, 1], [1, 2, 0, 1], [96, 3], [95, 80], [81]])
def test_append_8_bit_turns_queries_too(ctx, page, kv, d, news):
    """q_out is what the rotary gives for the tokens' indexes, however the call deals out its heads; rows behind stay."""
    lens = [n + 7 for n in news]
    c = Paged(12, lens, page, kv, d, BF16, codes=True, fill=1.0)
    g, tokens, r = gen(13), sum(news) + 2, L.Rotary.make([d], [1e4])
    q, k, v = randn(g, tokens, 5, d), randn(g, tokens, kv, d), randn(g, tokens, kv, d)
    q, k, v = q.to(BF16), k.to(BF16), v.to(BF16)
    out, want = torch.full_like(q, 5.0), torch.empty_like(q)
    L.cache_append_device(ctx, c.cache, c.batch(news, lengths=lens, tokens=tokens, max_new=max(news)), k, v, rotary=r, q=q,
                          q_out=out)
    index = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, news)] + [np.zeros(2, int)])
    L.rotary_device(ctx, r, q, want, ints(index)[:, None].contiguous())
    ctx.synchronize()
    assert torch.equal(out[:-2], want[:-2]) and (out[-2:] == 5.0).all()


def test_append_8_bit_keeps_what_it_cannot_hold_visible(ctx):
    c = Paged(11, [3], 16, 1, 32, BF16, codes=True, fill=1.0)
    v = torch.ones(3, 1, 32, device="cuda", dtype=BF16) * 448
    v[0, 0, 3], v[1, 0, 4], v[2, 0, 5] = float("inf"), -float("inf"), float("nan")
    L.cache_append_device(ctx, c.cache, c.batch([3]), v, v)
    got = c.dense("v", 0)
    want = v.double()
    want[~torch.isfinite(want)] = float("nan")
    assert float(c.vs[c.table[0, 0], 0]) == 1.0  # infinities do not count
    close(got, want, 0.0)
    # a value just above 448 takes the next power; zeros the smallest
    v = torch.full((3, 1, 32), 450.0, device="cuda", dtype=BF16)
    L.cache_append_device(ctx, c.cache, c.batch([3]), torch.zeros_like(v), v)
    p = int(c.table[0, 0])
    assert float(c.vs[p, 0]) == 2.0 and float(c.ks[p, 0]) == 2.0 ** -120
    ko = torch.empty(3, 1, 32, device="cuda", dtype=BF16)
    vo = torch.empty_like(ko)
    L.cache_gather_device(ctx, c.cache, c.batch([3]), ko, vo)
    assert (ko == 0).all() and torch.equal(vo.double(), c.dense("v", 0))


# ---------------------------------------------------------------- attention

def mask_of(length, n, causal, window, sinks, frame):
    p = torch.arange(length - n, length, device="cuda")[:, None]
    j = torch.arange(length, device="cuda")[None]
    f = torch.div(p, frame, rounding_mode="floor")
    seen = (p >= 0) & (j < length)
    if causal:
        seen = seen & (j < (f + 1) * frame)
    if window:
        seen = seen & ((j >= (f + 1 - window) * frame) | (j < sinks))
    return seen


def attention_64(q, k, v, seen, scale):
    """(out, tolerance parts): q [n, H, d], k, v [L, kv, d] in 64 bits, seen [n, L].

    What is not seen is cut away before any arithmetic, not multiplied by zero."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(n, heads, d, device="cuda", dtype=torch.float64)
    mass, reach, keys = torch.zeros_like(out), torch.zeros(n, heads, 1, device="cuda", dtype=torch.float64), 0
    if k.shape[0] == 0:
        return out, mass, reach, keys
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    score = torch.einsum("nhd,lhd->nhl", q, kk) * scale
    score = torch.where(seen[:, None], score, -math.inf)
    w = torch.softmax(score, -1)
    w = torch.where(seen[:, None], w, 0.0)
    clean = torch.where(torch.isfinite(vv), vv, 0.0)
    out = torch.einsum("nhl,lhd->nhd", w, clean)
    mass = torch.einsum("nhl,lhd->nhd", w, clean.abs())
    for j in (~torch.isfinite(vv)).any(-1).any(-1).nonzero().flatten().tolist():
        rows = seen[:, j]
        out[rows] += w[rows, :, j, None] * torch.where(torch.isfinite(vv[j]), 0.0, vv[j])
    reach = (torch.einsum("nhd,lhd->nhl", q.abs(), kk.abs()) * abs(scale)).nan_to_num(0, 0, 0)
    reach = torch.where(seen[:, None], reach, 0.0).amax(-1, keepdim=True)
    return out, mass, reach, int(seen.sum(1).max())


def attention_tolerance(out, mass, reach, keys, d, dtype, codes, v_scale):
    # a weight: its score's products and sums, (d + 6) roundings of |q||k| scale (in powers of two: the same
    # relative error), the exponential 2^-21; weights are rounded to the operands' type (fp16 for codes); sums
    # over the keys in 32 bits.  Codes: weights times the value scales' ratio may be subnormal halves.
    p = U(F16 if codes else dtype)
    each = E32 * (d + 6) * reach * 1.5 + 2.0 ** -21
    tol = mass * (p + 2 * each + 2 * (keys + 16) * E32) + rounded(dtype, out)
    return tol + (keys * 2.0 ** -25 * 448 * v_scale if codes else 0.0)


# Packed rows (all but the first few behind the last sequence) and a bound on the new tokens of a sequence that
# make the tensor-core kernel the cheaper one by the library's costs: 20000 / 16 row tiles of the other kernel
# against 20000 / 256 blocks of its own.
MANY = 20000


def check_attention(ctx, c, news, heads, seed, causal=True, window=0, sinks=0, frame=1, scale=None, q=None,
                    table=None, lengths=None, many=False, **kw):
    g = gen(seed)
    lengths = c.lengths if lengths is None else lengths
    tokens = sum(news) + 3  # rows behind the last sequence
    if many:
        tokens = MANY
        kw["max_new"] = MANY
        if q is not None:
            q = torch.cat([q, q[:1].expand(MANY - q.shape[0], -1, -1)])
    q = randn(g, tokens, heads, c.d, dtype=c.dtype) if q is None else q
    out = torch.full((tokens, heads, c.d), 5.0, device="cuda", dtype=c.dtype)
    b = c.batch(news, lengths=lengths, tokens=tokens, table=table, **kw)
    L.cache_attention_device(ctx, c.cache, b, q, out, scale=scale, causal=causal, window=window, sinks=sinks,
                             frame_tokens=frame)
    t, scale = 0, c.d ** -0.5 if scale is None else scale
    for s, (length, n) in enumerate(zip(lengths, news)):
        if n:
            parts = attention_64(q[t:t + n].double(), c.dense("k", s), c.dense("v", s),
                                 mask_of(length, n, causal, window, sinks, frame), scale)
            vs = float(c.vs[c.table[s]].nan_to_num(0).max()) if c.codes else 0.0
            close(out[t:t + n], parts[0], attention_tolerance(*parts, c.d, c.dtype, c.codes, vs))
        t += n
    assert (out[t:] == 5.0).all()
    return out


POOLS = [(BF16, False), (F16, False), (BF16, True), (F16, True)]


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_single_tokens(ctx, dtype, codes, d, page):
    c = Paged(20, [1, 2, 15, 16, 17, 64, 100, 333, 1030], page, 2, d, dtype, codes)
    c.fill_random(21)
    for heads in (2, 6, 40):
        check_attention(ctx, c, [1] * 9, heads, heads)
    check_attention(ctx, c, [1, 0, 1, 0, 0, 1, 1, 0, 1], 6, 5)


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("window,sinks,frame", [(0, 0, 1), (1, 0, 1), (5, 0, 1), (16, 4, 1), (33, 130, 1), (200, 1, 1),
                                                (0, 0, 7), (2, 3, 7), (3, 20, 49), (1, 0, 197)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_masks(ctx, dtype, codes, d, window, sinks, frame, causal):
    lengths = [1, 31, 130, 260, 407, 90]
    c = Paged(22, lengths, 32, 2, d, dtype, codes)
    c.fill_random(23)
    check_attention(ctx, c, [1, 31, 17, 40, 1, 0], 6, 24, causal, window, sinks, frame)
    check_attention(ctx, c, [1, 31, 17, 100, 1, 0], 6, 24, causal, window, sinks, frame, many=True)


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("kv,heads", [(1, 1), (1, 3), (2, 8), (3, 3), (1, 16)])
def test_attention_many_rows(ctx, dtype, codes, d, kv, heads):
    """Whole histories and chunks behind a history, at lengths around the tiles' borders."""
    lengths = [127, 128, 129, 255, 257, 700, 1025, 383]
    c = Paged(25, lengths, 64, kv, d, dtype, codes)
    c.fill_random(26)
    for many in (False, True):
        check_attention(ctx, c, [127, 128, 129, 200, 257, 130, 300, 0], heads, 27, many=many)
        check_attention(ctx, c, [127, 128, 129, 200, 257, 130, 300, 64], heads, 28, window=150, sinks=20, many=many)
        check_attention(ctx, c, [1, 128, 0, 200, 257, 130, 300, 383], heads, 29, causal=False, many=many)


@pytest.mark.parametrize("page", [16, 32, 128])
def test_attention_many_rows_pages(ctx, page):
    for codes in (False, True):
        for d in (64, 128):
            c = Paged(30, [300, 511], page, 2, d, BF16, codes)
            c.fill_random(31)
            check_attention(ctx, c, [260, 140], 4, 32, many=True)


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d,sequences,kv", [(64, 1, 1), (128, 1, 2), (32, 2, 1), (128, 3, 4)])
def test_attention_long_contexts_are_split_and_joined(ctx, dtype, codes, d, sequences, kv):
    c = Paged(33, [5000 - 7 * i for i in range(sequences)], 64, kv, d, dtype, codes)
    c.fill_random(34)
    check_attention(ctx, c, [1] * sequences, 4 * kv, 35)
    check_attention(ctx, c, [3] * sequences, 4 * kv, 36, window=3000, sinks=4)
    check_attention(ctx, c, [1] * sequences, 4 * kv, 37, max_length=17)  # a hint that is wrong changes no result


def test_attention_many_short_sequences(ctx):
    rng = np.random.default_rng(38)
    lengths = rng.integers(1, 60, 700).tolist()
    for codes in (False, True):
        c = Paged(39, lengths, 16, 1, 64, BF16, codes)
        c.fill_random(40)
        check_attention(ctx, c, [1] * 700, 3, 41, max_length=60)
        check_attention(ctx, c, [min(2, n) for n in lengths], 2, 42, max_length=60, window=20, sinks=2)


def test_attention_rows_that_see_nothing(ctx):
    """More rows than cached tokens, and empty sequences: zeros."""
    for dtype, codes in POOLS:
        c = Paged(43, [0, 4, 20, 150], 16, 1, 64, dtype, codes)
        c.fill_random(44)
        for many in (False, True):
            out = check_attention(ctx, c, [3, 9, 1, 170], 2, 45, many=many)
            assert (out[:3] == 0).all() and (out[3:8] == 0).all() and (out[13:33] == 0).all()
            out = check_attention(ctx, c, [200, 9, 1, 170], 2, 46, causal=False, many=many)
            assert (out[:205] == 0).all()


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("many", [False, True])
def test_attention_is_not_reached_by_what_it_does_not_see(ctx, dtype, codes, d, many):
    """NaN and infinities in later tokens, behind the window, in unused slots; pages that nobody sees are not looked up."""
    n = 200 if many else 12
    length = 600
    c = Paged(47, [length, length], 32, 1, d, dtype, codes)
    c.fill_random(48)
    table = c.table.copy()
    table[0, 1:(length - n - 100) // 32] = 1 << 30  # behind the window of every row, not in any pool
    pool = c.v.view(torch.uint8) if codes else c.v
    for s, j in ((0, length - 5), (0, length - n), (1, length - n - 90), (1, length - n // 2), (1, 3)):
        pool[int(c.table[s, j // 32]), 0, j % 32, 1::3] = 0x7f if codes else float("inf")
        if not codes:
            pool[int(c.table[s, j // 32]), 0, j % 32, 2::3] = float("nan")
    kpool = c.k.view(torch.uint8) if codes else c.k
    kpool[int(c.table[1, (length - 3) // 32]), 0, (length - 3) % 32] = 0x7f if codes else float("nan")
    out = check_attention(ctx, c, [n, n], 2, 49, window=100, sinks=2, table=table, many=many)
    assert torch.isnan(out[:2 * n]).any() and torch.isfinite(out[:2 * n]).any()


def test_attention_extreme_scores(ctx):
    """Scores far apart in both orders, all equal, all hugely negative, scale zero and negative."""
    for codes in (False, True):
        for many in (1, 150):
            c = Paged(50, [400], 64, 1, 64, F16, codes)
            c.fill_random(51)
            g = gen(52)
            ramp = torch.linspace(-60, 60, 400, device="cuda")[:, None, None] * torch.ones(1, 1, 64, device="cuda") / 8
            for sign in (1, -1):
                c.set("k", 0, ramp * sign)
                q = torch.ones(many + 3, 2, 64, device="cuda", dtype=F16)
                q[:, 1] = -4
                check_attention(ctx, c, [many], 2, 53, q=q, many=many > 1)
            c.set("k", 0, torch.full((400, 1, 64), -30.0, device="cuda"))
            q = torch.full((many + 3, 2, 64), 30.0, device="cuda", dtype=F16)
            check_attention(ctx, c, [many], 2, 54, q=q, many=many > 1)
            c.set("k", 0, randn(g, 400, 1, 64))
            check_attention(ctx, c, [many], 2, 55, scale=0.0, many=many > 1)
            check_attention(ctx, c, [many], 2, 56, scale=-0.3, many=many > 1)


def test_attention_small_and_large_queries_on_codes(ctx):
    """bf16 queries far outside fp16's range, brought there by a power of two a row."""
    c = Paged(57, [100], 16, 1, 64, BF16, True)
    c.fill_random(58)
    g = gen(59)
    for size in (2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 100):
        for n in (1, 90):
            q = (randn(g, n + 3, 2, 64) * size).to(BF16)
            check_attention(ctx, c, [n], 2, 60, q=q, scale=0.125 / size, many=n > 1)


def test_attention_strides_and_in_place(ctx):
    g = gen(61)
    c = Paged(62, [150, 33], 16, 2, 64)
    c.fill_random(63)
    for news, t in (([1, 1], 2), ([140, 20], 160), ([140, 20], MANY)):
        wide = randn(g, 8, t + 2, 80, dtype=BF16)
        q = wide[1:7, 1:t + 1, 8:72].transpose(0, 1)  # [t, 6, 64], heads first
        want = torch.empty(t, 6, 64, device="cuda", dtype=BF16)
        b = c.batch(news, tokens=t, max_new=t)
        want.copy_(q)
        L.cache_attention_device(ctx, c.cache, b, q.contiguous(), want)
        before = wide.clone()
        L.cache_attention_device(ctx, c.cache, b, q, q)
        assert torch.equal(q, want)
        before[1:7, 1:t + 1, 8:72] = q.transpose(0, 1)
        assert torch.equal(wide, before)


def test_attention_shared_pages_and_repeated_calls_agree(ctx):
    c = Paged(64, [96, 96, 96], 32, 2, 64)
    c.fill_random(65)
    c.table[1, :2] = c.table[0, :2]
    c.table[2] = c.table[0]
    q = randn(gen(66), 6, 4, 64, dtype=BF16)
    q[4:6] = q[0:2]
    out = check_attention(ctx, c, [2, 2, 2], 4, 67, q=torch.cat([q, q[:3]]))
    assert torch.equal(out[:2], out[4:6])
    again = check_attention(ctx, c, [2, 2, 2], 4, 67, q=torch.cat([q, q[:3]]))
    assert torch.equal(out, again)
    out = check_attention(ctx, c, [2, 2, 2], 4, 67, q=torch.cat([q, q[:3]]), many=True)
    again = check_attention(ctx, c, [2, 2, 2], 4, 67, q=torch.cat([q, q[:3]]), many=True)
    assert torch.equal(out[:2], out[4:6]) and torch.equal(out, again)


def test_cache_offsets_beyond_32_bits(ctx):
    """A pool of more than 2^32 bytes and 2^31 elements: the last pages."""
    pages, kv, page, d = 16400, 8, 128, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of device memory")
    k = torch.empty(pages, kv, page, d, device="cuda", dtype=BF16)
    v = torch.empty_like(k)
    cache = L.PagedCache(k, v)
    g = gen(68)
    x = randn(g, 300, kv, d, dtype=BF16)
    y = randn(g, 300, kv, d, dtype=BF16)
    table = ints([[pages - 1, 5, pages - 2]])
    b = L.CacheBatch(table, ints([0, 300]), ints([300]), 300)
    L.cache_append_device(ctx, cache, b, x, y)
    ko, vo = torch.empty_like(x), torch.empty_like(y)
    L.cache_gather_device(ctx, cache, b, ko, vo)
    assert torch.equal(ko, x) and torch.equal(vo, y)
    for n, t in ((1, 1), (300, MANY)):
        q = randn(g, t, kv, d, dtype=BF16)
        out = torch.empty_like(q)
        L.cache_attention_device(ctx, cache, L.CacheBatch(table, ints([0, n]), ints([300]), t, max_new=t), q, out)
        q, out = q[:n], out[:n]
        parts = attention_64(q.double(), x.double(), y.double(), mask_of(300, n, True, 0, 0, 1), d ** -0.5)
        close(out, parts[0], attention_tolerance(*parts, d, BF16, False, 0.0))


# ------------------------------------------------------------ bad batches

@pytest.mark.parametrize("many", [False, True])
def test_bad_batches_are_skipped_and_reported(ctx, many):
    n = 140 if many else 2
    c = Paged(70, [200, 200, 200], 64, 1, 64, fill=0.0)
    c.fill_random(71)
    g = gen(72)
    tokens = MANY if many else 3 * n
    q = randn(g, tokens, 2, 64, dtype=BF16)
    kv = randn(g, tokens, 1, 64, dtype=BF16)
    good = torch.empty_like(q)
    L.cache_attention_device(ctx, c.cache, c.batch([n] * 3, tokens=tokens, max_new=MANY if many else n), q, good)
    ctx.synchronize()

    def broken(what):
        table, starts, lengths = c.table.copy(), [0, n, 2 * n, 3 * n], [200, 200, 200]
        max_new = MANY if many else n
        if what == "page":
            table[1, 3] = c.k.shape[0]
        elif what == "negative page":
            table[1, 3] = -7
        elif what == "starts":
            starts = [0, n, n - 1, n - 1]
        elif what == "rows":
            starts = [0, n, tokens + 1, tokens + 1]
        elif what == "length":
            lengths[1] = 4 * 64 + 1
        elif what == "negative length":
            lengths[1] = -1
        elif what == "new":
            starts, max_new = [0, n - 1, 2 * n, 3 * n], n
            if many:  # its longest sequence alone; the kernel that looks is the same
                starts, max_new = [0, 0, MANY, MANY], MANY - 1
        return L.CacheBatch(ints(table), ints(starts), ints(lengths), tokens, max_new=max_new)

    for what, message in (("page", "not in the pool"), ("negative page", "not in the pool"),
                          ("starts", "out of order"), ("rows", "beyond the packed rows"),
                          ("length", "beyond its page table"), ("negative length", "negative"),
                          ("new", "more new tokens")):
        out = torch.full_like(q, 3.0)
        L.cache_attention_device(ctx, c.cache, broken(what), q, out)
        with pytest.raises(L.LwmError, match=message) as e:
            ctx.synchronize()
        assert e.value.status == "INVALID_ARGUMENT"
        ctx.synchronize()  # reported once
        if what not in ("new", "rows"):
            assert torch.equal(out[:n], good[:n]), what
        if what not in ("page", "negative page"):  # a skipped sequence's rows are zero or as they were
            rest = out[n:2 * n] if what != "new" else out[max(n - 1, 0):2 * n]
            assert ((rest == 3.0) | (rest == 0.0)).all() or what == "new", what
        before_k, before_v = c.k.clone(), c.v.clone()
        L.cache_append_device(ctx, c.cache, broken(what), kv, kv)
        with pytest.raises(L.LwmError, match=message):
            ctx.synchronize()
        if what not in ("page", "negative page"):  # nothing of the bad sequence was written
            rows = torch.tensor(c.table[1], device="cuda")
            assert torch.equal(c.k[rows], before_k[rows])
        c.k.copy_(before_k)
        c.v.copy_(before_v)


def test_appending_more_than_the_length_is_reported(ctx):
    c = Paged(73, [4], 16, 1, 32, fill=0.0)
    x = torch.ones(6, 1, 32, device="cuda", dtype=BF16)
    L.cache_append_device(ctx, c.cache, c.batch([6]), x, x)
    with pytest.raises(L.LwmError, match="more new tokens"):
        ctx.synchronize()
    assert (c.k == 0).all()


def test_wrong_tensors_are_refused(ctx):
    c = Paged(74, [20], 16, 2, 64)
    b = c.batch([2])
    q = torch.zeros(2, 4, 64, device="cuda", dtype=BF16)
    kv = torch.zeros(2, 2, 64, device="cuda", dtype=BF16)
    L.cache_attention_device(ctx, c.cache, b, q, torch.empty_like(q), window=1)
    for call, message in (
            (lambda: L.cache_attention_device(ctx, c.cache, b, q.half(), q), "q must be torch.bfloat16"),
            (lambda: L.cache_attention_device(ctx, c.cache, b, q[:1], q), "q must be"),
            (lambda: L.cache_attention_device(ctx, c.cache, b, q[:, :3], q[:, :3]), "multiple of kv_heads"),
            (lambda: L.cache_attention_device(ctx, c.cache, b, q.cpu(), q), "must be on cuda"),
            (lambda: L.cache_attention_device(ctx, c.cache, b, q, q.transpose(1, 2)), "out must be"),
            (lambda: L.cache_append_device(ctx, c.cache, b, kv, kv[:, :1]), "v must be"),
            (lambda: L.cache_append_device(ctx, c.cache, b, kv, kv, positions=ints([[1], [2]])), "need a rotary"),
            (lambda: L.cache_append_device(ctx, c.cache, b, kv, kv, q=q), "needs q_out"),
            (lambda: L.rotary_device(ctx, L.Rotary.make([32], [1e4]), q, q, ints([1, 2])), "positions must be"),
            (lambda: L.gated_norm_device(ctx, L.GatedNorm(), q[0], h=q[0], gate=torch.zeros(3, 64, device="cuda")),
             "gate must be"),
            (lambda: L.gated_norm_device(ctx, L.GatedNorm(), q[0], h=q[0], gate=torch.zeros(64, device="cuda")),
             "gate must be"),
            (lambda: L.gated_norm_device(ctx, L.GatedNorm(), q[0], h=q), "h must be"),
            (lambda: L.cache_attention_device(ctx, c.cache, b, q, q, window=-1), "window must be 0 to"),
            (lambda: L.cache_attention_device(ctx, c.cache, b, q, q, sinks=1 << 32), "sinks must be 0 to")):
        with pytest.raises(L.LwmError, match=message):
            call()


def test_empty_batches(ctx):
    """No rows, no sequences, sequences without new tokens: nothing runs, nothing is reported."""
    c = Paged(75, [20, 0], 16, 2, 64)
    q, kv = torch.zeros(0, 4, 64, device="cuda", dtype=BF16), torch.zeros(0, 2, 64, device="cuda", dtype=BF16)
    none = L.CacheBatch(torch.zeros(0, 2, device="cuda", dtype=torch.int32), ints([0]), ints([]), 0)
    for b in (c.batch([0, 0]), none):
        L.cache_append_device(ctx, c.cache, b, kv, kv, L.Rotary.make([64], [1e4]), q=q, q_out=q)
        L.cache_attention_device(ctx, c.cache, b, q, q)
        L.cache_gather_device(ctx, c.cache, b, kv, kv)
    L.rotary_device(ctx, L.Rotary.make([64], [1e4]), q, q, torch.zeros(0, 1, device="cuda", dtype=torch.int32))
    x = torch.zeros(0, 64, device="cuda", dtype=BF16)
    L.gated_norm_device(ctx, L.GatedNorm(), x, y=x, x_out=x, h=x, gate=x)
    ctx.synchronize()


# --------------------------------------------------------------- gated norm

def norm_64(x, kind, w, b, eps, mag):
    """(normed, magnitude that a rounding of 2^-24 is relative to)"""
    if kind == "none":
        return x, mag
    m = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
    d = (((x - m) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    out = (x - m) / d
    # errors of the row's values and of its statistics, all over the deviation
    mag = (mag.amax(-1, keepdim=True) / d).expand_as(x) * (1 + out.abs())
    if w is not None:
        out, mag = out * w, mag * w.abs()
    if b is not None:
        out, mag = out + b, mag + b.abs()
    return out, mag


def gated_64(x, y, o, gate, shift, scale, per):
    def cond(t):
        return t.double().repeat_interleave(per, 0)[:x.shape[0]]

    def wt(n):
        return None if o.get(n) is None else o[n].double()

    x, mag = x.double(), x.double().abs()
    if y is not None:
        y, my = norm_64(y.double(), o.get("post", "none"), wt("post_weight"), wt("post_bias"), 1e-6, y.double().abs())
        for f in (wt("residual_scale"), None if gate is None else cond(gate)):
            if f is not None:
                y, my = y * f, my * f.abs()
        x, mag = x + y, mag + my
    h, mh = norm_64(x, o.get("pre", "layer"), wt("pre_weight"), wt("pre_bias"), 1e-6, mag)
    if scale is not None:
        h, mh = h * (1 + cond(scale)), mh * (1 + cond(scale).abs())
    if shift is not None:
        h, mh = h + cond(shift), mh + cond(shift).abs()
    if o.get("out_weight") is not None:
        h, mh = norm_64(h, "layer", wt("out_weight"), wt("out_bias"), 1e-5, mh)
    return x, mag, h, mh


# sums over a row: 32 values a thread, 5 shuffles, 8 warps, and a few operations a value: under 64 roundings a norm
NORM_ROUNDINGS = 64


def check_norm(ctx, rows, width, x_dtype, dtype, cond_dtype=F32, per=1, gate=True, modulate=True, seed=0, pad=0, **o):
    g = gen(seed + 80)
    x = (2 * randn(g, rows, width + pad) + randn(g, width + pad)).to(x_dtype)[:, :width]
    y = randn(g, rows, width + pad, dtype=dtype)[:, :width]
    conds = -(-rows // per)
    table = (0.5 * randn(g, conds, 3 * width)).to(cond_dtype)
    ga = table[:, :width] if gate else None
    sh, sc = (table[:, width:2 * width], table[:, 2 * width:]) if modulate else (None, None)
    for n in list(o):
        if o[n] is True:
            o[n] = (randn(g, width) * 0.2 + (1.0 if n.endswith("weight") else 0.3))
    norm = L.GatedNorm(**o)
    x_out = torch.full((rows, width + pad), 7.0, device="cuda", dtype=x_dtype)[:, :width]
    h = torch.full((rows, width + pad), 7.0, device="cuda", dtype=dtype)[:, :width]
    L.gated_norm_device(ctx, norm, x, y, x_out, h, gate=ga, shift=sh, scale=sc, rows_per_cond=per)
    wx, mx, wh, mh = gated_64(x, y, o, ga, sh, sc, per)
    close(x_out, wx, NORM_ROUNDINGS * E32 * mx + rounded(x_dtype, wx))
    close(h, wh, 2 * NORM_ROUNDINGS * E32 * mh + rounded(dtype, wh))
    if pad:
        assert (x_out.as_strided((rows, pad), (width + pad, 1), width) == 7.0).all()
    return norm, x, y, x_out, h, ga, sh, sc


@pytest.mark.parametrize("width", [1, 7, 8, 64, 192, 193, 264, 768, 1000, 1024, 1032, 2048, 4096, 4100, 8192])
@pytest.mark.parametrize("x_dtype,dtype,cond_dtype", [(F32, F32, F32), (F32, BF16, BF16), (BF16, BF16, F32),
                                                      (F16, F16, F16)])
def test_gated_norm_widths_and_types(ctx, width, x_dtype, dtype, cond_dtype):
    check_norm(ctx, 5, width, x_dtype, dtype, cond_dtype, post="rms", pre="layer", post_weight=True, pre_weight=True,
               pre_bias=True, residual_scale=True, seed=width)


@pytest.mark.parametrize("post,pre", list(itertools.product(["none", "layer", "rms"], repeat=2)))
@pytest.mark.parametrize("gate,modulate,out", [(True, True, True), (False, True, False), (True, False, False),
                                               (False, False, True)])
def test_gated_norm_kinds(ctx, post, pre, gate, modulate, out):
    for width, pad in ((192, 0), (200, 3)):
        check_norm(ctx, 37, width, F32, F32, F32, 4, gate, modulate, pad=pad, post=post, pre=pre, post_weight=True,
                   post_bias=post == "layer" or None, pre_weight=True, pre_bias=True,
                   **(dict(out_weight=True, out_bias=True) if out else {}))


@pytest.mark.parametrize("rows,per", [(1, 1), (3, 2), (129, 197), (1000, 7), (4097, 1)])
def test_gated_norm_rows(ctx, rows, per):
    check_norm(ctx, rows, 192, F32, BF16, BF16, per, pre="layer", pre_weight=True)


def test_gated_norm_in_place_and_parts(ctx):
    norm, x, y, x_out, h, ga, sh, sc = check_norm(ctx, 33, 384, BF16, BF16, pre="rms", pre_weight=True)
    # in place: the residual stream, and h over y
    x2, y2 = x.clone(), y.clone()
    L.gated_norm_device(ctx, norm, x2, y2, x2, y2, gate=ga, shift=sh, scale=sc)
    assert torch.equal(x2, x_out) and torch.equal(y2, h)
    # only the residual, only the norm, no block output
    only = torch.empty_like(x)
    L.gated_norm_device(ctx, norm, x, y, x_out=only, gate=ga)
    assert torch.equal(only, x_out)
    L.gated_norm_device(ctx, norm, x, y, h=only, gate=ga, shift=sh, scale=sc)
    assert torch.equal(only, h)
    L.gated_norm_device(ctx, norm, x, h=only, shift=sh, scale=sc)
    _, _, want, mag = gated_64(x, None, dict(pre="rms", pre_weight=norm._keep["pre_weight"]), None, sh, sc, 1)
    close(only, want, 2 * NORM_ROUNDINGS * E32 * mag + rounded(BF16, want))


def test_gated_norm_is_the_predictors_block(ctx):
    """AdaLN of the LeWM predictor (LayerNorm 1e-6, modulate, LayerNorm 1e-5 with weights) on a constant and a
    large-offset row: the mean is taken out before the squares."""
    width = 192
    x = torch.zeros(3, width, device="cuda")
    x[0] = 5.0
    x[1] = 1000.0 + torch.linspace(-1, 1, width, device="cuda")
    x[2] = torch.linspace(-1e-3, 1e-3, width, device="cuda")
    g = gen(90)
    o = dict(pre="layer", out_weight=1 + 0.1 * randn(g, width), out_bias=0.1 * randn(g, width))
    sh, sc = randn(g, 3, width), 0.1 * randn(g, 3, width)
    h = torch.empty_like(x)
    L.gated_norm_device(ctx, L.GatedNorm(**o), x, h=h, shift=sh, scale=sc)
    _, _, want, mag = gated_64(x, None, o, None, sh, sc, 1)
    close(h, want, 2 * NORM_ROUNDINGS * E32 * mag)


# ------------------------------------------------------------ graphs, streams

def test_captured_step_replays_on_new_lengths(ctx):
    """append + attention of one token captured once; each replay reads the lengths, tables and inputs of its time."""
    for codes in (False, True):
        c = Paged(91, [40, 70], 16, 2, 64, BF16, codes, fill=1.0)
        c.table[c.table < 0] = 0
        c.fill_random(92)
        g = gen(93)
        qkv = randn(g, 2, 8, 64, dtype=BF16)
        out, q = torch.zeros(2, 4, 64, device="cuda", dtype=BF16), torch.zeros(2, 4, 64, device="cuda", dtype=BF16)
        lengths = ints([30, 60])
        b = L.CacheBatch(ints(c.table), ints([0, 1, 2]), lengths, 2, max_new=1)
        r = L.Rotary.make([64], [1e4])

        def step():
            L.cache_append_device(ctx, c.cache, b, qkv[:, 4:6], qkv[:, 6:], rotary=r, q=qkv[:, :4], q_out=q)
            L.cache_attention_device(ctx, c.cache, b, q, out, window=25, sinks=3)

        stream = ctx.torch_stream()
        graph = torch.cuda.CUDAGraph()
        ctx.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(4):
            qkv.copy_(randn(g, 2, 8, 64, dtype=BF16))
            lengths.copy_(ints([31 + i, 61 + i]))
            pools = [t.clone() for t in (c.k, c.v, c.ks, c.vs) if t is not None]
            graph.replay()
            got, got_q = out.clone(), q.clone()
            for t, p in zip((c.k, c.v, c.ks, c.vs), pools):
                t.view(torch.uint8).copy_(p.view(torch.uint8))
            step()
            assert torch.equal(got, out) and torch.equal(got_q, q)
            c.lengths = [31 + i, 61 + i]
            for s in range(2):
                parts = attention_64(q[s:s + 1].double(), c.dense("k", s), c.dense("v", s),
                                     mask_of(c.lengths[s], 1, True, 25, 3, 1), 0.125)
                vs = float(c.vs.max()) if codes else 0.0
                close(out[s:s + 1], parts[0], attention_tolerance(*parts, 64, BF16, codes, vs))


def test_captured_chunk_replays_on_new_lengths(ctx):
    """A chunk of tokens on the tensor-core kernel, captured once."""
    for codes in (False, True):
        c = Paged(97, [300, 200], 64, 2, 128, BF16, codes)
        c.fill_random(98)
        q = randn(gen(99), MANY, 4, 128, dtype=BF16)
        out = torch.zeros_like(q)
        lengths = ints([300, 200])
        b = L.CacheBatch(ints(c.table), ints([0, 130, 200]), lengths, MANY, max_new=MANY)
        ctx.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=ctx.torch_stream()):
            L.cache_attention_device(ctx, c.cache, b, q, out, window=64, sinks=3)
        for lens in ([300, 200], [131, 190], [260, 71]):
            lengths.copy_(ints(lens))
            graph.replay()
            got = out.clone()
            L.cache_attention_device(ctx, c.cache, b, q, out, window=64, sinks=3)
            assert torch.equal(got, out)
            c.lengths = lens
            for s, (a, z) in enumerate(((0, 130), (130, 200))):
                parts = attention_64(q[a:z].double(), c.dense("k", s), c.dense("v", s),
                                     mask_of(lens[s], z - a, True, 64, 3, 1), 128 ** -0.5)
                vs = float(c.vs[c.table[s]].nan_to_num(0).max()) if codes else 0.0
                close(out[a:z], parts[0], attention_tolerance(*parts, 128, BF16, codes, vs))


def test_two_contexts_at_once(ctx):
    """Two contexts' streams run the same calls side by side on shared pages."""
    import threading
    other = L.Context(0)
    try:
        c = Paged(94, [3000, 200], 64, 2, 128)
        c.fill_random(95)
        q = randn(gen(96), MANY, 4, 128, dtype=BF16)
        torch.cuda.synchronize()
        results = {}

        def work(name, cx):
            with torch.cuda.stream(cx.torch_stream()):
                for i in range(20):
                    for news, t in (([1, 1], 2), ([2, 140], 142), ([20, 1], MANY)):
                        out = torch.zeros(t, 4, 128, device="cuda", dtype=BF16)
                        b = c.batch(news, tokens=t, max_new=max(news) if t < MANY else t)
                        L.cache_attention_device(cx, c.cache, b, q[:t], out)
                        results[name, i, t] = out
                cx.synchronize()

        threads = [threading.Thread(target=work, args=(n, x)) for n, x in (("a", ctx), ("b", other))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for (name, i, n), out in results.items():
            assert torch.equal(out, results["a", 0, n])
    finally:
        other.close()


# ------------------------------------------------- together, under a planner

class WorldModel:
    """A two-layer AdaLN transformer over a vehicle's frames and actions: every
    candidate shares the history's pages and appends its own steps.  `plain`
    computes the same rollout in 64 bits, without a cache."""

    D, HEADS, KV, DIM, LAYERS, PAGE = 192, 6, 2, 64, 2, 16

    def __init__(self, seed):
        g = gen(seed)
        d, h, kv, w = self.D, self.HEADS, self.KV, self.DIM
        self.layers = []
        for _ in range(self.LAYERS):
            self.layers.append(dict(
                qkv=randn(g, d, (h + 2 * kv) * w, dtype=BF16) / d ** 0.5, out=randn(g, h * w, d, dtype=BF16) / 20,
                ada=0.3 * randn(g, 2, 3 * d), pre=1 + 0.1 * randn(g, d), post=1 + 0.1 * randn(g, d)))
        self.embed = randn(g, 2, d)
        self.dims, self.bases = [32, 32], [1e4, 1e2]

    def positions(self, steps, rows):
        return ints([[t, t % 3] for t in steps]).repeat(rows, 1) if rows else ints([[t, t % 3] for t in steps])

    def plain(self, x, actions, pos, windows):
        """x [T, D] one sequence in 64 bits -> [T, D]."""
        d, h, kv, w = self.D, self.HEADS, self.KV, self.DIM
        T = x.shape[0]
        for ly in self.layers:
            ada = actions @ ly["ada"].double()
            u, _ = norm_64(x, "layer", ly["pre"].double(), None, 1e-6, x.abs())
            u = u * (1 + ada[:, 2 * d:]) + ada[:, d:2 * d]
            y = (u @ ly["qkv"].double()).view(T, h + 2 * kv, w)
            q, _ = turned(y[:, :h], pos, self.dims, self.bases, False)
            k, _ = turned(y[:, h:h + kv], pos, self.dims, self.bases, False)
            o = attention_64(q, k, y[:, h + kv:], mask_of(T, T, True, *windows), w ** -0.5)[0]
            o = o.reshape(T, h * w) @ ly["out"].double()
            o, _ = norm_64(o, "rms", ly["post"].double(), None, 1e-6, o.abs())
            x = x + ada[:, :d] * o
        return x


@pytest.mark.parametrize("codes", [False, True])
def test_candidate_rollouts_under_a_planner(ctx, codes):
    """MPPI over a CallbackScorer whose model runs on the blocks; its scores against the plain model's."""
    m = WorldModel(100)
    B, S, T, A, H = 2, 24, 3, 2, 21  # vehicles, candidates, horizon, action dims, history
    d, h, kv, w, page = m.D, m.HEADS, m.KV, m.DIM, m.PAGE
    g = gen(101)
    history, past = randn(g, B, H, d), randn(g, B, H, A)
    goal = randn(g, B, d)
    windows = (16, 2, 1)
    full = H // page  # whole pages of history, shared; a candidate copies the rest
    per = -(-(H + T) // page)
    n = B * S
    pages = B * per + n * (per - full)
    pools = []
    for _ in range(m.LAYERS):
        shape = (pages, kv, page, w)
        if codes:
            k = torch.zeros(shape, device="cuda").to(F8)
            args = (k, k.clone(), torch.ones(pages, kv, device="cuda"), torch.ones(pages, kv, device="cuda"))
        else:
            k = torch.zeros(shape, device="cuda", dtype=BF16)
            args = (k, k.clone(), None, None)
        pools.append((args, L.PagedCache(*args, dtype=BF16)))
    own = np.arange(B * per).reshape(B, per)
    table = np.zeros((n, per), np.int32)
    table[:, :full] = np.repeat(own[:, :full], S, 0)
    table[:, full:] = B * per + np.arange(n * (per - full)).reshape(n, -1)
    rotary = L.Rotary.make(m.dims, m.bases)

    def forward(x, actions, pos, batch):
        """x [rows, D] f32 in place through the layers."""
        rows = x.shape[0]
        u = torch.empty(rows, d, device="cuda", dtype=BF16)
        out = None
        for i, ly in enumerate(m.layers):
            ada = actions @ ly["ada"]
            if i == 0:
                L.gated_norm_device(ctx, L.GatedNorm(pre="layer", pre_weight=ly["pre"]), x, h=u,
                                    shift=ada[:, d:2 * d], scale=ada[:, 2 * d:])
            qkv = (u @ ly["qkv"]).view(rows, h + 2 * kv, w)
            q, out = qkv[:, :h], torch.empty(rows, h, w, device="cuda", dtype=BF16)
            L.cache_append_device(ctx, pools[i][1], batch, qkv[:, h:h + kv], qkv[:, h + kv:], rotary=rotary,
                                  positions=pos, q=q, q_out=q)
            L.cache_attention_device(ctx, pools[i][1], batch, q, out, window=windows[0], sinks=windows[1])
            y = out.view(rows, h * w) @ ly["out"]
            if i + 1 < m.LAYERS:
                nxt = m.layers[i + 1]
                a2 = actions @ nxt["ada"]
                # gate of this layer, modulation of the next: one table
                both = torch.cat([ada[:, :d], a2[:, d:]], 1)
                L.gated_norm_device(ctx, L.GatedNorm(post="rms", post_weight=ly["post"], pre="layer",
                                                     pre_weight=nxt["pre"]), x, y, x, u, gate=both[:, :d],
                                    shift=both[:, d:2 * d], scale=both[:, 2 * d:])
            else:
                L.gated_norm_device(ctx, L.GatedNorm(post="rms", post_weight=ly["post"]), x, y, x, gate=ada[:, :d])
        return x

    def score(cands):
        # the history of every vehicle, once
        x = history.reshape(B * H, d).clone()
        batch = L.CacheBatch(ints(own), ints([H * b for b in range(B + 1)]), ints([H] * B), B * H, max_new=H)
        last = forward(x, past.reshape(B * H, A), m.positions(range(H), B), batch).view(B, H, d)[:, -1]
        # the partly filled page of the history, copied for each candidate
        for args, _ in pools:
            for t in args:
                if t is not None and H % page:
                    flat = t.view(torch.uint8) if t.element_size() == 1 else t
                    flat[table[:, full].astype(np.int64)] = flat[np.repeat(own[:, full], S).astype(np.int64)]
        x = last.repeat_interleave(S, 0)
        acts = cands.reshape(n, T, A)
        for t in range(T):
            batch = L.CacheBatch(ints(table), ints(np.arange(n + 1)), ints([H + t + 1] * n), n, max_new=1,
                                 max_length=H + T)
            x = x + acts[:, t] @ m.embed
            x = forward(x.clone(), acts[:, t].contiguous(), m.positions([H + t], n), batch)
        return ((x.view(B, S, d) - goal[:, None]) ** 2).mean(-1)

    scorer = L.CallbackScorer(ctx, B, score)
    planner = L.MppiPlanner(ctx, L.MppiConfig(T, S, A, seed=3, temperature=0.1))
    plan = planner.plan(scorer, batch=B)
    cands = L.device_tensor(planner.last_candidates_ptr(), (B, S, T, A)).clone()

    def plain(b, s):
        x = m.plain(history[b].double(), past[b].double(), m.positions(range(H), 0), windows)[-1]
        seq, acts = history[b].double(), past[b].double()
        for t in range(T):
            a = cands[b, s, t].double()
            seq, acts = torch.cat([seq, (x + a @ m.embed.double())[None]]), torch.cat([acts, a[None]])
            x = m.plain(seq, acts, m.positions(range(H + t + 1), 0), windows)[-1]
        return float(((x - goal[b].double()) ** 2).mean())

    # bf16 operands of a dozen products and norms: 12 roundings of 2^-8 at most on the state, twice that on its
    # square; 8-bit keys and values 2^-4 instead, averaged by the attention over at least 17 keys
    rel = 24 * 2.0 ** -8 if not codes else 24 * 2.0 ** -8 + 4 * 2.0 ** -4
    for b, s in ((0, 0), (0, 17), (1, 5), (1, 23)):
        want = plain(b, s)
        assert abs(float(plan.scores[b, s]) - want) <= rel * want, (b, s, float(plan.scores[b, s]), want)
    assert plan.best_indices == [int(i) for i in plan.scores.argmin(1)]
    planner.close()
    scorer.close()
