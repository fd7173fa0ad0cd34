"""Linear attention with decay against its recurrence in 64 bits: a few tokens
and whole histories, every width and type, shared heads, strided and ragged
batches, states in place, forked and from zero, extreme decays, infinities and
NaN, and what the calls skip and report.

Tolerances count roundings.  M is the same recurrence over absolute values, so
the sum of all magnitudes that enter a value.  In chunks the weights (of the
operands' type) and the state (bf16 or 11 bits) are rounded once, at most u =
half a step of the type each and of different parts of M; keys times decay
keep two parts at least, u^2.  In 32 bits a value passes through at most one product
and one sum a token, the sums over channels, and powers of the decay: 2^-24
each (|log lambda| 64 of them for the power's argument, 4 a chunk to carry
it)."""
import numpy as np
import pytest

import lewm_b200 as L

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E32 = 2.0 ** -24
DECAYS = {"mild": lambda h: -(2.0 ** -(3.0 + torch.arange(h, dtype=torch.float64) % 8)),
          "none": lambda h: torch.zeros(h, dtype=torch.float64),
          "strong": lambda h: torch.full((h,), -1.5, dtype=torch.float64),
          "afresh": lambda h: torch.full((h,), -float("inf"), dtype=torch.float64)}


def U(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(dtype, out):
    return U(dtype) * (out.abs() * 1.001 + torch.finfo(dtype).tiny)


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


def close(got, want, tol):
    got = got.double()
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(got == want)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {i}: {float(got[i])} for "
                             f"{float(want[i])}, tolerance {float(tol.expand_as(want)[i])}")


def recurrence(q, k, v, log_decay, news, source, scale):
    """(outputs, states after, and both with every value's magnitude) in 64 bits; source [sequences, heads, d, d]."""
    heads, d = q.shape[1:]
    share = heads // k.shape[1]
    lam = torch.exp(log_decay.double())[:, None, None]
    q, k, v = q.double(), k.double().repeat_interleave(share, 1), v.double().repeat_interleave(share, 1)
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    states, sizes, at = [], [], 0
    for s, n in enumerate(news):
        st = source[s].double().clone()
        size = st.abs()
        for i in range(at, at + n):
            st = lam * st + k[i][:, :, None] * v[i][:, None]
            size = lam * size + k[i].abs()[:, :, None] * v[i].abs()[:, None]
            out[i] = torch.einsum("hd,hde->he", q[i], st) * scale
            mag[i] = torch.einsum("hd,hde->he", q[i].abs(), size) * abs(scale)  # (a magnitude, whatever the sign)
        at += n
        states.append(st)
        sizes.append(size)
    return out, mag, torch.stack(states), torch.stack(sizes)


def tolerances(dtype, d, longest, log_decay, out, mag, sizes, stepwise):
    reach = float(torch.clamp(-log_decay, max=200.0).max()) * 64
    many = E32 * (2 * longest + d + 16 + reach + 4 * (longest / 64 + 1))
    state = many + (0.0 if stepwise else 1.01 * U(dtype) ** 2)
    weights = 0.0 if stepwise else 1.01 * U(dtype)
    # (f16 weights and keys end 2^-38 below the row's largest)
    return mag * (weights + state + 64 * 2.0 ** -38) + rounded(dtype, out), sizes * (state + 64 * 2.0 ** -38) + 1e-44


def call(ctx, g, dtype, d, heads, kv, news, decay, max_new, slots=None, source=None, target=None, scale=None, behind=3):
    s, tokens = len(news), sum(news)
    qkv = randn(g, tokens + behind, heads + 2 * kv, d, dtype=dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    out = torch.full((tokens + behind, heads, d), 7.0, device="cuda", dtype=dtype)
    states = randn(g, slots or s, heads, d, d)
    before = states.clone()
    a = DECAYS[decay](heads).cuda()
    starts = ints(np.concatenate([[0], np.cumsum(news)]))
    b = L.StateBatch(states, starts, tokens + behind, max_new, source=None if source is None else ints(source),
                     target=None if target is None else ints(target))
    L.linear_attention_device(ctx, b, q, k, v, out, a.float(), scale=scale)
    ctx.synchronize()
    src = list(range(s)) if source is None else source
    dst = list(range(s)) if target is None else target
    first = torch.stack([before[i] if i >= 0 else torch.zeros_like(before[0]) for i in src])
    want, mag, after, sizes = recurrence(q[:tokens], k[:tokens], v[:tokens], a.float(), news, first,
                                         d ** -0.5 if scale is None else scale)
    tol, state_tol = tolerances(dtype, d, max(news), a, want, mag, sizes, max_new <= 8)
    close(out[:tokens], want, tol)
    assert (out[tokens:] == 7.0).all()
    kept = [(i, t) for i, t in enumerate(dst) if t >= 0]
    if kept:
        i, t = (torch.tensor(x, device="cuda") for x in zip(*kept))
        close(states[t], after[i], state_tol[i])
    rest = [i for i in range(states.shape[0]) if i not in dst]
    assert torch.equal(states[rest], before[rest])
    return out, states


LENGTHS = [[1], [0, 1, 1], [3, 8, 1, 0], [9], [63, 64], [65, 0, 1, 130], [200, 17]]


@pytest.mark.parametrize("news", LENGTHS, ids=str)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (4, 2)])
def test_against_the_recurrence(ctx, news, d, dtype, heads, kv):
    call(ctx, gen(1), dtype, d, heads, kv, news, "mild", max(news))


@pytest.mark.parametrize("news", [[300, 63, 64, 65, 0, 1, 127], [128, 256, 129, 9], [600], [384, 2, 130] + [1] * 50], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_lengths_at_the_edges_of_longer_chunks(ctx, news, d):
    call(ctx, gen(22), BF16, d, 4, 2, news, "mild", max(news))


@pytest.mark.parametrize("news", [[1, 2], [5], [70, 129]], ids=str)
@pytest.mark.parametrize("decay", ["none", "strong", "afresh"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decays(ctx, news, decay, dtype):
    call(ctx, gen(2), dtype, 64, 2, 1, news, decay, max(news))


@pytest.mark.parametrize("max_new", [8, 9, 17])
def test_both_kernels_at_the_same_batch(ctx, max_new):
    call(ctx, gen(3), BF16, 64, 3, 3, [8, 0, 5, 1], "mild", max_new)


@pytest.mark.parametrize("news", [[1] * 5, [40, 0, 9, 1, 66]], ids=str)
def test_candidates_fork_from_one_state(ctx, news):
    call(ctx, gen(4), BF16, 64, 4, 4, news, "mild", max(news), slots=9, source=[2] * 5, target=[7, 0, -1, 8, 4])
    call(ctx, gen(5), F16, 32, 2, 2, news, "mild", max(news), slots=6, source=[-1, 5, -1, -7, 5], target=[0, 1, 2, 3, 4])


@pytest.mark.parametrize("news", [[4], [100]], ids=str)
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0])
def test_scale(ctx, news, scale):
    call(ctx, gen(6), BF16, 32, 2, 2, news, "mild", max(news), scale=scale)


def test_many_sequences_and_a_long_one(ctx):
    call(ctx, gen(7), BF16, 64, 2, 2, [1] * 700, "mild", 1)
    call(ctx, gen(8), BF16, 128, 1, 1, [1500], "mild", 1500)
    call(ctx, gen(9), F16, 64, 1, 1, [1100, 3], "none", 1100)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news", [[5000], [700, 0, 4700, 130, 1]], ids=str)
def test_long_sequences_are_cut_along_time(ctx, d, news):
    call(ctx, gen(19), BF16, d, 2, 1, news, "mild", max(news))
    n = len(news)
    call(ctx, gen(20), BF16, d, 1, 1, news, "none", max(news), slots=n + 2, source=[n + 1] * (n - 1) + [-1], target=list(range(n)))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_sums_are_rounded_not_cut_off(ctx, d, dtype):
    """Without decay the state is K^T V.  A rounding at every chunk of 64 tokens or more (two of them) moves its norm
    by 2^-24 sqrt(2 n / 64) / 2 or so, as their signs differ; sums that are cut off at every step of the tensor cores
    lean to one side, 4e-6 and more at this length."""
    g, n = gen(21), 16384
    q, k, v = (randn(g, n, 1, d, dtype=dtype) for _ in range(3))
    states, out = torch.zeros(1, 1, d, d, device="cuda"), torch.empty_like(q)
    L.linear_attention_device(ctx, L.StateBatch(states, ints([0, n]), n), q, k, v, out, torch.zeros(1, device="cuda"))
    ctx.synchronize()
    want = k[:, 0].double().T @ v[:, 0].double()
    assert (states[0, 0].double() - want).norm() <= E32 * (2 * (2 * n / 64) ** 0.5 + 16) * want.norm()


def test_half_precision_keeps_large_and_small_states(ctx):
    """Scores, keys and states far beyond f16's range on either side."""
    g, d, n = gen(10), 64, 130
    for size, key in ((3e6, 30.0), (1e-6, 1e-3)):
        q, k, v = randn(g, n, 1, d, dtype=F16), (randn(g, n, 1, d) * key).to(F16), (randn(g, n, 1, d) * 1e-3).to(F16)
        states = randn(g, 1, 1, d, d) * size
        before, out = states.clone(), torch.empty_like(q)
        a = torch.full((1,), -0.05, device="cuda", dtype=torch.float64)
        b = L.StateBatch(states, ints([0, n]), n)
        L.linear_attention_device(ctx, b, q, k, v, out, a.float(), scale=1e-3 / max(1.0, size))
        want, mag, after, sizes = recurrence(q, k, v, a.float(), [n], before, 1e-3 / max(1.0, size))
        tol, state_tol = tolerances(F16, d, n, a, want, mag, sizes, False)
        close(out, want, tol)
        close(states, after, state_tol)


@pytest.mark.parametrize("where", ["v", "k", "q"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinities_and_nan_reach_later_tokens_of_their_head_only(ctx, where, value, dtype):
    infinities(ctx, where, value, dtype, 64, 150, 77)


@pytest.mark.parametrize("where", ["v", "k", "q"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("d,n,at", [(64, 300, 77), (64, 3000, 1600), (128, 300, 200), (128, 3000, 700), (128, 70, 69)])
def test_infinities_and_nan_in_long_sequences(ctx, where, value, d, n, at):
    infinities(ctx, where, value, BF16, d, n, at)


def infinities(ctx, where, value, dtype, d, n, at):
    g = gen(11)
    x = {name: randn(g, n, 2, d, dtype=dtype) for name in "qkv"}
    x[where][at, 1, 5] = value
    states = randn(g, 1, 2, d, d)
    before, out = states.clone(), torch.empty_like(x["q"])
    a = DECAYS["mild"](2).cuda()
    L.linear_attention_device(ctx, L.StateBatch(states, ints([0, n]), n), x["q"], x["k"], x["v"], out, a.float())
    clean = {name: torch.nan_to_num(t, nan=0.0, posinf=0.0) for name, t in x.items()}
    want, mag, after, sizes = recurrence(clean["q"], clean["k"], clean["v"], a.float(), [n], before, d ** -0.5)
    tol, state_tol = tolerances(dtype, d, n, a, want, mag, sizes, False)
    close(out[:, 0], want[:, 0], tol[:, 0])
    close(out[:at], want[:at], tol[:at])
    close(states[0, 0], after[0, 0], state_tol[0, 0])
    if where == "q":
        close(out[at + 1:], want[at + 1:], tol[at + 1:])
        assert not torch.isfinite(out[at, 1]).any()
        close(states, after, state_tol)
    elif where == "k":
        assert not torch.isfinite(out[at:, 1]).any()
    else:
        assert not torch.isfinite(out[at:, 1, 5]).any()
        others = [c for c in range(d) if c != 5]
        close(out[:, 1][:, others], want[:, 1][:, others], tol[:, 1][:, others])
        close(states[0, 1][:, others], after[0, 1][:, others], state_tol[0, 1][:, others])
        assert not torch.isfinite(states[0, 1][:, 5]).any()


def test_out_may_be_q_and_results_repeat(ctx):
    g, n = gen(12), 300
    q, k, v = (randn(g, n, 3, 64, dtype=BF16) for _ in range(3))
    a = DECAYS["mild"](3).float().cuda()
    held = randn(g, 1, 3, 64, 64)
    for cut in (n, 5):
        outs, states = [], []
        for same in (False, True, False):
            st, qq = held.clone(), q.clone()
            out = qq if same else torch.empty_like(qq)
            b = L.StateBatch(st, ints([0, cut]), n, cut)
            L.linear_attention_device(ctx, b, qq, k, v, out, a)
            outs.append(out[:cut].clone())
            states.append(st)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        assert torch.equal(states[0], states[1]) and torch.equal(states[0], states[2])


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (F16, 64)])
@pytest.mark.parametrize("where,heads", [("q", 2), ("beside", 2), ("q", 12)])
def test_long_sequences_in_place(ctx, dtype, d, where, heads):
    """Out is q, or lies between the rows of a fused projection's output: no row of it may hold a state."""
    g, n, h = gen(24), 5000, heads
    fused = randn(g, n, 4 * h, d, dtype=dtype)
    kept = fused.clone()
    q, k, v, out = (fused[:, i * h:(i + 1) * h] for i in range(4))
    if where == "q":
        out = q
    a = DECAYS["mild"](h).cuda().float()
    states = torch.zeros(1, h, d, d, device="cuda")
    L.linear_attention_device(ctx, L.StateBatch(states, ints([0, n]), n), q, k, v, out, a)
    ctx.synchronize()
    first = torch.zeros_like(states)
    want, mag, after, sizes = recurrence(kept[:, :h], k, v, a, [n], first, d ** -0.5)
    tol, state_tol = tolerances(dtype, d, n, a, want, mag, sizes, False)
    close(out, want, tol)
    close(states, after, state_tol)
    rest = slice(h, None) if where == "q" else slice(0, 3 * h)
    assert torch.equal(fused[:, rest], kept[:, rest])


def test_a_rollout_in_pieces_is_the_whole(ctx):
    """A history in one call, or in chunks and single tokens with the state handed on."""
    g, n = gen(13), 150
    q, k, v = (randn(g, n, 2, 64, dtype=BF16) for _ in range(3))
    a = DECAYS["mild"](2).cuda()
    states, out = torch.zeros(1, 2, 64, 64, device="cuda"), torch.empty_like(q)
    at = 0
    for m in (100, 1, 1, 30, 8, 10):
        b = L.StateBatch(states, ints([0, m]), m)
        L.linear_attention_device(ctx, b, q[at:at + m], k[at:at + m], v[at:at + m], out[at:at + m], a.float())
        at += m
    assert at == n
    want, mag, after, sizes = recurrence(q, k, v, a.float(), [n], torch.zeros_like(states), 64 ** -0.5)
    tol, state_tol = tolerances(BF16, 64, n, a, want, mag, sizes, False)
    close(out, want, tol)
    close(states, after, state_tol + 6 * E32 * sizes)


@pytest.mark.parametrize("m,d", [(1, 64), (90, 64), (300, 64), (3000, 64), (300, 128), (3000, 128)])
def test_captured_calls_replay(ctx, m, d):
    g = gen(14)
    q, k, v = (randn(g, 2 * m, 2, d, dtype=BF16) for _ in range(3))
    a = DECAYS["mild"](2).float().cuda()
    states, out = randn(g, 2, 2, d, d), torch.empty_like(q)
    held = states.clone()
    b = L.StateBatch(states, ints([0, m, 2 * m]), 2 * m, m)
    L.linear_attention_device(ctx, b, q, k, v, out, a)
    first, once = out.clone(), states.clone()
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        L.linear_attention_device(ctx, b, q, k, v, out, a)
    states.copy_(held)
    out.zero_()
    graph.replay()
    ctx.synchronize()
    assert torch.equal(out, first) and torch.equal(states, once)
    del graph


@pytest.mark.parametrize("n", [300, 5000])
def test_infinite_queries_leave_the_other_rows(ctx, n):
    """Rows that are not finite for their own queries' sake, at finite values: theirs alone."""
    g, d = gen(23), 64
    q, k, v = (randn(g, n, 2, d, dtype=BF16) for _ in range(3))
    a = DECAYS["mild"](2).cuda().float()
    clean, out = torch.empty_like(q), torch.empty_like(q)
    for o, x in ((clean, q), (out, q.clone())):
        if o is out:
            x[7::50, 1] = float("inf")
            x[n - 1, 0, 3] = float("nan")
        b = L.StateBatch(torch.zeros(1, 2, d, d, device="cuda"), ints([0, n]), n)
        L.linear_attention_device(ctx, b, x, k, v, o, a)
    ctx.synchronize()
    rows = torch.ones(n, 2, dtype=torch.bool, device="cuda")
    rows[7::50, 1] = rows[n - 1, 0] = False
    assert torch.equal(out[rows], clean[rows])
    assert torch.isnan(out[n - 1, 0]).all() and not torch.isfinite(out[7::50, 1]).any()


@pytest.mark.parametrize("news,d", [(1, 32), (70, 32), (300, 64), (3000, 64), (300, 128), (3000, 128)])
def test_what_does_not_fit_is_skipped_and_reported(ctx, news, d):
    g, tokens = gen(15), 3 * news
    q, k, v = (randn(g, tokens, 1, d, dtype=BF16) for _ in range(3))
    a = torch.zeros(1, device="cuda")
    for starts, source, target, message in (
            ([0, news, tokens + 1, tokens], [0, 1, 2], [0, 1, 2], "sequence [12]: starts are out of order or beyond the packed rows"),
            ([0, news, 2 * news, tokens], [0, 9, 2], [0, 1, 2], "sequence 1: state slot 9 is not in the pool"),
            ([0, news, 2 * news, tokens], [0, 1, 2], [0, 3, 2], "sequence 1: state slot 3 is not in the pool"),
            ([0, news, news, tokens], [0, 1, 2], [0, 1, 2], "sequence 2: more new tokens")):
        states = randn(g, 3, 1, d, d)
        before, out = states.clone(), torch.full_like(q, 5.0)
        b = L.StateBatch(states, ints(starts), tokens, news, ints(source), ints(target))
        L.linear_attention_device(ctx, b, q, k, v, out, a)
        with pytest.raises(L.LwmError, match=message):
            ctx.synchronize()
        ctx.synchronize()
        s = 2 if "sequence 2" in message else 1
        assert torch.equal(states[s], before[s])
        want, mag, after, sizes = recurrence(q[:news], k[:news], v[:news], a, [news], before[:1], d ** -0.5)
        tol, state_tol = tolerances(BF16, d, news, a, want, mag, sizes, news <= 8)
        close(out[:news], want, tol)
        close(states[:1], after, state_tol)
