"""Linear attention where a call could go wrong unseen: values that are not
finite in the first chunk of many blocks at once."""
import pytest

import lewm_b200 as L
from test_gpu_linear import BF16, DECAYS, E32, F16, close, gen, ints, randn, recurrence, tolerances

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_infinities_in_the_first_chunk_of_many_sequences(ctx, d, dtype):
    """A value that is not finite among the first tokens reaches those before it in no block, whichever of its warps
    sees it first."""
    g, n, sequences, heads, at = gen(30), 20, 400, 2, 11
    q, k, v = (randn(g, sequences * n, heads, d, dtype=dtype) for _ in range(3))
    news = [n] * sequences
    a = DECAYS["mild"](heads).cuda()
    states = randn(g, sequences, heads, d, d)
    want, mag, _, sizes = recurrence(q, k, v, a.float(), news, states, d ** -0.5)
    tol, _ = tolerances(dtype, d, n, a, want, mag, sizes, False)
    v[at::n, :, 3] = float("inf")
    out = torch.empty_like(q)
    b = L.StateBatch(states, ints([n * i for i in range(sequences + 1)]), sequences * n, n)
    L.linear_attention_device(ctx, b, q, k, v, out, a.float())
    ctx.synchronize()
    before = (torch.arange(sequences * n, device="cuda") % n) < at
    close(out[before], want[before], tol[before])
    assert not torch.isfinite(out[~before][:, :, 3]).any()
    others = [c for c in range(d) if c != 3]
    close(out[:, :, others], want[:, :, others], tol[:, :, others])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_few_tokens_use_every_channel(ctx, d, dtype):
    """Values whose channels differ by powers of two, over several tokens: each is read from where it was put."""
    g, n, heads = gen(31), 5, 3
    q, k = (randn(g, n, heads, d, dtype=dtype) for _ in range(2))
    v = (randn(g, n, heads, d) * torch.exp2((torch.arange(d, device="cuda") % 9 - 4).float())).to(dtype)
    a = DECAYS["mild"](heads).cuda()
    states, out = randn(g, 1, heads, d, d), torch.empty_like(q)
    want, mag, after, sizes = recurrence(q, k, v, a.float(), [n], states, d ** -0.5)
    L.linear_attention_device(ctx, L.StateBatch(states, ints([0, n]), n), q, k, v, out, a.float())
    ctx.synchronize()
    tol, state_tol = tolerances(dtype, d, n, a, want, mag, sizes, True)
    close(out, want, tol)
    close(states, after, state_tol)


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (F16, 64), (BF16, 32)])
@pytest.mark.parametrize("news", [[1, 8], [300, 70, 1400], [5000]], ids=str)
@pytest.mark.parametrize("where", ["k", "v"])
def test_out_may_be_the_keys_or_the_values(ctx, where, news, dtype, d):
    """In place of k or v, of heads of their own: what a token's state and outputs read is read before it is written."""
    g, n, heads = gen(32), sum(news), 3
    x = {name: randn(g, n, heads, d, dtype=dtype) for name in "qkv"}
    kept = {name: t.clone() for name, t in x.items()}
    a = DECAYS["mild"](heads).cuda()
    states = torch.zeros(len(news), heads, d, d, device="cuda")
    starts = [sum(news[:i]) for i in range(len(news) + 1)]
    L.linear_attention_device(ctx, L.StateBatch(states, ints(starts), n, max(news)), x["q"], x["k"], x["v"], x[where], a.float())
    ctx.synchronize()
    want, mag, after, sizes = recurrence(kept["q"], kept["k"], kept["v"], a.float(), news, torch.zeros_like(states), d ** -0.5)
    tol, state_tol = tolerances(dtype, d, max(news), a, want, mag, sizes, max(news) <= 8)
    close(x[where], want, tol)
    close(states, after, state_tol)
    for name in "qkv":
        assert name == where or torch.equal(x[name], kept[name])


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_out_over_values_that_are_not_finite(ctx, value):
    g, n, heads, d, at = gen(33), 700, 2, 128, 200
    q, k, v = (randn(g, n, heads, d, dtype=BF16) for _ in range(3))
    a = DECAYS["mild"](heads).cuda()
    states = torch.zeros(1, heads, d, d, device="cuda")
    want, mag, _, sizes = recurrence(q, k, v, a.float(), [n], states, d ** -0.5)
    tol, _ = tolerances(BF16, d, n, a, want, mag, sizes, False)
    v[at, 1, 5] = value
    L.linear_attention_device(ctx, L.StateBatch(states, ints([0, n]), n), q, k, v, v, a.float())
    ctx.synchronize()
    close(v[:at], want[:at], tol[:at])
    assert not torch.isfinite(v[at:, 1, 5]).any()
    others = [c for c in range(d) if c != 5]
    close(v[:, :, others], want[:, :, others], tol[:, :, others])


@pytest.mark.parametrize("layout", ["rows", "heads", "planes"])
@pytest.mark.parametrize("n", [300, 1500])
def test_out_between_keys_and_values(ctx, layout, n):
    """Fused layouts of which out is a part: no element of it is theirs."""
    g, heads, d = gen(34), 2, 128
    shape = {"rows": (n, 4, heads, d), "heads": (n, heads, 4, d), "planes": (heads, 4, n, d)}[layout]
    fused = randn(g, *shape, dtype=BF16)
    order = {"rows": (1, 0, 2, 3), "heads": (2, 0, 1, 3), "planes": (1, 2, 0, 3)}[layout]
    q, k, out, v = fused.permute(order).unbind(0)
    kept = [t.clone() for t in (q, k, v)]
    a = DECAYS["mild"](heads).cuda()
    states = torch.zeros(1, heads, d, d, device="cuda")
    L.linear_attention_device(ctx, L.StateBatch(states, ints([0, n]), n), q, k, v, out, a.float())
    ctx.synchronize()
    want, mag, after, sizes = recurrence(*kept, a.float(), [n], torch.zeros_like(states), d ** -0.5)
    tol, state_tol = tolerances(BF16, d, n, a, want, mag, sizes, False)
    close(out, want, tol)
    close(states, after, state_tol)
    assert all(torch.equal(x, y) for x, y in zip((q, k, v), kept))


def test_out_over_keys_or_values_that_heads_share_is_refused(ctx):
    n, d = 70, 64
    fused = torch.zeros(n, 8, d, device="cuda", dtype=BF16)
    q, other = fused[:, :4], fused[:, 4:]
    a = torch.zeros(4, device="cuda")
    b = L.StateBatch(torch.zeros(1, 4, d, d, device="cuda"), ints([0, n]), n)
    apart = torch.zeros(n, 2, d, device="cuda", dtype=BF16)
    for name, k, v in (("k", other[:, :2], apart), ("v", apart, other[:, :2])):
        with pytest.raises(L.LwmError, match=f"out may be {name} only with as many kv_heads as heads and the same strides"):
            L.linear_attention_device(ctx, b, q, k, v, other, a)
    with pytest.raises(L.LwmError, match="out may be k only"):  # other strides
        L.linear_attention_device(ctx, b, q, torch.as_strided(other, (n, 4, d), (4 * d, d, 1), other.storage_offset()), q, other, a)


# ---- what a state keeps while nothing is added to it, or little

FADES = [(9, -0.5), (64, -0.27), (64, -1.0), (128, -0.135), (130, -0.5), (300, -0.2), (700, -0.1), (5000, -0.012), (3000, -2.0 ** -12),
         (2000, 0.0)]


def kept_tolerance(dtype, n, rate, out, mag, sizes):
    """A chunk of 64 tokens or more (or a part of them) multiplies the state once: the exponent is off by 2^-24 of it,
    its exponential by two steps of 2^-24 and what follows by two more, the sums of a chunk by three; a cut along time
    joins parts once more.  Keys of a chunk: in two parts or more of the type (f16 down to 2^-38 of the largest of a
    channel).  Outputs: the state's rounding for its product with q, and their own."""
    u = torch.finfo(dtype).eps / 2
    state = E32 * (2 * abs(rate) * n + 8 * (n / 64 + 2)) + 1.01 * u * u + 64 * 2.0 ** -38
    return mag * (state + 1.01 * u + 200 * E32) + u * (out.abs() * 1.001 + torch.finfo(dtype).tiny), sizes * state + 1e-44


@pytest.mark.parametrize("n,rate", FADES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("keys", [0, 40])
def test_states_that_nothing_is_added_to_keep_what_is_left(ctx, d, dtype, n, rate, keys):
    """Tokens whose keys are zero (behind some whose keys are not): the state is what the decay leaves of it, to the
    precision of what is left, however little that is."""
    g, heads, n = gen(35), 2, n + keys
    q, k, v = (randn(g, n, heads, d, dtype=dtype) for _ in range(3))
    k[keys:] = 0
    a = torch.tensor([rate, rate / 2], device="cuda", dtype=torch.float64)
    states, out = randn(g, 1, heads, d, d), torch.empty_like(q)
    want, mag, after, sizes = recurrence(q, k, v, a.float(), [n], states, d ** -0.5)
    L.linear_attention_device(ctx, L.StateBatch(states, ints([0, n]), n), q, k, v, out, a.float())
    ctx.synchronize()
    tol, state_tol = kept_tolerance(dtype, n, rate, want, mag, sizes)
    close(states, after, state_tol)
    close(out, want, tol)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_many_short_sequences_keep_what_is_left(ctx, d, dtype):
    """The same for more sequences than are cut along time, of one chunk and of two."""
    g, heads, news = gen(36), 4, [64, 128, 130, 0, 100] * 12
    n, s = sum(news), len(news)
    q, v = (randn(g, n, heads, d, dtype=dtype) for _ in range(2))
    k = torch.zeros_like(q)
    a = torch.tensor([-0.1, -0.2, -0.35, -0.5], device="cuda", dtype=torch.float64)
    states, out = randn(g, s, heads, d, d), torch.empty_like(q)
    want, mag, after, sizes = recurrence(q, k, v, a.float(), news, states, d ** -0.5)
    L.linear_attention_device(ctx, L.StateBatch(states, ints([sum(news[:i]) for i in range(s + 1)]), n, 130), q, k, v, out, a.float())
    ctx.synchronize()
    tol, state_tol = kept_tolerance(dtype, 130, -0.5, want, mag, sizes)
    close(states, after, state_tol)
    close(out, want, tol)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("keys", [0.0, 1.0 / 64])
def test_single_tokens_forget_as_a_history_does(ctx, d, dtype, keys):
    """4096 calls of a token each, at log decays whose factor lies between two floats.  A state rounds twice a token,
    half a step at most each, their signs at random: its norm moves by 2^-24 sqrt(2 n) or less (twice that allowed,
    and 16 steps for what is common to all).  Without keys the signs are not at random: a token takes |a| 2^23 steps
    and more off an element, whose part of a step stays alike until the element has moved, so c = a^2 n 2^23 times
    in the run (once at least) a new sign begins, and the norm moves by n / c sqrt(c) times the root mean square of a
    rounding, 0.29 steps of 2^-23 at most.  A factor that is rounded once is off by up to 2^-25 a token, all to one
    side: 2^-13 after so many."""
    g, n, a = gen(37), 4096, torch.tensor([-2.0 ** -12, -3e-5, -1e-6, -0.01], device="cuda", dtype=torch.float64)
    heads = a.numel()
    q, k, v = (randn(g, n, heads, d, dtype=dtype) for _ in range(3))
    k *= keys
    first = randn(g, 1, heads, d, d)
    a = a.float().double()
    left = torch.exp(a[None] * torch.arange(n - 1, -1, -1, device="cuda", dtype=torch.float64)[:, None])[..., None]
    want = torch.exp(a * n)[:, None, None] * first[0].double() + torch.einsum("nhk,nhv->hkv", k.double() * left, v.double())
    limit = E32 * (2 * (2 * n) ** 0.5 + 16 + (0.58 * n / (a * a * n * 2.0 ** 23).clamp(min=1.0).sqrt() if keys == 0 else 0.0))
    steps, out = first.clone(), torch.empty_like(q)
    b = L.StateBatch(steps, ints([0, 1]), 1)
    for i in range(n):
        L.linear_attention_device(ctx, b, q[i:i + 1], k[i:i + 1], v[i:i + 1], out[i:i + 1], a.float())
    history = first.clone()
    L.linear_attention_device(ctx, L.StateBatch(history, ints([0, n]), n), q, k, v, torch.empty_like(q), a.float())
    eights = first.clone()
    for i in range(0, n, 8):
        L.linear_attention_device(ctx, L.StateBatch(eights, ints([0, 8]), 8), q[i:i + 8], k[i:i + 8], v[i:i + 8], out[i:i + 8], a.float())
    ctx.synchronize()
    for got in (steps, history, eights):
        off = (got[0].double() - want).norm(dim=(1, 2)) / want.norm(dim=(1, 2))
        assert (off <= limit + (1.01 * (torch.finfo(dtype).eps / 2) ** 2 if got is history else 0.0)).all(), off
