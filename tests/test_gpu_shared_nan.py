"""NaN and infinities in what a sequence has behind its shared prefix, where it
is all that the sequence sees there: tails of one token and of a few, keys,
page scales and queries, one row a kv head and two, beside a finite prefix and
for a sequence of no group.  The same batch by the plain attention is not a
number where the call is not, and the rest is compared with 64 bits."""
import pytest

import lewm_b200 as L
from test_gpu_blocks import gen, randn
from test_gpu_shared import POOLS, Groups

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


def both(ctx, g, news, heads, q, max_tail):
    """The call, checked against 64 bits, and the plain attention of the same batch."""
    _, out = g.call(ctx, news, heads, q=q, max_tail=max_tail)
    plain = torch.full_like(out, 5.0)
    L.cache_attention_device(ctx, g.c.cache, g.c.batch(news, tokens=q.shape[0]), q, plain)
    ctx.synchronize()
    return out, plain


def put(g, s, at, kv, value, which="k"):
    """Token `at` of sequence s, kv head kv: every channel."""
    c = g.c
    pool = c.k if which == "k" else c.v
    page, slot = int(c.table[s, at // c.page]), at % c.page
    if c.codes:
        assert value != value
        pool.view(torch.uint8)[page, kv, slot] = 0x7f
    else:
        pool[page, kv, slot] = value


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("max_tail", [100, 0])
def test_keys_that_are_not_a_number(ctx, dtype, codes, d, rows, max_tail):
    """max_tail is for the shape of the launch, whichever kernel that is."""
    prefix, tails = 64, [1, 3, 3, 2, 17, 90]
    g = Groups(40, [(prefix, tails)], 32, 2, d, dtype, codes, alone=[1, 9])
    news, heads = [1] * 8, 2 * rows
    put(g, 0, prefix, 1, NAN)  # all of a tail of one token
    for i in range(3):
        put(g, 1, prefix + i, 1, NAN)  # all of a tail
    put(g, 2, prefix + 1, 1, NAN)  # one of three
    for i in range(16):
        put(g, 4, prefix + i, 1, NAN)  # a whole first run of keys
    put(g, 6, 0, 1, NAN)  # all of a sequence of no group
    out, plain = both(ctx, g, news, heads, randn(gen(41), 8 + 3, heads, d, dtype=dtype), max_tail)
    assert torch.equal(torch.isnan(out), torch.isnan(plain))
    bad = torch.isnan(out[:8])
    assert bad[[0, 1, 2, 4, 6], rows:].all() and not bad[:, :rows].any() and not bad[[3, 5, 7]].any()


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("value", [NAN, INF])
def test_queries_that_are_not_finite(ctx, dtype, codes, d, value):
    """In a group, and in sequences of none, with one row a kv head and two tokens.  A query of infinities has scores
    of infinities: not a number, but zero where all that it sees scores minus infinity."""
    for news in ([1] * 5, [2, 2, 2, 2, 1]):
        g = Groups(42, [(96, [2, 40, 5])], 32, 2, d, dtype, codes, alone=[2, 50])
        q = randn(gen(43), sum(news) + 3, 2, d, dtype=dtype)
        starts = [sum(news[:s]) for s in range(5)]
        rows = [starts[s] for s in (1, 3, 4)]
        finite = q.clone()
        q[rows, 1, 3] = value
        check = g.check
        g.check = lambda *_: None
        out, plain = both(ctx, g, news, 2, q, 60)
        assert torch.equal(torch.isnan(out), torch.isnan(plain)) and (out[rows, 1] == 0).equal(plain[rows, 1] == 0)
        assert (torch.isnan(out[rows, 1]) | (out[rows, 1] == 0)).all()
        # the other rows, against 64 bits
        g.check = check
        _, clean = g.call(ctx, news, 2, q=finite, max_tail=60)
        clean[rows, 1] = out[rows, 1]
        assert ((out == clean) | (torch.isnan(out) & torch.isnan(clean))).all()
        if value != value:
            assert torch.isnan(out[rows, 1]).all()
        assert not torch.isnan(out[:sum(news), 0]).any() and not torch.isnan(out[starts[2], 1]).any()


@pytest.mark.parametrize("dtype", [p[0] for p in POOLS[:2]])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_key_scales_that_are_not_finite(ctx, dtype, d, value):
    """A scale multiplies the product with a key's codes: infinite ones make scores of either infinity, of which minus
    infinity weighs nothing, as in the plain attention."""
    g = Groups(44, [(64, [1, 6, 40])], 32, 1, d, dtype, True, alone=[3])
    for s in (0, 1, 3):
        g.c.ks[int(g.c.table[s, 0 if s == 3 else 2])] = value
    if value == value:
        g.check = lambda *_: None
    out, plain = both(ctx, g, [1] * 4, 1, randn(gen(45), 7, 1, d, dtype=dtype), 60)
    assert torch.equal(torch.isnan(out), torch.isnan(plain))
    assert torch.isnan(out[[0, 1, 3]]).all() or value == value
    assert not torch.isnan(out[2]).any()


@pytest.mark.parametrize("dtype", [p[0] for p in POOLS[:2]])
def test_scores_of_minus_infinity_weigh_nothing(ctx, dtype):
    """A tail whose scores are all minus infinity leaves the prefix's result, whatever its values are; a sequence of
    no group that sees nothing else is zero."""
    g = Groups(46, [(64, [1, 6, 40])], 32, 1, 64, dtype, alone=[3])
    for s, n in ((0, 1), (1, 6)):
        for i in range(n):
            put(g, s, 64 + i, 0, -INF)
            put(g, s, 64 + i, 0, INF, "v")
    for i in range(3):
        put(g, 3, i, 0, -INF)
        put(g, 3, i, 0, NAN, "v")
    q = randn(gen(47), 7, 1, 64, dtype=dtype).abs() + 0.25
    out = torch.full_like(q, 5.0)
    c, news = g.c, [1] * 4
    p = L.SharedPrefix(torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([64], dtype=torch.int32, device="cuda"),
                       None, 64, 60)
    b = g.batch(news, 7, 0)
    size = L.shared_attention_workspace(c.cache, b, p, 1)
    assert size > 0
    L.cache_attention_shared_device(ctx, c.cache, b, p, q, out, torch.empty(size, device="cuda", dtype=torch.uint8))
    ctx.synchronize()
    assert torch.isfinite(out).all() and (out[3] == 0).all() and (out[4:] == 5.0).all()
    # as without those tokens: the prefix alone
    lead = c.dense("k", 0)[:64, 0], c.dense("v", 0)[:64, 0]
    for s in (0, 1):
        w = torch.softmax(q[s, 0].double() @ lead[0].T / 8, -1)
        want = w @ lead[1]
        u = torch.finfo(dtype).eps / 2
        # the weights' rounding, the scores' (64 + 6 products and sums, twice), the exponentials and the join's 2^-15
        tol = (w @ lead[1].abs()) * (u + 2.0 ** -15 + 2.0 ** -16) + u * want.abs() * 1.001
        assert ((out[s, 0].double() - want).abs() <= tol).all()
