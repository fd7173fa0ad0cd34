"""The transformer blocks at calls that their documentation allows and that
are easy to get wrong: conditioning shared by all rows, many bad sequences at
once, rows with nothing to weigh, batches above their bounds."""
import re

import numpy as np
import pytest

import lewm_b200 as L
from test_gpu_blocks import (BF16, F16, F32, MANY, Paged, check_norm, close, gen, ints, on_context_stream,  # noqa: F401
                             randn)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per", [33, 34, (1 << 31) - 1, 1 << 31, (1 << 31) + 1, (1 << 32) - 1])
@pytest.mark.parametrize("width", [192, 193])
def test_one_conditioning_row_for_all(ctx, per, width):
    """rows_per_cond may be anything from the rows up."""
    norm, x, y, x_out, h, gate, shift, scale = check_norm(ctx, 33, width, F32, BF16, BF16, 33, pre="layer")
    x2, h2 = torch.empty_like(x_out), torch.empty_like(h)
    L.gated_norm_device(ctx, norm, x, y, x2, h2, gate=gate, shift=shift, scale=scale, rows_per_cond=per)
    assert torch.equal(x2, x_out) and torch.equal(h2, h)


@pytest.mark.parametrize("call", ["append", "gather", "attention", "many rows"])
@pytest.mark.parametrize("what", ["page", "length", "both"])
def test_a_report_names_one_sequence_of_many(ctx, call, what):
    """Thousands of sequences are wrong at once, each in its own way: the report belongs to one of them."""
    n, kv, d = 3000, 2, 64
    c = Paged(230, [16], 16, kv, d, fill=0.0)
    table, lengths = np.arange(n)[:, None] + 10 ** 6, np.full(n, 16)
    if what != "page":
        lengths[:: 1 if what == "length" else 2] = -1000 - np.arange(n)[:: 1 if what == "length" else 2]
    rows = 2 * MANY if call == "many rows" else n
    b = L.CacheBatch(ints(table), ints(np.arange(n + 1)), ints(lengths), rows, max_new=MANY if call == "many rows" else 1)
    x, q = torch.zeros(rows, kv, d, device="cuda", dtype=BF16), torch.zeros(rows, 4, d, device="cuda", dtype=BF16)
    for _ in range(5):
        if call == "append":
            L.cache_append_device(ctx, c.cache, b, x, x)
        elif call == "gather":
            L.cache_gather_device(ctx, c.cache, b, x, x)
        else:
            L.cache_attention_device(ctx, c.cache, b, q, q)
        with pytest.raises(L.LwmError) as e:
            ctx.synchronize()
        m = re.search(r"sequence (\d+): (?:page (\d+) is not|length (-\d+) is)", e.value.message)
        assert m, e.value.message
        s, page, length = int(m[1]), m[2], m[3]
        if length:
            assert what != "page" and int(length) == lengths[s], e.value.message
        else:
            assert what != "length" and int(page) == 10 ** 6 + s and lengths[s] == 16, e.value.message
        ctx.synchronize()  # reported once


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("lengths,news,kw", [
    ([40, 1, 300], [1, 1, 1], {}), ([40, 1, 300], [3, 1, 12], dict(window=20)), ([4000], [1], {}),
    ([40] * 600, [1] * 600, dict(max_length=40)), ([300, 260], [140, 260], {}), ([700], [300], dict(window=160, sinks=3))])
def test_rows_whose_scores_are_all_minus_infinity_are_zero(ctx, dtype, d, lengths, news, kw):
    """Nothing weighs, also where the values are infinities or NaN."""
    many = max(news) > 100
    c = Paged(231, lengths, 16, 1, d, dtype, fill=0.0)
    c.fill_random(232)
    c.k[..., 0] = -float("inf")
    c.v[..., 1::5], c.v[..., 2::5] = float("inf"), float("nan")
    rows = MANY if many else sum(news)
    q = randn(gen(233), rows, 2, d, dtype=dtype)
    q[..., 0] = 1.0
    out = torch.full_like(q, 5.0)
    kw = dict(kw)
    b = c.batch(news, tokens=rows, max_length=kw.pop("max_length", 0), **(dict(max_new=MANY) if many else {}))
    L.cache_attention_device(ctx, c.cache, b, q, out, **kw)
    assert (out[:sum(news)] == 0).all() and (out[sum(news):] == 5.0).all()


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("many", [False, True])
def test_a_sequence_above_max_new_is_left_out(ctx, codes, many):
    """Its rows are zero or as they were, its pages too; the sequences around it get what they get without it."""
    n, most = (140, MANY) if many else (3, 3)
    news = [n, most + 1, n]
    c = Paged(234, [200, 200, 200], 64, 2, 64, BF16, codes, fill=1.0)
    c.fill_random(235)
    g, rows = gen(236), sum(news)
    q, k, v = randn(g, rows, 4, 64, dtype=BF16), randn(g, rows, 2, 64, dtype=BF16), randn(g, rows, 2, 64, dtype=BF16)

    def run(batch):
        pools = [t.clone() for t in (c.k, c.v, c.ks, c.vs) if t is not None]
        cache = L.PagedCache(*pools, dtype=BF16)
        out, ko, vo, qo = (torch.full_like(t, 5.0) for t in (q, k, v, q))
        L.cache_attention_device(ctx, cache, batch, q, out)
        L.cache_append_device(ctx, cache, batch, k, v, rotary=L.Rotary.make([64], [1e4]), q=q, q_out=qo)
        L.cache_gather_device(ctx, cache, batch, ko, vo)
        return [out, ko, vo, qo], pools

    def batch(lengths):
        return L.CacheBatch(ints(c.table), ints([0, n, n + most + 1, rows]), ints(lengths), rows, max_new=most)

    got, pools = run(batch([200, 200, 200]))
    with pytest.raises(L.LwmError, match=f"sequence 1: more new tokens \\({most + 1}\\)"):
        ctx.synchronize()
    # (the second run's rows are packed without the sequence, so its inputs are moved there first)
    moved = [torch.cat([t[:n], t[-n:], t[n:-n]]) for t in (q, k, v)]
    for t, m in zip((q, k, v), moved):
        t.copy_(m)
    want, want_pools = run(L.CacheBatch(ints(c.table[[0, 2]]), ints([0, n, 2 * n]), ints([200, 200]), rows, max_new=most))
    ctx.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[:n], b[:n]) and torch.equal(a[-n:], b[n:2 * n])
        assert ((a[n:-n] == 5.0) | (a[n:-n] == 0.0)).all()
    for a, b in zip(pools, want_pools):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("turn", [False, True])
def test_scales_next_to_a_border(ctx, dtype, turn):
    """A page's scale is the least power of two that holds its largest value: on 448 powers exactly, one step above
    and one below; what is not turned has no allowance."""
    kv, d, page = 8, 32, 16
    top = 2.0 ** torch.arange(-9, 7, device="cuda") * 448.0  # one token a page
    step = 2.0 ** (-7 if dtype == BF16 else -10) * 2.0 ** torch.arange(-9, 7, device="cuda") * 256.0
    for move, power in ((0.0, 0), (1.0, 1), (-1.0, 0)):
        c = Paged(237, [1] * 16, page, kv, d, dtype, codes=True, fill=2.0 ** 60)
        x = torch.zeros(16, kv, d, device="cuda")
        x[:, :, 5] = -(top + move * step)[:, None]
        x = x.to(dtype)
        L.cache_append_device(ctx, c.cache, c.batch([1] * 16), x, x, rotary=L.Rotary.make([d], [1e4]) if turn else None)
        want = (2.0 ** (torch.arange(-9, 7, device="cuda") + power))[:, None].expand(16, kv)
        pages = torch.tensor(c.table[:, 0], device="cuda")
        assert torch.equal(c.vs[pages], want)
        assert torch.equal(c.ks[pages], want)  # (at position 0 a turn is exact)
