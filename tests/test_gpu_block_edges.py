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
