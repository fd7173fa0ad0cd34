"""Drawn tokens against the definition in 64 bits, equal for every row: the
filters alone and together, every type and the sizes at which the kernel
changes its shape, ties, empty rows, infinities and NaN, parameters of each
row, and the edges of the random number.

Log-probabilities: weights carry 2^-43 (absolute, against a largest weight of
one) and 1e-13, so the logarithm of a drawn weight w is off by 2^-44 / w and
the rounding to 32 bits; a drawn weight is compared where w > 2^-20."""
import math

import numpy as np
import pytest

import lewm_b200 as L

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


def definition(row, u, temperature, top_k, top_p, min_p):
    """(token, log-probability) of one row (float64 numpy)."""
    row = np.where(np.isnan(row), -np.inf, row)
    top = row.max()
    if top == -np.inf:
        return -1, -np.inf
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    with np.errstate(invalid="ignore"):
        w = (row == np.inf).astype(float) if top == np.inf else np.exp((row - top) / temperature)
    order = np.lexsort((np.arange(len(row)), -row))
    order = order[row[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1.0:
        sums = np.cumsum(w[order])
        order = order[:1 + int(np.searchsorted(sums, max(top_p, 0.0) * sums[-1], side="left"))]
    kept = np.sort(order[w[order] >= min_p])
    sums = np.cumsum(w[kept])
    i = min(int(np.searchsorted(sums, min(max(u, 0.0), 1.0) * sums[-1], side="right")), len(kept) - 1)
    return int(kept[i]), math.log(w[kept[i]] / sums[-1]) if w[kept[i]] > 0 else -np.inf


def run(ctx, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, check_weights=True):
    rows = logits.shape[0]
    tokens = torch.full((rows,), -9, device="cuda", dtype=torch.int32)
    logs = torch.full((rows,), 9.0, device="cuda")
    L.sample_tokens_device(ctx, logits, u, tokens, logs, temperature, top_k, top_p, min_p)
    ctx.synchronize()

    def at(x, i):
        return float(x[i]) if hasattr(x, "data_ptr") else x
    got, got_logs = tokens.cpu().numpy(), logs.double().cpu().numpy()
    x, uu = logits.double().cpu().numpy(), u.double().cpu().numpy()
    for i in range(rows):
        want, log = definition(x[i], uu[i], at(temperature, i), int(at(top_k, i)), at(top_p, i), at(min_p, i))
        assert got[i] == want, (i, got[i], want)
        if log == -np.inf:
            assert got_logs[i] == -np.inf
        elif check_weights:
            assert abs(got_logs[i] - log) <= 2.0 ** -24 * abs(log) * 1.01 + 2.0 ** -22, (i, got_logs[i], log)
    return tokens, logs


def logits_of(rows, vocab, dtype, seed=0, spread=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype), \
        torch.rand(rows, generator=g, device="cuda")


VOCABS = [1, 2, 7, 129, 1000, 1024, 1025, 4096, 4097, 16384, 16385, 32000, 50257, 131072, 200001, 262144]
FILTERS = [(0, 1.0, 0.0), (1, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (200, 0.8, 0.001), (3000, 0.99, 0.0),
           (0, 0.999, 0.0)]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_every_size(ctx, vocab, dtype):
    logits, u = logits_of(5, vocab, dtype, vocab)
    for top_k, top_p, min_p in FILTERS:
        run(ctx, logits, u, 0.8, top_k, top_p, min_p)


@pytest.mark.parametrize("temperature", [0.0, 0.05, 1.0, 30.0])
@pytest.mark.parametrize("spread", [0.0, 0.01, 20.0])
def test_sharp_and_flat_rows(ctx, temperature, spread):
    """All logits alike is a threshold inside thousands of ties."""
    for vocab, dtype in ((900, F32), (3000, BF16), (9000, F16), (40000, BF16)):
        logits, u = logits_of(3, vocab, dtype, 1, spread)
        for top_k, top_p, min_p in FILTERS:
            run(ctx, logits, u, temperature, top_k, top_p, min_p)


def test_ties_go_to_the_lowest_index(ctx):
    g = torch.Generator("cuda").manual_seed(2)
    for vocab in (50, 5000, 40000):
        logits = torch.randint(-3, 3, (6, vocab), generator=g, device="cuda").to(BF16)
        logits[1] = -0.0
        logits[1, ::2] = 0.0  # the two zeros are alike
        u = torch.rand(6, generator=g, device="cuda")
        for top_k, top_p, min_p in FILTERS + [(17, 0.5, 0.0), (0, 0.25, 0.0), (vocab // 2, 0.5, 0.0)]:
            run(ctx, logits, u, 1.0, top_k, top_p, min_p)


@pytest.mark.parametrize("many", [131072, 262044])
@pytest.mark.parametrize("step", [3, 40])
def test_many_tokens_in_one_bin_of_a_large_vocabulary(ctx, many, step):
    """The most tokens there can be at one logit below a hundred larger ones, at temperatures where it is the first of
    its bin: a bin's mass is the largest that it can be."""
    x = torch.full((12, 262144), -float("inf"), device="cuda")
    x[:, :many] = -float(step)
    x[:, many:many + 100] = 0.0
    # (bins are 45 / 512 powers of two: a step of the logits each, or a little less)
    temperature = torch.tensor([512 / 45 * 1.4426950408889634 * (1 - i * 2.0 ** -21) for i in range(12)], device="cuda")
    u = torch.rand(12, generator=torch.Generator("cuda").manual_seed(5), device="cuda")
    for top_p in (0.3, 0.999):
        run(ctx, x, u, temperature, 0, top_p)
    run(ctx, x, u, temperature, 60000, 0.9)


def test_random_numbers_at_the_edges(ctx):
    for vocab in (5, 3000, 20000):
        logits, _ = logits_of(8, vocab, F32, 3)
        u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, 2.0 ** -149, 0.5, float("-inf")], device="cuda")
        for top_k, top_p, min_p in FILTERS:
            run(ctx, logits, u, 1.0, top_k, top_p, min_p)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_masked_rows_infinities_and_nan(ctx, dtype):
    inf, low = float("inf"), torch.finfo(dtype).min
    for vocab in (40, 2000, 20000):
        logits, u = logits_of(10, vocab, dtype, 4)
        logits[0] = -inf
        logits[1] = float("nan")
        logits[2, 1:] = -inf
        logits[3, : vocab - 1] = low
        logits[4] = low
        logits[5, 7] = float("nan")
        logits[6, 3] = inf
        logits[7, 3] = logits[7, 30] = inf
        logits[8, ::3] = -inf
        logits[9, ::2] = float("nan")
        logits[9, 1::2] = -inf
        for top_k, top_p, min_p in FILTERS:
            run(ctx, logits, u, 0.7, top_k, top_p, min_p)


def test_parameters_of_each_row(ctx):
    nan = float("nan")
    temperature = torch.tensor([1.0, 0.0, -2.0, nan, 0.3, 5.0, 1.0, 1.0], device="cuda")
    top_k = torch.tensor([0, 5, 0, 9, -4, 10 ** 9, 1, 40], device="cuda", dtype=torch.int32)
    top_p = torch.tensor([0.9, 0.5, 1.0, 0.5, 1.5, 0.8, 0.0, -1.0], device="cuda")
    min_p = torch.tensor([0.0, 0.1, 0.2, 0.0, -1.0, 0.01, 1.0, 2.0], device="cuda")
    for vocab in (300, 30000):
        logits, u = logits_of(8, vocab, F32, 5)
        tokens, _ = run(ctx, logits, u, temperature, top_k, top_p, torch.clamp(min_p, max=1.0))
        again = torch.empty_like(tokens)
        L.sample_tokens_device(ctx, logits, u, again, None, temperature, top_k, top_p, min_p)
        top_p[0] = nan  # keeps all
        run(ctx, logits, u, temperature, top_k, torch.nan_to_num(top_p, nan=1.0), min_p.clamp(max=1.0))
        assert torch.equal(tokens, again)
        L.sample_tokens_device(ctx, logits, u, again, None, temperature, top_k, top_p, min_p)
        want, _ = run(ctx, logits, u, temperature, top_k, torch.nan_to_num(top_p, nan=1.0), min_p.clamp(max=1.0))
        assert torch.equal(want, again)
        top_p[0] = 0.9


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_any_stride_and_alignment(ctx, dtype):
    for vocab, width, skip in ((100, 131, 3), (5000, 5003, 1), (33000, 33008, 8)):
        big, u = logits_of(4, width, dtype, 6)
        run(ctx, big[:, skip:skip + vocab], u, 1.0, 30, 0.9, 0.0)
        one = logits_of(1, vocab, dtype, 7)[0].expand(4, vocab)  # the same row four times
        run(ctx, one, u, 1.0, 0, 0.9, 0.01)


def test_nothing_else_is_written_and_calls_repeat(ctx):
    logits, u = logits_of(33, 20000, BF16, 8)
    before = logits.clone()
    tokens, logs = torch.full((40,), -9, device="cuda", dtype=torch.int32), torch.full((40,), 9.0, device="cuda")
    seen = []
    for _ in range(4):
        L.sample_tokens_device(ctx, logits, u, tokens[3:36], logs[3:36], 0.9, 0, 0.95, 0.001)
        seen.append((tokens.clone(), logs.clone()))
    ctx.synchronize()
    assert all(torch.equal(a, seen[0][0]) and torch.equal(b, seen[0][1]) for a, b in seen)
    assert (tokens[:3] == -9).all() and (tokens[36:] == -9).all() and (logs[36:] == 9.0).all()
    assert torch.equal(before, logits)


def test_captured_calls_replay(ctx):
    logits, u = logits_of(7, 40000, F32, 9)
    tokens, logs = torch.empty(7, device="cuda", dtype=torch.int32), torch.empty(7, device="cuda")
    L.sample_tokens_device(ctx, logits, u, tokens, logs, 1.0, 50, 0.9)
    ctx.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        L.sample_tokens_device(ctx, logits, u, tokens, logs, 1.0, 50, 0.9)
    other, v = logits_of(7, 40000, F32, 10)
    logits.copy_(other)
    u.copy_(v)
    graph.replay()
    got = tokens.clone()
    want, _ = run(ctx, logits, u, 1.0, 50, 0.9)
    assert torch.equal(got, want)
    del graph


def test_shares_of_many_draws(ctx):
    """Evenly spaced random numbers draw each token as often as its probability says, to one draw."""
    n, vocab = 4096, 37
    logits = logits_of(1, vocab, F32, 11)[0]
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens = torch.empty(n, device="cuda", dtype=torch.int32)
    L.sample_tokens_device(ctx, logits.expand(n, vocab), u, tokens, None, 1.5)
    p = torch.softmax(logits[0].double() / 1.5, 0)
    count = torch.bincount(tokens.long(), minlength=vocab).double()
    assert ((count - n * p).abs() <= 1.0 + 1e-6).all()
