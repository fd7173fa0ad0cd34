"""Offsets beyond 32 bits: pages at the end of a large pool, rows and state
slots far apart, rows of logits far apart."""
import pytest

import lewm_b200 as L
from test_gpu_blocks import gen, ints, randn
from test_gpu_linear import DECAYS, close, recurrence, tolerances
from test_gpu_sample import run
from test_gpu_shared import Groups

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("heads,news", [(4, [1, 1]), (16, [1, 1]), (4, [3, 2])])
def test_shared_pages_at_the_end_of_a_large_pool(ctx, codes, heads, news):
    g = Groups(31, [(300, [9, 3])], 64, 4, 128, BF16, codes)
    c = g.c
    n, total = c.k.shape[0], 2 ** 32 // (4 * 64 * 128) + c.k.shape[0]
    for name in ("k", "v", "ks", "vs"):
        small = getattr(c, name)
        if small is not None:
            large = torch.empty((total,) + small.shape[1:], device="cuda", dtype=small.dtype)
            bits = (lambda t: t.view(torch.uint8)) if codes and small.dim() == 4 else (lambda t: t)
            bits(large)[total - n:] = bits(small)
            setattr(c, name, large)
    c.table[c.table >= 0] += total - n
    c.cache = L.PagedCache(c.k, c.v, c.ks, c.vs, dtype=BF16)
    g.call(ctx, news, heads)


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (F16, 64)])
def test_linear_rows_far_apart(ctx, dtype, d):
    g, h, n = gen(32), 2, 2300
    wide = torch.empty(n, 1 << 20, device="cuda", dtype=dtype)
    q, k, v, out = (wide[:, i * h * d:(i + 1) * h * d].view(n, h, d) for i in range(4))
    for x in (q, k, v):
        x.copy_(randn(g, n, h, d, dtype=dtype))
    out.fill_(7.0)
    a = DECAYS["mild"](h).cuda().float()
    states = torch.zeros(1, h, d, d, device="cuda")
    for news in ([n], [1, n - 9]):
        s = len(news)
        starts = ints([0] + [sum(news[:i + 1]) for i in range(s)])
        b = L.StateBatch(states, starts, n, max(news), source=ints([-1] * s), target=ints([-1] * (s - 1) + [0]))
        L.linear_attention_device(ctx, b, q, k, v, out, a)
        ctx.synchronize()
        want, mag, after, sizes = recurrence(q, k, v, a, news, torch.zeros(s, h, d, d, device="cuda"), d ** -0.5)
        tol, state_tol = tolerances(dtype, d, max(news), a, want, mag, sizes, False)
        m = sum(news)
        close(out[:m], want[:m], tol[:m])
        close(states, after[-1:], state_tol[-1:])


@pytest.mark.parametrize("new", [1, 70, 700])
def test_state_slots_far_apart(ctx, new):
    g, h, d, slots = gen(33), 4, 64, 140000
    states = torch.empty(slots, h, d, d, device="cuda")
    states[-1] = randn(g, h, d, d)
    before = states[-1:].clone()
    q, k, v = (randn(g, new, h, d, dtype=BF16) for _ in range(3))
    out = torch.empty_like(q)
    a = DECAYS["mild"](h).cuda().float()
    b = L.StateBatch(states, ints([0, new]), new, source=ints([slots - 1]), target=ints([slots - 2]))
    L.linear_attention_device(ctx, b, q, k, v, out, a)
    ctx.synchronize()
    want, mag, after, sizes = recurrence(q, k, v, a, [new], before, d ** -0.5)
    tol, state_tol = tolerances(BF16, d, new, a, want, mag, sizes, new <= 8)
    close(out, want, tol)
    close(states[-2:-1], after, state_tol)
    assert torch.equal(states[-1:], before)


@pytest.mark.parametrize("vocab,top_k", [(1000, 0), (40000, 0), (200000, 50)])
def test_rows_of_logits_far_apart(ctx, vocab, top_k):
    g = gen(34)
    wide = torch.empty(20, 1 << 28, device="cuda", dtype=BF16)
    logits = wide[:, :vocab]
    logits.copy_(randn(g, 20, vocab, dtype=BF16) * 3)
    run(ctx, logits, torch.rand(20, generator=g, device="cuda"), 0.9, top_k, 0.9)
