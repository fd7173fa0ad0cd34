"""Linear attention where a call could go wrong unseen: values that are not
finite in the first chunk of many blocks at once."""
import pytest

import lewm_b200 as L
from test_gpu_linear import BF16, DECAYS, F16, close, gen, ints, randn, recurrence, tolerances

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
