"""Shared prefixes at their edges: groups that share nothing."""
import pytest

import lewm_b200 as L
from test_gpu_blocks import gen, randn
from test_gpu_shared import Groups, POOLS

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


@pytest.mark.parametrize("dtype,codes", POOLS)
@pytest.mark.parametrize("max_tail,window", [(60, 0), (200, 0), (0, 60)])
def test_tokens_before_the_first_cached_one(ctx, dtype, codes, max_tail, window):
    """A group without a prefix, beside one with: its sequences may have more new tokens than cached ones, as in the
    plain attention, and what lies before the first cached token sees nothing."""
    g = Groups(50, [(0, [1, 5, 2, 40]), (64, [3, 9])], 16, 2, 64, dtype, codes)
    for news in ([2, 1, 2, 2, 1, 2], [1, 1, 1, 1, 1, 1], [2, 5, 6, 3, 3, 4]):
        for heads in (2, 4):
            q = randn(gen(51), sum(news) + 3, heads, 64, dtype=dtype)
            _, out = g.call(ctx, news, heads, q=q, max_tail=max_tail, max_length=64, window=window)
            assert news[0] == 1 or (out[:news[0] - 1] == 0).all()
            if news[2] == 6:
                at = news[0] + news[1]
                assert (out[at:at + 4] == 0).all()
