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
