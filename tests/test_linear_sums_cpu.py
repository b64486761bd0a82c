"""What the exact sums of the linear layer's GPU tests see: a lost step of rows changes
the gradients of the weights at each of their sizes.  No GPU."""
from __future__ import annotations

import pytest

import linear_exact as exact
from linear_sizes import ONE_PASS, RESIDENT, STREAMED
from test_gpu_linear_sums import SEED
from test_gpu_nn import DTYPES, IDS
import torch


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,inner,outer", [s for s in ONE_PASS + RESIDENT + STREAMED if s[0] * max(s[1:]) < 7_000_000])
def test_a_lost_step_shows(dtype, rows, inner, outer):
    """A step of the pass over rows (64 of them in 16-bit types, 32 in float32): the
    first, one in the middle, the last whole one and what is left."""
    x, w, dy, z = exact.operands(rows, inner, outer, SEED)
    step = 32 if dtype is torch.float32 else 64
    for act in (None, "silu"):
        _, dw, db = exact.gradients(x, w, dy, z, act)
        for first in {0, rows // step // 2 * step, max(rows // step - 1, 0) * step, (rows - 1) // step * step}:
            part = slice(first, first + step)
            _, dw_part, db_part = exact.gradients(x[part], w, dy[part], z[part], act)
            changed = [not torch.equal(exact.rounded(t, dtype), exact.rounded(t - p, dtype))
                       for t, p in ((dw, dw_part), (db, db_part))]
            assert any(changed), (first, act)
