"""The 4-bit KV cache attention where it is joined from parts, and where its inputs are uneven: against the definition in float64.

The plan cuts keys over CTAs for long caches of few rows (dealt blocks, one launch more) and for long caches of many rows (splits);
the sizes here reach both on 148 SMs, which the workspace's size shows."""
import math

import pytest
import torch

from kv_helpers import Batch, check
from moelab_b200 import _lib, ops

pytestmark = pytest.mark.gpu

FMTS = ("q4", "mxfp4")


def attend(b, c, **kw):
    kw.setdefault("max_q", max([1] + list(b.rows)))
    return ops.kv_attention(b.q, c, b.table, b.lens_t, cu=b.cu, **kw)


# ------------------------------------------------------------------ queries that are not finite
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (3, 150))
@pytest.mark.parametrize("split", (False, True))
def test_queries_that_see_nothing_are_not_looked_at(fmt, n, split):
    """NaN and infinities in the rows before a sequence's start: zeros like any row that sees nothing."""
    L = 9000 if split else 300
    b = Batch([n - 2, L], [n - 2, n], 4, 1, 128, fmt, page=64, seed=51)
    c = b.cache(ops)
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    q = torch.cat([torch.full((2, 4, 128), math.nan, dtype=torch.bfloat16, device="cuda"), b.q])
    q[1, :, 5:] = math.inf
    ref, bound, _ = b.reference()
    for sink in (None, torch.full((4,), 0.5, device="cuda")):
        y, lse = ops.kv_attention(q, c, b.table, b.lens_t, cu=cu, max_q=n, sink_logits=sink, return_lse=True)
        assert not y[:2].any()
        assert (lse[:2] == (-math.inf if sink is None else 0.5)).all()
        if sink is None:
            check(y[2:], ref, bound)
