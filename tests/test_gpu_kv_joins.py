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


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,L", [(1, 1), (1, 3), (3, 300), (2, 9000), (150, 300)])
@pytest.mark.parametrize("bad", (math.inf, -math.inf, math.nan))
def test_queries_that_are_not_finite_give_nan_and_touch_no_other_row(fmt, n, L, bad):
    """inf - inf is in every softmax of such a row, over one key as well, whatever the sign of its scores."""
    b = Batch([L, L + 5], [n, n], 4, 2, 64, fmt, page=16, seed=52)
    c = b.cache(ops)
    ref, bound, _ = b.reference()
    b.q[n - 1, 1, 7] = bad
    y, lse = attend(b, c, return_lse=True)
    assert y[n - 1, 1].isnan().all() and lse[n - 1, 1].isnan()
    rest = torch.ones(2 * n, 4, dtype=torch.bool)
    rest[n - 1, 1] = False
    check(y.cpu()[rest], ref[rest], bound[rest])
