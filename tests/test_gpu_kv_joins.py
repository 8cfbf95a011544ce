"""The 4-bit KV cache attention where it is joined from parts, and where its inputs are uneven: against the definition in float64.

The plan cuts keys over CTAs for long caches of few rows (dealt blocks, one launch more) and for long caches of many rows (splits);
the sizes here reach both on 148 SMs, which the workspace's size shows."""
import math

import pytest
import torch

from kv_helpers import U_BF16, U_FP16, Batch, check, stored
from moelab_b200 import _lib, ops

pytestmark = pytest.mark.gpu

FMTS = ("q4", "mxfp4")


def attend(b, c, **kw):
    kw.setdefault("max_q", max([1] + list(b.rows)))
    return ops.kv_attention(b.q, c, b.table, b.lens_t, cu=b.cu, **kw)


def reference(b, scale=None, window=0, sinks=0, sink_logits=None, steep=False):
    """(y, bound, lse) in float64, and per row only from what the row sees.

    The bound, with A = sum_j p_j |v_j| over the softmax's weights p: the result is rounded to bf16 (2^-8 of it). Values may be
    rounded to fp16 (2^-11 of A); so may weights, times A again with MXFP4 (codes are exact), and for int4 times
    sum_j p_j 2 max_group |v_j|, as a weight scales s code <= 15 s and s <= 2 / 15 of the group's largest magnitude. A key may be
    rounded to fp16, which moves its score by 2^-11 |scale| sum |q| |k|; the score's own sums are fp32, for int4 over terms as
    large as the group's largest |k| (2^-20 of sum_g |q|_1 2 max_group |k|, two dozen roundings of 2^-24). A score moved by e
    moves the weighted mean by 2 e A at most. fp32 sums and exponentials: 2^-15 of A.

    steep: scores so far apart that weights become fp16 subnormals, whose roundings are 2^-25 and not relative. With many rows the
    weights are 2^6 times p / max p or more, so a key's is off by 2^-31 max p; with few they are scaled by the values' power of
    two, which puts the largest scale so far at 2^8 or more, so weight times value is off by 2^-33 max p max |v| 6 at most (codes
    of E2M1 up to 6; int4's are 15 times their scale and those 2 / 15 max |v|). Over n keys: n 2^-30 max p max |v| covers both.
    It shows in values that the row's heaviest keys have as zero."""
    scale = b.D ** -0.5 if scale is None else scale
    G = b.H // b.Hkv
    y = torch.zeros(b.T, b.H, b.D, dtype=torch.float64)
    bound, lse = torch.zeros_like(y), torch.full((b.T, b.H), -math.inf, dtype=torch.float64)
    ks, vs = (stored(x, b.fmt).double().to(b.device) for x in (b.k, b.v))
    gs = 64 if b.fmt == "q4" else 32
    group = lambda x: x.abs().nan_to_num().unflatten(-1, (-1, gs)).amax(-1, keepdim=True).expand(-1, -1, gs).flatten(1)
    q, at = b.q.double(), 0
    for s, (L, n) in enumerate(zip(b.lens, b.rows)):
        pos, key = torch.arange(L - n, L, device=b.device), torch.arange(max(L, 0), device=b.device)
        see = key[None] <= pos[:, None]
        if window:
            see &= (key[None] > pos[:, None] - window) | (key[None] < sinks)
        for h in range(b.H):
            kk, vv, qq = ks[s, :L, h // G], vs[s, :L, h // G], q[at:at + n, h]
            e = (U_FP16 * qq.abs() @ kk.abs().nan_to_num().T + 2.0 ** -19 * qq.abs() @ group(kk).T) * abs(scale)
            e = e.masked_fill(~see, 0.0).amax(-1, keepdim=True) if L else torch.zeros(n, 1, device=b.device, dtype=torch.float64)
            x = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
            if sink_logits is not None:
                x = torch.cat([x, sink_logits[h].double().to(b.device).expand(n, 1)], -1)
            if x.shape[1] == 0:
                continue
            m = x.amax(-1, keepdim=True)
            m = torch.where(m == -math.inf, 0.0, m)
            p = torch.exp(x - m)
            tot = p.sum(-1, keepdim=True)
            p = (p / torch.where(tot == 0, 1.0, tot))[:, :L]
            seen = lambda v: torch.where((p != 0)[:, :, None], p[:, :, None] * v[None], 0.0).sum(1) if v.isnan().any() else p @ v
            out, A = seen(vv), p @ vv.abs().nan_to_num()
            Ap = p @ group(vv) * 2 if b.fmt == "q4" else A
            if steep:
                Ap = Ap + see.sum(-1, keepdim=True) * 2.0 ** -30 / U_FP16 * p.amax(-1, keepdim=True) * vv.abs().max()
            y[at:at + n, h] = out.cpu()
            bound[at:at + n, h] = (U_BF16 * out.abs() + ((2 * e + U_FP16 + 2.0 ** -15) * A + U_FP16 * Ap) * (1 + U_BF16)).cpu() + 1e-36
            lse[at:at + n, h] = (m + torch.log(tot)).squeeze(-1).cpu()
        at += n
    return y, bound, lse


def within(y, ref, bound, what=""):
    y = y.double().cpu()
    assert torch.isfinite(y).all(), what
    off = (y - ref).abs() - bound
    assert (off <= 0).all(), (what, int((off > 0).sum()), (off / bound).max().item(), (off > 0).nonzero()[:4].tolist())


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


# ------------------------------------------------------------------ keys and values of sizes far apart
@pytest.mark.parametrize("fmt,D", [("q4", 64), ("q4", 128), ("mxfp4", 64), ("mxfp4", 128)])
@pytest.mark.parametrize("n,L", [(1, 300), (3, 300), (3, 9000), (150, 257), (150, 300), (150, 9000)])
@pytest.mark.parametrize("what", ("key", "value", "unattended", "first"))
@pytest.mark.parametrize("power", (13, 17, 19, 30, 60, 96))
def test_sizes_far_apart(fmt, D, n, L, what, power):
    """A key or value 2^power times the others' size that some rows do not see (the last token's) or give no weight (a token with
    a score far below the rest), or others that are that much larger than the first token's, the only one that row 0 sees: the
    other rows' results are as accurate as without it."""
    if what == "first":
        L = n
    b = Batch([L], [n], 4, 1, D, fmt, page=32, seed=53)
    far = 2.0 ** power
    rows = torch.arange(n)
    if what == "key":
        b.k[0, L - 1] = (b.k[0, L - 1].float() * far).to(torch.bfloat16)
        rows = rows[:-1]  # the last row's scores are that large too
    elif what == "value":
        b.v[0, L - 1] = (b.v[0, L - 1].float() * far).to(torch.bfloat16)
    elif what == "unattended":
        b.q = b.q.abs()
        b.k[0, 5] = -14.0 * (128 / D) ** 0.5  # weight below 2^-100
        b.v[0, 5] = (b.v[0, 5].float() * far).to(torch.bfloat16)
    else:
        b.v[0, 0] = (b.v[0, 0].float() / far).to(torch.bfloat16)
        b.k[0, 0] = (b.k[0, 0].float() / far).to(torch.bfloat16)
    c = b.cache(ops)
    y, lse = attend(b, c, return_lse=True)
    ref, bound, lref = reference(b)
    if len(rows):
        within(y[rows], ref[rows], bound[rows])
        assert (lse[rows].double().cpu() - lref[rows]).abs().max() < 5e-3
    assert c.read_error() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (1, 3, 150))
def test_sizes_far_apart_in_window_and_batch(fmt, n):
    """The same beside windows, first tokens, sink logits and ordinary sequences, NaN where no row looks; the calls repeat."""
    b = Batch([700, 9000, 431], [n, n, n], 8, 2, 64, fmt, page=16, seed=54, pad=2)
    b.v[1, 8990, 0] = (b.v[1, 8990, 0].float() * 2.0 ** 40).to(torch.bfloat16)
    b.v[2, 0] = (b.v[2, 0].float() * 2.0 ** -30).to(torch.bfloat16)
    b.k[0, 690, 1] = 0.0
    b.v[0, 100] = math.nan  # out of the window of every row
    logits = torch.linspace(-3, 3, 8, device="cuda")
    c = b.cache(ops)
    ref, bound, lref = reference(b, window=380, sinks=3, sink_logits=logits)
    out = torch.full((b.T, 8, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    y, lse = attend(b, c, window=380, sinks=3, sink_logits=logits, return_lse=True, out=out)
    within(y[:-2], ref[:-2], bound[:-2])
    assert (y[-2:] == 9).all()
    assert (lse[:-2].double().cpu() - lref[:-2]).abs().max() < 5e-3
    assert torch.equal(attend(b, c, window=380, sinks=3, sink_logits=logits)[:-2], y[:-2])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("n,L", [(1, 300), (3, 9000), (150, 300), (150, 9000)])
@pytest.mark.parametrize("size", (2.0 ** 10, -2.0 ** 16, 2.0 ** 20, -2.0 ** 60, 2.0 ** 100))
def test_scores_of_any_size_pick_the_largest(fmt, D, n, L, size):
    """Keys of one value each, from 1 to 8 or -1 to -8, one of them larger: the scores differ by at least `size` and more than
    their rounding, so the result is that key's value."""
    b = Batch([L], [n], 4, 1, D, fmt, page=32, seed=55)
    g = torch.Generator().manual_seed(7)
    best = min(L - n, 130)
    k = torch.randint(1, 9, (L,), generator=g).float()
    k[best] = 12.0
    b.k[0, :, 0] = (k * (1 if size > 0 else -1))[:, None].to(torch.bfloat16)
    b.q[:] = size
    c = b.cache(ops)
    y, lse = attend(b, c, return_lse=True)
    want = stored(b.v, fmt)[0, best, 0].double()
    assert torch.isfinite(y).all()
    assert ((y.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * want.abs().max()).all()
    top = 12.0 * abs(size) * D ** 0.5
    assert ((lse.double() - top).abs() <= 2.0 ** -20 * top).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (1, 3, 150))
@pytest.mark.parametrize("power", (121, 126, -119, -124))
def test_queries_at_the_ends_of_the_range(fmt, n, power):
    """Queries of 2^power and keys that make ordinary scores of them, where the cache has such keys (int4's are zero below 2^-24,
    then all weights are the same); rows of zeros beside them, and with 2^126 times more than 4 an infinite query, whose row is NaN.
    The scale's half of the exponents is a user's to choose too."""
    b = Batch([300], [n], 4, 2, 64, fmt, page=32, seed=56)
    b.k = (b.k.float() * 2.0 ** -power).to(torch.bfloat16)
    b.q = (b.q.float() * 2.0 ** power).to(torch.bfloat16)
    b.q[0, 0] = 0.0
    c = b.cache(ops)
    ref, bound, lref = reference(b)
    y, lse = attend(b, c, return_lse=True)
    fine = torch.isfinite(b.q).all(-1).cpu()
    within(y.cpu()[fine], ref[fine], bound[fine])
    assert (lse.double().cpu() - lref)[fine].abs().max() < 5e-3
    assert y.cpu()[~fine].isnan().all() and lse.cpu()[~fine].isnan().all()
    b.k = (b.k.float() * 2.0 ** power).to(torch.bfloat16)
    c = b.cache(ops)
    if abs(power) < 120:  # the scale is a normal fp32 number
        ref, bound, lref = reference(b, scale=2.0 ** -power / 8)
        within(attend(b, c, scale=2.0 ** -power / 8), ref, bound)


# ------------------------------------------------------------------ joined parts
def joined(b, **kw):
    """The call's workspace: parts are joined where it is not empty."""
    return _lib.load().moeb_kv_attention_workspace_bytes(b.T, len(b.lens), b.table.shape[1], b.page, b.H, b.Hkv, b.D, max(b.rows),
                                                        kw.get("window", 0), kw.get("sinks", 0), 1) > 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("n", (1, 4, 90))
@pytest.mark.parametrize("kw", [dict(), dict(window=5000), dict(window=5000, sinks=4), dict(window=5003, sinks=300),
                                dict(window=4700, sinks=4000)])
def test_joined_parts(fmt, D, n, kw):
    """Long caches, whose keys several CTAs share: windows and first tokens (a part may end or begin between them), sink logits, lse,
    a sequence that begins inside the call's rows."""
    b = Batch([9100, n, 12007], [n] * 3, 8, 1 if n == 90 else 2, D, fmt, page=64, seed=60, peak=2.0)
    c = b.cache(ops)
    assert joined(b, **kw)
    ref, bound, lref = reference(b, **kw)
    y, lse = attend(b, c, return_lse=True, **kw)
    within(y, ref, bound)
    assert (lse.double().cpu() - lref).abs().max() < 5e-3
    logits = torch.linspace(-4, 9, 8, device="cuda")
    logits[2] = -math.inf
    ref, bound, lref = reference(b, sink_logits=logits, **kw)
    y, lse = attend(b, c, return_lse=True, sink_logits=logits, **kw)
    within(y, ref, bound)
    assert (lse.double().cpu() - lref).abs().max() < 5e-3
    if n > 1:  # rows before the second sequence's start
        lens = b.lens_t.clone()
        lens[1] = n - 2
        y2, lse2 = ops.kv_attention(b.q, c, b.table, lens, cu=b.cu, max_q=n, return_lse=True, sink_logits=logits, **kw)
        assert torch.equal(y2[:n], y[:n]) and torch.equal(y2[2 * n:], y[2 * n:]) and torch.equal(lse2[2 * n:], lse[2 * n:])
        # lse is the logit times log2(e) and back times ln(2): two rounded constants and two rounded products, 2^-24 each
        assert not y2[n:n + 2].any() and torch.allclose(lse2[n:n + 2], logits.expand(2, 8), rtol=2 ** -22, atol=0)
    assert c.read_error() == 0


@pytest.mark.parametrize("fmt,D", [("q4", 128), ("mxfp4", 64), ("mxfp4", 128)])  # rows of more than one group
@pytest.mark.parametrize("n", (1, 3, 130))
def test_nan_through_joined_parts(fmt, D, n):
    """A NaN value makes its group NaN in the rows that see it, a NaN key the whole row, through the joins; other rows, heads and
    groups are as without."""
    gs = 64 if fmt == "q4" else 32
    b = Batch([9000, 8200], [n, n], 4, 2, D, fmt, page=64, seed=61)
    assert joined(b)
    ref, bound, _ = reference(b)
    b.v[0, 4000, 0, 3] = math.nan             # every row of the first sequence, heads 0 and 1
    b.v[1, 8200 - 1, 1, gs] = math.inf        # the last row of the second, heads 2 and 3
    b.k[1, 8200 - 1, 0, 1] = math.nan         # the last row, heads 0 and 1
    c = b.cache(ops)
    y = attend(b, c).cpu()
    nan = torch.zeros(2 * n, 4, D, dtype=torch.bool)
    nan[:n, :2, :gs] = True
    nan[2 * n - 1, 2:, gs:2 * gs] = True
    nan[2 * n - 1, :2] = True
    assert torch.equal(y.isnan(), nan)
    within(y[~nan], ref[~nan], bound[~nan])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("n,L", [(1, 300), (3, 9000), (150, 300), (90, 9000)])
@pytest.mark.parametrize("scale", (-0.2, 0.0, -1e-3, 1.5))
def test_scales_of_any_sign(fmt, D, n, L, scale):
    b = Batch([L, n], [n, n], 4, 1, D, fmt, page=32, seed=62, peak=0.5)
    c = b.cache(ops)
    ref, bound, lref = reference(b, scale=scale, steep=True)
    y, lse = attend(b, c, scale=scale, return_lse=True)
    within(y, ref, bound)
    assert (lse.double().cpu() - lref).abs().max() < 5e-3


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("far", (False, True))
@pytest.mark.parametrize("n,L", [(1, 300), (3, 300), (3, 9000), (150, 300), (150, 9000)])
def test_results_over_the_queries(fmt, far, n, L):
    """out may be q itself."""
    b = Batch([L, L + 70], [n, n], 4, 1, 128, fmt, page=32, seed=63)
    if far:
        b.v[:, 40] = (b.v[:, 40].float() * 2.0 ** 40).to(torch.bfloat16)
    c = b.cache(ops)
    want = attend(b, c)
    q = b.q.clone()
    y = ops.kv_attention(q, c, b.table, b.lens_t, cu=b.cu, max_q=n, out=q)
    assert y is q and torch.equal(y, want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (1, 150))
def test_a_captured_call_follows_values_that_come_to_be_far_apart(fmt, n):
    b = Batch([9000, 300], [n, n], 4, 1, 64, fmt, page=32, seed=64)
    c = b.cache(ops)
    attend(b, c)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = attend(b, c)
    for power in (0, 50, 0):
        k, v = b.k.clone(), b.v.clone()
        b.v[:, 290] = (b.v[:, 290].float() * 2.0 ** power).to(torch.bfloat16)
        fresh = b.cache(ops)
        for name in ("kq", "ks", "vq", "vs"):
            getattr(c, name).copy_(getattr(fresh, name))
        g.replay()
        torch.cuda.synchronize()
        ref, bound, _ = reference(b)
        within(y, ref, bound, power)
        assert torch.equal(y, attend(b, fresh))
        b.k, b.v = k, v
