"""The 4-bit KV cache and attention over it against the oracle's quantizers (bit-exact) and float64 attention."""
import math

import pytest
import torch

from kv_helpers import Batch, check, stored
from moelab_b200 import _lib, ops

pytestmark = pytest.mark.gpu

FMTS = ("q4", "mxfp4")


def attend(b, c, **kw):
    kw.setdefault("max_q", max([1] + list(b.rows)))
    return ops.kv_attention(b.q, c, b.table, b.lens_t, cu=b.cu, **kw)


# ------------------------------------------------------------------ writing and reading
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("lens,page,Hkv", [([1], 16, 1), ([17, 1, 64, 0, 33], 16, 3), ([130, 5], 64, 8), ([300], 128, 2)])
def test_write_then_read_is_the_oracles_quantization(fmt, D, lens, page, Hkv):
    b = Batch(lens, lens, Hkv, Hkv, D, fmt, page=page, seed=len(lens))
    c = b.cache(ops)
    k, v = ops.kv_read(c, b.table, b.cu, b.T)
    for got, w in ((k, b.k), (v, b.v)):
        assert torch.equal(got.cpu(), b.flat(stored(w, fmt)).to(torch.bfloat16).cpu())
    assert c.read_error() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_extreme_rows(fmt):
    """Zero groups, one value, subnormals, the largest values, both signs of zero, ties of the codes: bit for bit."""
    D = 128
    rows = [torch.zeros(D), torch.full((D,), 5.0), torch.full((D,), -3.0), torch.arange(D).float() - 64, torch.full((D,), 1e-39),
            torch.linspace(-1e38, 1e38, D), torch.linspace(0, 7.875, D), -torch.linspace(0, 7.875, D), torch.full((D,), -0.0),
            torch.linspace(3e38, 3.3e38, D), torch.linspace(-1e-30, 1e-30, D)]
    g = torch.Generator().manual_seed(1)
    rows += [torch.randint(-48, 49, (D,), generator=g) / 8.0 for _ in range(40)]  # many ties
    w = torch.stack(rows).to(torch.bfloat16).view(-1, 1, D)
    n = w.shape[0]
    c = ops.KVCache(8, 1, D, page_size=16, fmt=fmt)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
    ops.kv_write(c, w.cuda(), w.flip(0).cuda(), table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    k, v = ops.kv_read(c, table, None, n)
    ref = stored(w, fmt).to(torch.bfloat16)
    assert torch.equal(k.cpu().view(torch.int16), ref.view(torch.int16))
    assert torch.equal(v.cpu().view(torch.int16), ref.flip(0).view(torch.int16))


@pytest.mark.parametrize("fmt", FMTS)
def test_many_rows_are_the_oracles_quantization(fmt):
    """16,000 groups and more of each kind, from 2^-60 to 2^60: normal, all of one sign, around a large middle, small integers
    (codes that lie on a half all the time)."""
    g = torch.Generator().manual_seed(11)
    w = torch.randn(2048, 8, 128, generator=g)
    w[1::4] = w[1::4].abs()
    w[2::4] += 30 * torch.randn(512, 8, 1, generator=g)
    w[3::4] = torch.randint(-128, 129, (512, 8, 128), generator=g).float()
    w = (w * torch.exp2(torch.randint(-60, 61, (2048, 8, 1), generator=g).float())).to(torch.bfloat16)
    c = ops.KVCache(32, 8, 128, page_size=64, fmt=fmt)
    table = torch.arange(32, dtype=torch.int32, device="cuda").view(1, 32)
    ops.kv_write(c, w.cuda(), w.flip(0).cuda(), table, torch.tensor([2048], dtype=torch.int32, device="cuda"))
    k, v = ops.kv_read(c, table, None, 2048)
    ref = stored(w, fmt).to(torch.bfloat16)
    assert torch.equal(k.cpu().view(torch.int16), ref.view(torch.int16))
    assert torch.equal(v.cpu().view(torch.int16), ref.flip(0).view(torch.int16))


@pytest.mark.parametrize("fmt", FMTS)
def test_group_with_a_nan_reads_back_as_nan_alone(fmt):
    D, gs = 128, 64 if fmt == "q4" else 32
    w = torch.randn(4, 2, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    bad = w.clone()
    bad[1, 0, 3], bad[2, 1, D - 1], bad[3, 0, gs] = math.nan, math.inf, -math.inf
    c = ops.KVCache(1, 2, D, page_size=16, fmt=fmt)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    ops.kv_write(c, bad.cuda(), w.cuda(), table, torch.tensor([4], dtype=torch.int32, device="cuda"))
    k, v = (t.cpu() for t in ops.kv_read(c, table, None, 4))
    ref = stored(w, fmt).to(torch.bfloat16)
    nan = torch.zeros(4, 2, D, dtype=torch.bool)
    nan[1, 0, :gs] = nan[2, 1, D - gs:] = nan[3, 0, gs:2 * gs] = True
    assert torch.equal(k.isnan(), nan)
    assert torch.equal(k[~nan], ref[~nan]) and torch.equal(v, ref)


@pytest.mark.parametrize("fmt", FMTS)
def test_append_token_by_token_equals_one_write(fmt):
    b = Batch([37, 5, 20], [1, 1, 1], 2, 2, 64, fmt, page=16, seed=3)
    whole, c = b.cache(ops), b.cache(ops, fill=False)
    for t in range(max(b.lens)):
        at = torch.tensor([min(t + 1, n) for n in b.lens], dtype=torch.int32, device="cuda")
        rows = [[b.k, b.v][i][torch.arange(3), (at.cpu() - 1).long()].cuda() for i in range(2)]
        ops.kv_write(c, *rows, b.table, at)
    for n in ("kq", "ks", "vq", "vs"):
        assert torch.equal(getattr(c, n), getattr(whole, n)), n


def test_write_takes_views_of_a_fused_projection_and_leaves_other_rows():
    Hkv, D, T = 2, 128, 21
    qkv = torch.randn(T, (4 + 2 * Hkv) * D, device="cuda").to(torch.bfloat16)
    k, v = (qkv[:, (4 + i * Hkv) * D:(4 + (i + 1) * Hkv) * D].unflatten(1, (Hkv, D)) for i in range(2))
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([25], dtype=torch.int32, device="cuda")
    a, b = (ops.KVCache(3, Hkv, D, page_size=16) for _ in range(2))
    ops.kv_write(a, k, v, table, lens)
    ops.kv_write(b, k.contiguous(), v.contiguous(), table, lens)
    for n in ("kq", "ks", "vq", "vs"):
        assert torch.equal(getattr(a, n), getattr(b, n))
        x = getattr(a, n)
        assert not x[1].any() and not x[2, :, :4].any() and not x[0, :, 9:].any()  # positions 4 .. 24 only


def test_padding_rows_bad_pages_and_negative_positions():
    D, page = 64, 16
    c = ops.KVCache(2, 1, D, page_size=page)
    w = torch.randn(8, 1, D, device="cuda").to(torch.bfloat16)
    lens = torch.tensor([2, 40, 0], dtype=torch.int32, device="cuda")
    table = torch.tensor([[1, -1], [0, -1], [0, 0]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 3, 5, 6], dtype=torch.int32, device="cuda")  # rows 6, 7: padding
    ops.kv_write(c, w, w, table, lens, cu=cu)  # row 0 at -1; rows 3, 4 at 38, 39: outside the table; row 5 at -1
    assert c.read_error() == _lib.DEVERR_PAGE and c.read_error() == 0
    assert c.kq[1, 0, :2].any() and not c.kq[0].any() and not c.kq[1, 0, 2:].any()
    for bad in (-1, 2, 2 ** 31 - 1, -2 ** 31):
        t = torch.full((1, 1), bad, dtype=torch.int32, device="cuda")
        ops.kv_write(c, w[:1], w[:1], t, torch.ones(1, dtype=torch.int32, device="cuda"))
        assert c.read_error() == _lib.DEVERR_PAGE
    out = [torch.full((8, 1, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = ops.kv_read(c, table, cu, 8, first=torch.tensor([0, 15, -1], dtype=torch.int32, device="cuda"), out=out)
    assert c.read_error() == _lib.DEVERR_PAGE
    assert k is out[0] and (k[6:] == 7).all() and (v[6:] == 7).all()  # behind the last sequence: as they were
    assert (k[4] == 0).all() and (k[5] == 0).all() and k[0].any()
    k2, _ = ops.kv_read(c, table, cu, 8)
    assert not k2[6:].any()


def test_no_tokens():
    c = ops.KVCache(1, 1, 64, page_size=16)
    e = torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    ops.kv_write(c, e, e, table, lens)
    assert ops.kv_read(c, table, None, 0)[0].shape == (0, 1, 64)
    assert ops.kv_attention(torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda"), c, table, lens).shape == (0, 2, 64)
    y = ops.kv_attention(torch.ones(2, 2, 64, dtype=torch.bfloat16, device="cuda"), c, table, lens)
    assert not y.any()  # sequences of length zero: rows before their start see nothing
    # rows, but no sequences: all of them are behind the last one
    rows, junk = torch.ones(300, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.full((1 << 20,), 7.0, device="cuda")
    del junk
    for t, n in ((table[:0], lens[:0]),):
        assert not ops.kv_attention(rows, c, t, n).any() and not ops.kv_attention(rows, c, t, n, cu=lens[:1]).any()
        assert not ops.kv_read(c, t, None, 300)[0].any()
        ops.kv_write(c, rows[:, :1], rows[:, :1], t, n)
    assert c.read_error() == 0 and not c.kq.any()


# ------------------------------------------------------------------ attention
HEADS = [(1, 1), (4, 4), (6, 2), (32, 4), (16, 1), (40, 2), (7, 1)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("H,Hkv", HEADS)
def test_decode(fmt, D, H, Hkv):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 777]
    b = Batch(lens, [1] * len(lens), H, Hkv, D, fmt, page=16, seed=H, peak=2.0)
    c = b.cache(ops)
    y, lse = attend(b, c, return_lse=True)
    ref, bound, lref = b.reference()
    check(y, ref, bound)
    assert (lse.double().cpu() - lref).abs().max() < 5e-3
    assert torch.equal(y, ops.kv_attention(b.q, c, b.table, b.lens_t))  # cu None: one row each
    assert c.read_error() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("page", (16, 64, 256))
@pytest.mark.parametrize("H,Hkv,D,rows", [(8, 2, 128, [5, 1, 8, 3]), (8, 8, 64, [9, 2, 16, 17]), (16, 1, 64, [2, 33, 1, 4]),
                                          (4, 2, 128, [70, 128, 1, 300])])
def test_rows_of_uneven_sequences(fmt, page, H, Hkv, D, rows):
    """A few rows each (drafted tokens), prompts, single tokens, in one call; page ends inside tiles; padding rows."""
    lens = [rows[0], rows[1] + 60, rows[2] + 301, rows[3] + 129]
    b = Batch(lens, rows, H, Hkv, D, fmt, page=page, seed=page, pad=3)
    c = b.cache(ops)
    out = torch.full((b.T, H, D), 9.0, dtype=torch.bfloat16, device="cuda")
    y = attend(b, c, out=out)
    ref, bound, _ = b.reference()
    assert y is out and (y[-3:] == 9).all()
    check(y[:-3], ref[:-3], bound[:-3])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (1, 3, 200))
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (100, 4), (128, 0), (33, 70), (10000, 2), (0, 5)])
def test_window_and_first_tokens(fmt, n, window, sinks):
    b = Batch([max(n, 1), n + 64, n + 517], [n] * 3, 8, 2, 128 if window != 128 else 64, fmt, page=32, seed=window)
    c = b.cache(ops)
    y, lse = attend(b, c, window=window, sinks=sinks, return_lse=True)
    ref, bound, lref = b.reference(window=window, sinks=sinks)
    check(y, ref, bound)
    assert (lse.double().cpu() - lref).abs().max() < 5e-3


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (1, 150))
def test_sink_logits(fmt, n):
    b = Batch([n, n + 300], [n, n], 16, 2, 64, fmt, page=16, seed=5)
    c = b.cache(ops)
    logits = torch.linspace(-30, 12, 16, device="cuda")
    logits[3] = -math.inf
    y, lse = attend(b, c, sink_logits=logits, window=128, scale=0.2, return_lse=True)
    ref, bound, lref = b.reference(sink_logits=logits, window=128, scale=0.2)
    check(y, ref, bound)
    assert (lse.double().cpu() - lref).abs().max() < 5e-3


@pytest.mark.parametrize("n", (3, 40, 200))
def test_rows_before_the_start_see_nothing(n):
    """More rows than tokens: the first rows' positions are negative. Zero, and lse -inf or the sink logit."""
    b = Batch([n - 2, n + 10], [n - 2, n], 4, 2, 64, "q4", page=16, seed=6)
    c = b.cache(ops)
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    q = torch.cat([b.q[:2], b.q])
    y, lse = ops.kv_attention(q, c, b.table, b.lens_t, cu=cu, max_q=n, return_lse=True)
    ref, bound, _ = b.reference()
    assert not y[:2].any() and (lse[:2] == -math.inf).all()
    check(y[2:], ref, bound)
    sink = torch.full((4,), 0.5, device="cuda")
    y, lse = ops.kv_attention(q, c, b.table, b.lens_t, cu=cu, max_q=n, sink_logits=sink, return_lse=True)
    assert not y[:2].any() and ((lse[:2] - 0.5).abs() < 1e-6).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (1, 4, 90))
def test_long_cache(fmt, n):
    b = Batch([9001, 20, 4100], [n, min(n, 20), n], 8, 1, 128, fmt, page=64, seed=8, peak=3.0)
    c = b.cache(ops)
    ref, bound, _ = b.reference()
    check(attend(b, c), ref, bound)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", (1, 3, 130))
def test_nan_and_infinity_stay_with_the_rows_that_see_them(fmt, n):
    """Values that a row must not see (later tokens, tokens outside its window, what lies behind the end of its last page)
    may be NaN: they do not reach it. A visible NaN value makes its group NaN and no other; a visible NaN key makes the row
    NaN."""
    gs = 64 if fmt == "q4" else 32
    L = 300
    b = Batch([L, L], [n, n], 4, 1, 128, fmt, page=64, seed=9)
    v = b.v.clone()
    v[0, 100, 0, 5] = math.nan       # outside the window of every row
    v[0, L - 1, 0, 0] = math.inf     # seen by the last row only
    k = b.k.clone()
    k[1, L - 1, 0, 0] = math.nan     # seen by the last row only
    w = 64
    ref, bound, _ = b.reference(window=w)
    b.k, b.v = k, v
    c = b.cache(ops)
    # what lies behind the sequences' ends on their last pages
    for s in range(2):
        pid = int(b.table[s, L // 64])
        off = L % 64
        for par in (c.ks, c.vs):
            par[pid, :, off:] = 0x7fff7fff if fmt == "q4" else 255
        c.kq[pid, :, off:] = -1
        c.vq[pid, :, off:] = -1
    y = attend(b, c, window=w).double().cpu()
    rows = torch.ones(2 * n, dtype=torch.bool)
    rows[n - 1] = rows[2 * n - 1] = False
    # rows whose own window reaches token 100: none when n <= L - 100 - w
    assert n + 100 + w <= L
    if rows.any():
        check(y[rows], ref[rows], bound[rows])
    assert y[n - 1, :, :gs].isnan().all()
    good = y[n - 1, :, gs:]
    assert ((good - ref[n - 1, :, gs:]).abs() <= bound[n - 1, :, gs:]).all()
    assert y[2 * n - 1].isnan().all()


@pytest.mark.parametrize("n", (1, 4, 140))
def test_pages_out_of_sight_are_not_read_and_bad_pages_are_passed_over(n):
    b = Batch([400, 333], [n, n], 8, 2, 64, "q4", page=16, seed=10)
    c = b.cache(ops)
    w, s = 50, 5
    ref, bound, _ = b.reference(window=w, sinks=s)
    first_seen = [(L - n - w + 1) // 16 for L in b.lens]
    for i, p in enumerate(first_seen):
        if p > 1:
            b.table[i, 1:p] = torch.tensor([-1, 10 ** 9, -7, 2 ** 30], device="cuda", dtype=torch.int32).repeat(p)[:p - 1]
    check(attend(b, c, window=w, sinks=s), ref, bound)
    assert c.read_error() == 0
    b.table[0, 24] = b.pages  # tokens 384 .. 399 of the first sequence
    y = attend(b, c, window=w, sinks=s)
    assert c.read_error() == _lib.DEVERR_PAGE
    ref, bound, _ = b.reference(window=w, sinks=s, hole=(0, 384, 400))
    check(y, ref, bound)


@pytest.mark.parametrize("n", (1, 3, 140))
def test_lengths_beyond_the_table(n):
    """lens that name more tokens than the page table holds: those keys are not there, and the error bit says so; the rows'
    positions, and with them the others' window, are as lens has it. Lengths of garbage size end too."""
    b = Batch([256 + n], [n], 4, 2, 64, "q4", page=64, seed=40)
    c = b.cache(ops)
    assert c.read_error() == 0
    short = b.table[:, :4].contiguous()  # 256 tokens: the last n have no page
    for kw in (dict(), dict(window=n + 40, sinks=3)):
        y = ops.kv_attention(b.q, c, short, b.lens_t, **kw)
        assert c.read_error() == _lib.DEVERR_PAGE
        ref, bound, _ = b.reference(**kw, hole=(0, 256, 256 + n))
        check(y, ref, bound)
    far = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda")
    y = ops.kv_attention(b.q, c, short, far)
    assert torch.isfinite(y).all() and c.read_error() == _lib.DEVERR_PAGE
    assert not ops.kv_attention(b.q, c, short, far, window=100).any() and c.read_error() == _lib.DEVERR_PAGE
    assert not ops.kv_attention(b.q, c, short[:, :0], b.lens_t).any() and c.read_error() == _lib.DEVERR_PAGE
    ops.kv_write(c, b.new(b.k), b.new(b.v), short, far)
    assert c.read_error() == _lib.DEVERR_PAGE


@pytest.mark.parametrize("n", (1, 200))
def test_windows_and_first_tokens_of_any_size(n):
    """Bounds past the sequence are no bounds, up to the largest integers."""
    b = Batch([n + 300], [n], 4, 2, 64, "mxfp4", page=64, seed=41)
    c = b.cache(ops)
    y = attend(b, c)
    for w, s in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (n + 300, 0), (5, 2 ** 31 - 1), (5, n + 300), (2 ** 32 + 5, 0),
                 (5, 2 ** 32 + 5)):
        assert torch.equal(attend(b, c, window=w, sinks=s), y) or torch.allclose(
            attend(b, c, window=w, sinks=s).float(), y.float(), rtol=2 ** -7, atol=1e-3), (w, s)


@pytest.mark.parametrize("n", (1, 60))
def test_pages_that_sequences_share(n):
    """Two sequences with the same first pages, and one that has a page twice: read as if each had its own."""
    b = Batch([300, 300], [n, n], 8, 2, 128, "q4", page=32, seed=43)
    b.k[1, :192], b.v[1, :192] = b.k[0, :192], b.v[0, :192]
    for t in (b.k, b.v):
        t[:, 32:64] = t[:, :32]
    c = b.cache(ops)
    table = b.table.clone()
    table[1, :6] = table[0, :6]
    table[:, 1] = table[:, 0]
    ref, bound, _ = b.reference()
    check(ops.kv_attention(b.q, c, table, b.lens_t, cu=b.cu, max_q=n), ref, bound)
    k, _ = ops.kv_read(c, table, None, 600)
    assert torch.equal(k, ops.kv_read(c, b.table, None, 600)[0])


def test_more_rows_than_max_q_says():
    """A bound that is too small: the rows are left and the error word says so."""
    b = Batch([60, 70], [1, 3], 8, 1, 64, "q4", page=16, seed=42)
    c = b.cache(ops)
    out = torch.full((4, 8, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.kv_attention(b.q, c, b.table, b.lens_t, cu=b.cu, max_q=1, out=out)
    assert c.read_error() == _lib.DEVERR_ROWS
    ref, bound, _ = b.reference()
    check(out[:1], ref[:1], bound[:1])
    assert (out[1:] == 5).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("ksc,vsc,qsc", [(1e-20, 1e-20, 1e20), (1e4, 1e5, 1e-4), (1e20, 1e30, 1e-20), (1.0, 1e-30, 1.0)])
@pytest.mark.parametrize("n", (1, 150))
def test_far_magnitudes(fmt, ksc, vsc, qsc, n):
    """bf16 has fp32's range: keys, values and queries far from one, with ordinary scores, lose nothing."""
    b = Batch([300], [n], 4, 2, 64, fmt, page=16, seed=11)
    b.k, b.v, b.q = (b.k.float() * ksc).to(torch.bfloat16), (b.v.float() * vsc).to(torch.bfloat16), \
        (b.q.float() * qsc).to(torch.bfloat16)
    c = b.cache(ops)
    ref, bound, _ = b.reference()
    check(attend(b, c), ref, bound)


@pytest.mark.parametrize("n", (1, 130))
def test_uneven_magnitudes_along_a_sequence(n):
    """Values that grow and shrink by many orders along the cache: the sums keep the large ones' accuracy."""
    b = Batch([700], [n], 4, 1, 128, "q4", page=32, seed=12)
    size = torch.exp2(torch.linspace(-30, 30, 700)).view(1, 700, 1, 1)
    for order in (size, size.flip(1)):
        b.v = (torch.randn(1, 700, 1, 128, generator=torch.Generator().manual_seed(1)) * order).to(torch.bfloat16)
        ref, bound, _ = b.reference()
        check(attend(b, b.cache(ops)), ref, bound)


def test_strided_queries_and_scale():
    b = Batch([90, 31], [4, 4], 4, 2, 64, "q4", page=16, seed=13)
    c = b.cache(ops)
    wide = torch.zeros(8, 9, 80, dtype=torch.bfloat16, device="cuda")
    view = wide[:, 2:6, 8:72]
    view.copy_(b.q)
    ref, bound, _ = b.reference(scale=0.31)
    y = ops.kv_attention(view, c, b.table, b.lens_t, cu=b.cu, scale=0.31)
    check(y, ref, bound)
    turned = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.kv_attention(turned, c, b.table, b.lens_t, scale=0.31, cu=b.cu), y)


def test_wide_page_table_view():
    b = Batch([90, 31], [1, 1], 4, 2, 64, "q4", page=16, seed=14)
    c = b.cache(ops)
    y = attend(b, c)
    big = torch.full((2, 50), -1, dtype=torch.int32, device="cuda")
    big[:, 10:10 + b.table.shape[1]] = b.table
    assert torch.equal(ops.kv_attention(b.q, c, big[:, 10:], b.lens_t), y)


@pytest.mark.parametrize("n", (1, 200))
def test_calls_repeat_bit_for_bit(n):
    b = Batch([2000, 5, 900], [n, 5 if n > 1 else 1, n], 16, 2, 128, "q4", page=64, seed=15)
    c = b.cache(ops)
    y = attend(b, c).clone()
    for _ in range(5):
        assert torch.equal(attend(b, c), y)


# ------------------------------------------------------------------ a run of the operators together
@pytest.mark.parametrize("fmt", FMTS)
def test_prompt_then_decode_steps(fmt):
    """A conversation: the prompt in two pieces, then single tokens, then a few drafted ones, each written and attended in
    its call; equal to the reference of the whole at every step."""
    total, H, Hkv, D = 260, 8, 2, 64
    pieces = [151, 93] + [1] * 5 + [4, 7]
    assert sum(pieces) == total
    whole = Batch([total], [total], H, Hkv, D, fmt, page=32, seed=20)
    ref, bound, _ = whole.reference(window=100, sinks=2)
    c = whole.cache(ops, fill=False)
    at = 0
    for n in pieces:
        lens = torch.tensor([at + n], dtype=torch.int32, device="cuda")
        ops.kv_write(c, whole.k[0, at:at + n].cuda(), whole.v[0, at:at + n].cuda(), whole.table, lens)
        y = ops.kv_attention(whole.q[at:at + n], c, whole.table, lens, window=100, sinks=2)
        check(y, ref[at:at + n], bound[at:at + n], what=(at, n))
        at += n
    k, v = ops.kv_read(c, whole.table, None, total)
    assert torch.equal(k.cpu(), stored(whole.k[0], fmt).to(torch.bfloat16))
    assert c.read_error() == 0


@pytest.mark.parametrize("n", (1, 3, 80))
def test_captured_step_replays_with_new_lengths(n):
    """One decode step (write, attend) captured in a CUDA graph: replays follow the tensors' new contents, two graphs with
    their own streams at once, and eager calls in between."""
    H, Hkv, D, L = 8, 2, 128, 400
    b = Batch([L, L - 77], [n, n], H, Hkv, D, "q4", page=32, seed=21)
    c = b.cache(ops)
    lens, q = b.lens_t.clone(), b.q.clone()
    k, v = b.new(b.k), b.new(b.v)

    def step():
        ops.kv_write(c, k, v, b.table, lens)
        return ops.kv_attention(q, c, b.table, lens)

    side = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for s in side:
        with torch.cuda.stream(s):
            step()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step())
        graphs.append(g)
    torch.cuda.synchronize()
    ref, bound, _ = b.reference()
    for _ in range(3):
        for s, g in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for y in outs:
        check(y, ref, bound)
    # shorter sequences: the same graph, other positions
    lens -= 31
    k.copy_(torch.cat([b.k[i, x - n - 31:x - 31] for i, x in enumerate(b.lens)]))
    v.copy_(torch.cat([b.v[i, x - n - 31:x - 31] for i, x in enumerate(b.lens)]))
    torch.cuda.synchronize()
    graphs[1].replay()
    torch.cuda.synchronize()
    short = Batch([L - 31, L - 77 - 31], [n, n], H, Hkv, D, "q4", page=32, seed=21)
    short.k, short.v, short.q = b.k[:, :L - 31], b.v[:, :L - 31], b.q
    ref, bound, _ = short.reference()
    check(outs[1], ref, bound)
    assert torch.equal(step(), outs[1])


def test_calls_on_two_streams():
    bs = [Batch([1500, 40], [1, 1], 8, 2, 128, "q4", page=64, seed=30 + i) for i in range(2)]
    cs = [b.cache(ops) for b in bs]
    want = [attend(b, c).clone() for b, c in zip(bs, cs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attend(bs[i], cs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("n", (1, 5, 40))
def test_without_cu_every_row_is_written(n):
    """Without cu the results are not cleared first: rows before a sequence's start, and their lse, are written all the same.
    Views of q too."""
    b = Batch([300, 40, 130], [n, n, n], 8, 2, 128, "q4", page=32, seed=45)
    c = b.cache(ops)
    lens = b.lens_t.clone()
    lens[1] = n - 1
    want, want_lse = ops.kv_attention(b.q, c, b.table, lens, cu=b.cu, max_q=n, return_lse=True)
    wide = torch.cat([b.q, b.q], dim=1)
    for q in (b.q, wide[:, :8]):
        for shape, dtype in ((b.q.shape, torch.bfloat16), (want_lse.shape, torch.float32)):
            junk = torch.full(shape, 7.0, dtype=dtype, device="cuda")
            del junk  # the next tensors of these sizes
        y, lse = ops.kv_attention(q, c, b.table, lens, return_lse=True)
        assert y.shape == b.q.shape and y.is_contiguous()
        # two kernels' results: 2^-8 of each by the last rounding, 2^-10 of the values (below 1 on average) by those inside
        assert torch.allclose(y.float(), want.float(), rtol=2 ** -7, atol=2e-3)
        assert not y[n].any() and lse[n].isneginf().all()
        seen = ~want_lse.isneginf()
        assert torch.equal(seen, ~lse.isneginf()) and torch.allclose(lse[seen], want_lse[seen], rtol=1e-4, atol=1e-4)


def test_another_current_device(monkeypatch):
    """Calls made while another device is current are made again with the cache's: here the first look says so."""
    b = Batch([70, 33], [1, 1], 8, 2, 128, "q4", page=16, seed=44)
    c = b.cache(ops)
    want, rows = attend(b, c, return_lse=True), ops.kv_read(c, b.table, None, 2)
    fresh = b.cache(ops, fill=False)
    looks = []
    monkeypatch.setattr(ops, "_current_device", lambda: 0 if len(looks) % 2 else 1)
    real = torch.cuda.device
    monkeypatch.setattr(torch.cuda, "device", lambda i: (looks.append(i), real(i))[1])
    cu = torch.tensor([0, 70, 103], dtype=torch.int32, device="cuda")
    ops.kv_write(fresh, b.flat(b.k), b.flat(b.v), b.table, b.lens_t, cu=cu)
    looks.append(None)
    got = ops.kv_attention(b.q, fresh, b.table, b.lens_t, cu=b.cu, max_q=1, return_lse=True)
    looks.append(None)
    back = ops.kv_read(fresh, b.table, None, 2)
    assert looks == [0, None, 0, None, 0]
    assert all(torch.equal(x, y) for x, y in zip((*got, *back), (*want, *rows)))


def test_refusals():
    b = Batch([20], [1], 4, 2, 64, "q4", page=16)
    c = b.cache(ops)
    k = b.new(b.k)
    t, n = b.table, b.lens_t
    for bad, match in [
            (lambda: ops.kv_write(c, k.float(), k, t, n), "bfloat16"), (lambda: ops.kv_write(c, k[:, :1], k, t, n), "heads"),
            (lambda: ops.kv_write(c, k, k.repeat(2, 1, 1), t, n), "rows"), (lambda: ops.kv_write(c, k[..., :32], k, t, n), "64"),
            (lambda: ops.kv_write(c, k, k, t.long(), n), "int32"), (lambda: ops.kv_write(c, k, k, t, n.long()), "int32"),
            (lambda: ops.kv_write(c, k, k, t, n.repeat(2)), "lens"), (lambda: ops.kv_write(c, k, k, t, n, cu=n), "cu"),
            (lambda: ops.kv_write(c, k, k, t.expand(3, -1), n.repeat(3)), "overlap"),
            (lambda: ops.kv_write(c, k, k, t.cpu(), n), "CUDA"),
            (lambda: ops.kv_write(c, torch.zeros(1, 2, 66, device="cuda", dtype=torch.bfloat16)[..., 1:65], k, t, n), "aligned"),
            (lambda: ops.kv_read(c, t, None, 1, out=(k[..., :32], k)), "out"),
            (lambda: ops.kv_attention(b.q[:, :3], c, t, n), "heads"), (lambda: ops.kv_attention(b.q, c, t, n, window=-1), "negative"),
            (lambda: ops.kv_attention(b.q, c, t, n, sink_logits=torch.zeros(2, device="cuda")), "sink_logits"),
            (lambda: ops.kv_attention(b.q, c, t, n, cu=b.cu, max_q=0), "max_q"),
            (lambda: ops.kv_attention(b.q, c, t, n, out=b.q.float()), "out"),
            (lambda: ops.kv_attention(b.q.repeat(3, 1, 1), c, t.repeat(2, 1), n.repeat(2)), "rows")]:
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises(_lib.MoebError, match="finite"):
        ops.kv_attention(b.q, c, t, n, scale=float("nan"))
