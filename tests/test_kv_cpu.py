"""The 4-bit KV cache's argument checks, which run before any device work: here without a GPU, with made-up addresses."""
import ctypes

import pytest
import torch

from moelab_b200 import _lib, ops


def _cache(**kw):
    f = dict(kq=4096, ks=4096, vq=4096, vs=4096, err=4096, pages=4, page_size=16, kv_heads=2, head_dim=64, format=0)
    f.update(kw)
    return ctypes.pointer(_lib.KvCacheStruct(*f.values()))


def _write(cache, k=4096, k_row=128, k_head=64, T=2, cu=None, lens=4096, table=4096, trow=4, B=2, P=4):
    _lib.call("moeb_kv_write", cache, k, k_row, k_head, 4096, 128, 64, T, cu, lens, table, trow, B, P, None)


def _read(cache, T=2, table=4096, B=2, k=4096):
    _lib.call("moeb_kv_read", cache, T, None, None, table, 4, B, 4, k, 4096, None)


def _attend(cache, q=4096, q_row=256, T=2, H=4, B=2, P=4, max_q=1, scale=0.125, window=0, sinks=0, y=4096, ws=4096,
            ws_bytes=1 << 40):
    _lib.call("moeb_kv_attention", cache, q, q_row, 64, T, H, None, 4096, 4096, P, B, P, max_q, scale, window, sinks, None, y,
              None, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,match", [
    (dict(kq=0), "null"), (dict(err=0), "null"), (dict(vs=8), "aligned"), (dict(format=2), "format"),
    (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(page_size=8192), "page_size"), (dict(pages=0), "positive"), (dict(kv_heads=-1), "positive")])
def test_bad_cache_is_refused(kw, match):
    for f in (_write, _read, _attend):
        with pytest.raises(_lib.MoebError, match=match):
            f(_cache(**kw))


def test_null_cache_is_refused():
    for f in (_write, _read, _attend):
        with pytest.raises(_lib.MoebError, match="null"):
            f(None)


@pytest.mark.parametrize("kw,match", [
    (dict(T=-1), "negative"), (dict(B=-1), "negative"), (dict(P=-1), "negative"), (dict(T=3), "multiple of B"),
    (dict(lens=None), "null"), (dict(table=None), "null"), (dict(trow=3), "overlap"), (dict(k=None), "16-byte"),
    (dict(k=4100), "16-byte"), (dict(k_row=4), "16-byte"), (dict(k_head=63), "16-byte"), (dict(T=1 << 27), "2\\^26"),
    (dict(P=1 << 27, trow=1 << 27), "2\\^30"), (dict(B=1 << 24, T=1 << 24), "2\\^24"),
    (dict(B=1 << 22, T=1 << 22, P=1 << 16, trow=1 << 16), "2\\^38")])
def test_bad_write_is_refused(kw, match):
    with pytest.raises(_lib.MoebError, match=match):
        _write(_cache(), **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(H=3), "multiple"), (dict(H=0), "multiple"), (dict(H=8192), "4096"), (dict(window=-1), "negative"),
    (dict(sinks=-1), "negative"), (dict(scale=float("inf")), "finite"), (dict(scale=float("nan")), "finite"),
    (dict(scale=3e38), "finite"), (dict(scale=-3e38), "finite"),
    (dict(max_q=0), "max_q"), (dict(q=4104), "16-byte"), (dict(q_row=4), "16-byte"), (dict(y=None), "aligned"),
    (dict(y=8), "aligned"), (dict(T=-2), "negative"), (dict(T=1 << 22, H=2048), "2\\^31"), (dict(ws_bytes=16, P=512), "small"),
    (dict(ws=None, P=512), "workspace"), (dict(ws=4104, P=512), "workspace")])
def test_bad_attention_is_refused(kw, match):
    with pytest.raises(_lib.MoebError, match=match):
        _attend(_cache(), **kw)


def test_bad_read_is_refused():
    with pytest.raises(_lib.MoebError, match="aligned"):
        _read(_cache(), k=4104)
    with pytest.raises(_lib.MoebError, match="null"):
        _read(_cache(), table=None)


def test_calls_without_rows_do_nothing():
    for kw in (dict(T=0), dict(B=0, T=0)):
        _write(_cache(), **kw)
        _read(_cache(), **kw)
        _attend(_cache(), **kw)


def test_error_word_pointer_is_checked():
    with pytest.raises(_lib.MoebError, match="null"):
        _lib.call("moeb_kv_read_error", _cache(), None, None)


def test_python_checks():
    with pytest.raises(ValueError, match="format"):
        ops.KVCache(4, 2, 64, fmt="int8")
    with pytest.raises(ValueError, match="head_dim"):
        ops.KVCache(4, 2, 80)
    with pytest.raises(ValueError, match="page_size"):
        ops.KVCache(4, 2, 64, page_size=24)
    with pytest.raises(ValueError, match="positive"):
        ops.KVCache(0, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.KVCache(4, 2, 64, device="cpu")

    class Fake:
        device, index, kv_heads, head_dim = torch.device("cuda", 0), 0, 2, 64
    cpu = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_write(Fake, cpu, cpu, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_attention(cpu, Fake, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_read(Fake, torch.zeros(2, 1, dtype=torch.int32), None, 2)


def test_calls_from_python_reach_the_same_entries():
    """The CPython module over the calls: its arguments in the header's order, what does not convert is refused, the status of
    the entry comes back."""
    hot, c = _lib.hot(), _cache()
    a = ctypes.addressof(c.contents)
    write = (a, 4096, 128, 64, 4096, 128, 64, 0, None, 4096, 4096, 4, 2, 4, None)
    read = (a, 0, None, None, 4096, 4, 2, 4, 4096, 4096, None)
    attend = (a, 4096, 256, 64, 0, 4, None, 4096, 4096, 4, 2, 4, 1, 0.125, 0, 0, None, 4096, None, 4096, 0, None)
    for name, args in (("moeb_kv_write", write), ("moeb_kv_read", read), ("moeb_kv_attention", attend)):
        f = getattr(hot, name)
        assert f(*args) == _lib.MOEB_OK
        assert len(args) == len(_lib.SIGNATURES[name][1])
        assert f(None, *args[1:]) == _lib.MOEB_EINVAL and b"null" in _lib.load().moeb_last_error()
        for i, (kind, v) in enumerate(zip(_lib.SIGNATURES[name][1], args)):
            with pytest.raises(TypeError):
                f(*args[:i], "x", *args[i + 1:])
            if kind is ctypes.c_int:
                with pytest.raises(OverflowError):
                    f(*args[:i], 2 ** 31, *args[i + 1:])
                with pytest.raises(OverflowError):
                    f(*args[:i], 2 ** 70, *args[i + 1:])
        with pytest.raises(TypeError, match="arguments"):
            f(*args[1:])
    assert hot.moeb_kv_attention(*attend[:14], -1, *attend[15:]) == _lib.MOEB_EINVAL  # the window
    with pytest.raises(_lib.MoebError, match="moeb_kv_read failed with status 1"):
        _lib.failed("moeb_kv_read", 1)
