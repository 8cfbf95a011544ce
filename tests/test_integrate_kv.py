"""Model integration of the 4-bit KV cache (moelab_b200/integrate.py): Hugging Face models decode over it. Host logic on the
CPU with torch stand-ins for the operators; on the GPU against stock attention over the same stored values."""
import pytest
import torch

from moelab_b200 import integrate, ops

transformers = pytest.importorskip("transformers")
from test_integrate import _deepseek, _gptoss, _logits, _mixtral, _qwen3  # noqa: E402


class _StandIn:
    """ops.KVCache in plain torch: rows kept as they are; kv_write / kv_attention / kv_read with the operators' meaning."""

    def __init__(self, pages, kv_heads, head_dim, page_size=64, fmt="q4", device=None):
        self.page_size, self.kv_heads, self.head_dim, self.device = page_size, kv_heads, head_dim, torch.device("cpu")
        self.k, self.v = (torch.zeros(pages * page_size, kv_heads, head_dim) for _ in range(2))

    def at(self, table, b, p):
        return int(table[b, p // self.page_size]) * self.page_size + p % self.page_size


def _write(c, k, v, table, lens, cu=None):
    n = k.shape[0] // len(lens)
    for b in range(len(lens)):
        for i in range(n):
            at = c.at(table, b, int(lens[b]) - n + i)
            c.k[at], c.v[at] = k[b * n + i].float(), v[b * n + i].float()


def _read(c, table, cu, rows, first=None, out=None):
    n = rows // table.shape[0]
    at = [c.at(table, b, p) for b in range(table.shape[0]) for p in range(n)]
    return c.k[at].to(torch.bfloat16), c.v[at].to(torch.bfloat16)


def _attend(q, c, table, lens, cu=None, max_q=None, scale=None, window=0, sinks=0, sink_logits=None):
    T, H, D = q.shape
    n, G = T // len(lens), H // c.kv_heads
    y = torch.zeros(T, H, D)
    for b in range(len(lens)):
        for i in range(n):
            p = int(lens[b]) - n + i
            at = [c.at(table, b, j) for j in range(p + 1) if not window or j > p - window]
            for h in range(H):
                s = scale * (c.k[at, h // G] @ q[b * n + i, h].float())
                if sink_logits is not None:
                    s = torch.cat([s, sink_logits[h:h + 1]])
                y[b * n + i, h] = torch.softmax(s, 0)[:len(at)] @ c.v[at, h // G]
    return y.to(q.dtype)


@pytest.fixture
def stand_in(monkeypatch):
    for name, f in (("KVCache", _StandIn), ("kv_write", _write), ("kv_read", _read), ("kv_attention", _attend)):
        monkeypatch.setattr(ops, name, f)
    # rows stay in float32: what is tested is which rows meet which
    monkeypatch.setattr(integrate, "_rows", lambda t: t.transpose(1, 2).reshape(-1, t.shape[1], t.shape[3]))


MODELS = {"qwen3": _qwen3, "mixtral": _mixtral, "gptoss": _gptoss}


def _sinks(m):
    """The stock init leaves gpt-oss's sink logits undefined or zero: give them values."""
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.endswith("sinks"):
                p.copy_(torch.randn(p.shape, generator=g).to(p.dtype))
    return m


@pytest.mark.parametrize("family", sorted(MODELS))
def test_prompt_and_steps_follow_the_stock_model(family, stand_in):
    """A prompt longer than gpt-oss's window in two calls, then steps, two sequences: logits of the stock model's eager
    attention and cache, in float32 throughout."""
    m = _sinks(MODELS[family](dtype=torch.float32)).eval()
    m.set_attn_implementation("eager")
    ids = torch.randint(0, 512, (2, 83), generator=torch.Generator().manual_seed(1))
    cuts = [0, 70, 79, 80, 81, 83]
    stock, want = transformers.DynamicCache(config=m.config), []
    with torch.no_grad():
        for a, b in zip(cuts, cuts[1:]):
            want.append(m(ids[:, a:b], past_key_values=stock).logits)
    assert integrate.patch_hf_attention(m) == "eager"
    cache = integrate.quantized_kv_cache(m, 2, 96, page_size=16)
    with torch.no_grad():
        for (a, b), ref in zip(zip(cuts, cuts[1:]), want):
            got = m(ids[:, a:b], past_key_values=cache).logits
            assert cache.get_seq_length() == b
            assert (got - ref).norm() / ref.norm() < 1e-4, (a, b)
        plain = m(ids).logits  # without a 4-bit cache: plain torch
        assert (plain[:, :70] - want[0]).norm() / want[0].norm() < 1e-4
        back = cache.to_stock()
        assert back.get_seq_length() == 83
    assert integrate.unpatch_hf_attention(m) and not integrate.unpatch_hf_attention(m)
    assert m.config._attn_implementation == "eager"
    with torch.no_grad():
        assert torch.equal(m(ids[:, :70], past_key_values=transformers.DynamicCache(config=m.config)).logits, want[0])


def test_generate(stand_in):
    m = _qwen3(dtype=torch.float32).eval()
    ids = torch.randint(0, 512, (1, 9), generator=torch.Generator().manual_seed(2))
    kw = dict(max_new_tokens=6, do_sample=False, pad_token_id=0)
    with torch.no_grad():
        ref = m.generate(ids, **kw)
        integrate.patch_hf_attention(m)
        got = m.generate(ids, past_key_values=integrate.quantized_kv_cache(m, 1, 32, page_size=16), **kw)
    assert torch.equal(got[:, :10], ref[:, :10]) and got.shape == ref.shape


def test_refusals(stand_in):
    m = _qwen3(dtype=torch.float32).eval()
    integrate.patch_hf_attention(m)
    cache = integrate.quantized_kv_cache(m, 2, 16, page_size=16)
    ids = torch.zeros(2, 5, dtype=torch.long)
    with torch.no_grad():
        with pytest.raises(ValueError, match="padded"):
            m(ids, attention_mask=torch.tensor([[1, 1, 1, 1, 1], [0, 0, 1, 1, 1]]), past_key_values=cache)
        with pytest.raises(ValueError, match="sequences"):
            m(ids[:1], past_key_values=cache)
        with pytest.raises(ValueError, match="holds"):
            m(torch.zeros(2, 17, dtype=torch.long), past_key_values=integrate.quantized_kv_cache(m, 2, 16, page_size=16))
    with pytest.raises(ValueError, match="latent"):
        integrate.patch_hf_attention(_deepseek())
    wide = transformers.Qwen3MoeConfig(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=80)
    with pytest.raises(ValueError, match="80"):
        integrate._head_dim(wide)


@pytest.mark.parametrize("family", ["qwen3", "gptoss"])
def test_without_the_cache_masks_are_the_stock_models(family):
    """A patched model called without a 4-bit cache: padded batches, the caller's own mask and a static cache give the eager
    attention's logits; gradients are its gradients."""
    m = _sinks(MODELS[family](dtype=torch.float32)).eval()
    m.set_attn_implementation("eager")
    ids = torch.randint(0, 512, (2, 12), generator=torch.Generator().manual_seed(5))
    pad = torch.ones(2, 12, dtype=torch.long)
    pad[0, :4] = 0
    own = torch.ones(12, 12, dtype=torch.bool).tril().expand(2, 1, 12, 12).clone()
    own[:, :, 6:, :6] = False  # two documents in a row
    first = lambda: transformers.StaticCache(config=m.config, max_cache_len=40)

    def grads():
        m.zero_grad()
        m(ids, attention_mask=pad).logits[pad.bool()].square().mean().backward()
        return [p.grad.clone() for n, p in m.named_parameters() if "q_proj.weight" in n or "k_proj.weight" in n]

    # the eager attention adds whatever mask it is given: a bool one would be 0 and 1 there, so it gets the additive form
    added = torch.zeros(own.shape).masked_fill(~own, torch.finfo(torch.float32).min)

    def calls(own):
        with torch.no_grad():
            yield m(ids, attention_mask=pad).logits[pad.bool()]
            yield m(ids, attention_mask=own).logits
            yield m(ids, past_key_values=first()).logits

    want, want_grads = list(calls(added)), grads()
    integrate.patch_hf_attention(m)
    for mask in (own, added):
        for got, ref in zip(calls(mask), want):
            assert (got - ref).norm() / ref.norm() < 1e-4
    for got, ref in zip(grads(), want_grads):
        assert (got - ref).norm() / ref.norm() < 1e-3


def test_cache_gives_tokens_up_and_refuses_the_rest(stand_in):
    m = _qwen3(dtype=torch.float32).eval()
    integrate.patch_hf_attention(m)
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(6))
    new = lambda: integrate.quantized_kv_cache(m, 2, 32, page_size=16)
    with torch.no_grad():
        want, cache = m(ids, past_key_values=new()).logits, new()
        m(ids.flip(1), past_key_values=cache)
        cache.crop(-5)
        assert cache.get_seq_length() == 15
        cache.reset()
        m(ids[:, :17], past_key_values=cache)
        cache.crop(11)
        got = m(ids[:, 11:], past_key_values=cache).logits
        assert (got - want[:, 11:]).norm() / want[:, 11:].norm() < 1e-4
        with pytest.raises(ValueError, match="own"):
            m(ids[:, :3], attention_mask=torch.ones(2, 1, 3, 23, dtype=torch.bool), past_key_values=cache)
        with pytest.raises(NotImplementedError):
            m.generate(ids[:1], past_key_values=new(), num_beams=2, max_new_tokens=3, do_sample=False, pad_token_id=0,
                       attention_mask=torch.ones(1, 20, dtype=torch.long))
        with pytest.raises(ValueError, match="eval"):
            m.train()(ids, past_key_values=new())
    for call in (lambda c: c.reorder_cache(torch.tensor([1, 0])), lambda c: c.batch_repeat_interleave(2),
                 lambda c: c.batch_select_indices(torch.tensor([0]))):
        with pytest.raises(NotImplementedError):
            call(new())


# ------------------------------------------------------------------ GPU
class _Stored(transformers.DynamicCache):
    """The stock cache, with every row replaced by what the 4-bit cache stores of it."""

    def __init__(self, config, fmt):
        super().__init__(config=config)
        self.fmt = fmt

    def update(self, k, v, layer_idx, cache_kwargs=None):
        from kv_helpers import stored
        return super().update(*(stored(t, self.fmt).to(t.device, t.dtype) for t in (k, v)), layer_idx)


@pytest.mark.gpu
@pytest.mark.parametrize("family", sorted(MODELS))
@pytest.mark.parametrize("fmt", ["q4", "mxfp4"])
def test_logits_match_stock_attention_on_the_stored_values(family, fmt):
    """Prompt, a second piece, single tokens: the patched model against eager attention over the oracle's stored values of the
    same rows, in float32. Queries and results pass bf16 in the library: rows differ by that (2^-8 per rounding, two layers),
    but for the few where it tips a router's near-tie and another expert answers."""
    m = _sinks(MODELS[family](dtype=torch.float32)).cuda().eval()
    m.set_attn_implementation("eager")
    ids = torch.randint(0, 512, (2, 90), generator=torch.Generator().manual_seed(1)).cuda()
    cuts = [0, 75, 84, 85, 86, 90]
    stock, want = _Stored(m.config, fmt), []
    with torch.no_grad():
        for a, b in zip(cuts, cuts[1:]):
            want.append(m(ids[:, a:b], past_key_values=stock).logits)
        integrate.patch_hf_attention(m)
        cache, rows = integrate.quantized_kv_cache(m, 2, 128, fmt=fmt, page_size=32), []
        for (a, b), ref in zip(zip(cuts, cuts[1:]), want):
            got = m(ids[:, a:b], past_key_values=cache).logits
            rows.append((got - ref).norm(dim=-1) / ref.norm(dim=-1))
    rows = torch.cat(rows, dim=1).flatten()
    assert (rows < 2e-2).float().mean() >= 0.9, rows.sort().values[-20:]
    assert all(c.read_error() == 0 for c in cache.moeb_layers)


@pytest.mark.gpu
def test_decode_with_quantized_experts_and_cache():
    """Both patches at once: greedy decoding with int4 experts and the 4-bit cache, then on from to_stock()."""
    m = _qwen3().cuda().eval()
    integrate.patch_hf_moe(m)
    integrate.patch_hf_attention(m)
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(4)).cuda()
    cache = integrate.quantized_kv_cache(m, 2, 64)
    # the mask is given: generate() takes ids equal to pad_token_id for padding otherwise, which the cache refuses
    out = m.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, max_new_tokens=8, do_sample=False,
                     pad_token_id=0)
    assert out.shape == (2, 28) and cache.get_seq_length() == 27
    assert all(c.read_error() == 0 for c in cache.moeb_layers)
    with torch.no_grad():
        a = m(out[:, 27:], past_key_values=cache).logits.float()
        stock = cache.to_stock()  # 28 tokens; drop the last, which the next call brings again
        integrate.unpatch_hf_attention(m)
        stock.crop(27)
        b = m(out[:, 27:], past_key_values=stock).logits.float()
    # the last token's own key and value are the unrounded ones in the stock cache: 4 bits of 1 in 28 rows
    assert (a - b).norm() / b.norm() < 0.2
    assert torch.isfinite(_logits(m, ids)).all()
