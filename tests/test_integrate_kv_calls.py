"""Calls of a model patched for the 4-bit KV cache that are not its ordinary prompt and steps: what the stock attention does in
calls without the cache, and what is refused with it. On the CPU, with the stand-ins of test_integrate_kv."""
import pytest
import torch

from moelab_b200 import integrate

transformers = pytest.importorskip("transformers")
from test_integrate import _gptoss, _qwen3  # noqa: E402
from test_integrate_kv import _sinks, _write, stand_in  # noqa: E402, F401


def _ids(rows, n, seed=1):
    return torch.randint(0, 512, (rows, n), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("family,stock", [(_qwen3, "eager"), (_qwen3, "sdpa"), (_gptoss, "eager")])
def test_calls_without_the_cache_are_the_stock_attention(family, stock):
    """Inference, a padded batch, training with dropout on the attention weights, gradients: bit for bit the stock model's, which
    ran the same function."""
    m = _sinks(family(dtype=torch.float32))
    m.config.attention_dropout = 0.5
    for x in m.modules():
        if hasattr(x, "attention_dropout"):
            x.attention_dropout = 0.5
    m.set_attn_implementation(stock)
    ids, pad = _ids(2, 12), torch.ones(2, 12, dtype=torch.long)
    pad[0, :4] = 0

    def calls():
        m.eval()
        with torch.no_grad():
            yield m(ids).logits
            yield m(ids, attention_mask=pad).logits
        m.train()
        torch.manual_seed(5)
        m.zero_grad()
        y = m(ids, attention_mask=pad).logits
        y.square().mean().backward()
        yield y.detach()
        yield m.model.layers[0].self_attn.k_proj.weight.grad.clone()

    want = list(calls())
    assert integrate.patch_hf_attention(m) == stock and integrate.patch_hf_attention(m) == stock
    for got, ref in zip(calls(), want):
        assert torch.equal(got, ref)
    integrate.unpatch_hf_attention(m)
    assert m.config._attn_implementation == stock
    for got, ref in zip(calls(), want):
        assert torch.equal(got, ref)


# ------------------------------------------------------------------ refused with the cache
BASE = dict(vocab_size=512, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=2,
            num_key_value_heads=1, head_dim=64, max_position_embeddings=128)


def _keyed(m, batch=1):
    """Arguments of a call of the attention function as a layer of m makes it, its key marked by a cache."""
    integrate.patch_hf_attention(m)
    cache = integrate.quantized_kv_cache(m, batch, 32, page_size=16)
    k = torch.randn(batch, 2, 3, 64)
    key, value = cache.update(k, k, 0)
    return (m.eval().model.layers[0].self_attn, torch.randn(batch, 4, 3, 64), key, value)


def test_capped_scores_are_refused(stand_in):
    m = transformers.Gemma2ForCausalLM(transformers.Gemma2Config(**BASE))
    with pytest.raises(ValueError, match="capped"):
        integrate.patch_hf_attention(m)
    with pytest.raises(ValueError, match="capped"):
        integrate.quantized_kv_cache(m, 1, 32)
    m.config.attn_logit_softcapping = None
    integrate.patch_hf_attention(m)


def test_arguments_the_kernel_does_not_know_are_refused(stand_in):
    call = _keyed(_qwen3(dtype=torch.float32))
    fine = dict(scaling=0.125, dropout=0.0, sliding_window=None, softcap=None, position_ids=torch.arange(3), use_cache=True)
    y, _ = integrate._attention(*call, None, **fine)
    assert y.shape == (1, 3, 4, 64)
    for kw in (dict(softcap=50.0), dict(cu_seq_lens_q=torch.tensor([0, 3])), dict(dropout=0.1), dict(is_causal=False), dict(bias=1)):
        with pytest.raises(ValueError, match="causal"):
            integrate._attention(*call, None, **{**fine, **kw})
    call[0].is_causal = False
    with pytest.raises(ValueError, match="causal"):
        integrate._attention(*call, None, **fine)


def _llama4(**kw):
    return transformers.Llama4ForCausalLM(transformers.Llama4TextConfig(**BASE, num_local_experts=2, **kw))


def test_masks_that_are_not_causal_or_a_window_are_refused(stand_in):
    """Chunked attention (stated through the mask alone), packed sequences, both directions. A window that the model states
    through the mask alone is the kernel's."""
    from transformers import masking_utils as mu
    m = _llama4(attention_chunk_size=8).eval()
    m.config.layer_types, types = None, m.config.layer_types  # the patch refuses them: here the calls
    integrate.patch_hf_attention(m)
    cache = integrate.quantized_kv_cache(m, 1, 32, page_size=16)
    m.config.layer_types = types
    with torch.no_grad(), pytest.raises(ValueError, match="other than the causal"):
        m(_ids(1, 20), past_key_values=cache)
    assert integrate._window(mu.causal_mask_function, None) == 0
    assert integrate._window(mu.sliding_window_causal_mask_function(9), 9) == 9
    packed = mu.and_masks(mu.causal_mask_function, mu.packed_sequence_mask_function(torch.zeros(1, 4, dtype=torch.long)))
    for f, n in ((mu.sliding_window_causal_mask_function(9), 8), (mu.sliding_window_causal_mask_function(9), None), (packed, None),
                 (mu.bidirectional_mask_function, None), (mu.chunked_causal_mask_function(8, torch.zeros(1, dtype=torch.int)), 8),
                 (lambda b, h, q, k: k <= q, None), (mu.sliding_window_bidirectional_mask_function(9), 9)):
        with pytest.raises(ValueError, match="other than the causal"):
            integrate._window(f, n)

    call = _keyed(_qwen3(dtype=torch.float32))
    got = [integrate._attention(*call, integrate._Causal(w), scaling=0.125, **kw)[0]
           for w, kw in ((2, {}), (2, dict(sliding_window=2)), (0, {}))]
    assert torch.equal(got[0], got[1]) and not torch.equal(got[0], got[2])
    with pytest.raises(ValueError, match="window"):
        integrate._attention(*call, integrate._Causal(0), scaling=0.125, sliding_window=2)
    with pytest.raises(ValueError, match="as they are"):  # the key is not the one that the cache marked
        integrate._attention(*call[:2], call[2].clone(), call[3], integrate._Causal(0), scaling=0.125)


def test_padded_batches_are_refused_token_by_token(stand_in):
    m = _qwen3(dtype=torch.float32).eval()
    integrate.patch_hf_attention(m)
    ids = _ids(2, 4)
    cache = integrate.quantized_kv_cache(m, 2, 32, page_size=16)
    with torch.no_grad():
        with pytest.raises(ValueError, match="padded"):
            m(ids[:, :1], attention_mask=torch.tensor([[1], [0]]), past_key_values=cache)
        assert cache.get_seq_length() == 0
        for i in range(3):
            m(ids[:, i:i + 1], attention_mask=torch.ones(2, i + 1, dtype=torch.long), past_key_values=cache)
        for late in (0, 3):
            mask = torch.ones(2, 4, dtype=torch.long)
            mask[1, late] = 0
            with pytest.raises(ValueError, match="padded"):
                m(ids[:, 3:], attention_mask=mask, past_key_values=cache)
    assert cache.get_seq_length() == 3


@pytest.mark.parametrize("frozen", [(), ("q_proj",), ("q_proj", "k_proj"), ("k_proj", "v_proj")])
def test_gradients_through_the_cache_are_an_error(stand_in, frozen):
    """In eval mode with gradients on the logits are those without, and a backward pass through the cached attention is refused,
    whichever of its inputs needs one. Where none does the rest of the model has its gradients."""
    m = _qwen3(dtype=torch.float32).eval()
    integrate.patch_hf_attention(m)
    ids = _ids(1, 5)
    with torch.no_grad():
        want = m(ids, past_key_values=integrate.quantized_kv_cache(m, 1, 32, page_size=16)).logits
    for n, p in m.named_parameters():
        p.requires_grad_("lm_head" in n or ("_proj" in n and "self_attn" in n and not any(f in n for f in frozen)))
    y = m(ids, past_key_values=integrate.quantized_kv_cache(m, 1, 32, page_size=16)).logits
    assert torch.equal(y.detach(), want)
    with pytest.raises(NotImplementedError, match="backward"):
        y.sum().backward()
    for n, p in m.named_parameters():
        p.requires_grad_("lm_head" in n)
    m(ids, past_key_values=integrate.quantized_kv_cache(m, 1, 32, page_size=16)).logits.sum().backward()
    assert m.lm_head.weight.grad.any()


def test_lengths_follow_the_layer_that_calls(stand_in):
    """A model whose first layer does not write keys: the rows of the next one are where its own count says, and read back."""
    m = _qwen3(dtype=torch.float32)
    integrate.patch_hf_attention(m)
    cache = integrate.quantized_kv_cache(m, 2, 32, page_size=16)
    k = torch.randn(2, 2, 5, 64)
    for a, b in ((0, 3), (3, 4), (4, 5)):
        cache.update(k[:, :, a:b], -k[:, :, a:b], 1)
        assert cache.moeb_lens.tolist() == [b, b] and cache.moeb_seen == [0, b]
    stored = cache.moeb_layers[1]
    assert torch.equal(stored.k[:5], k[0].transpose(0, 1)) and torch.equal(stored.v[32:37], -k[1].transpose(0, 1))
    cache.crop(0)
    cache.update(k, k, 0)
    assert cache.moeb_lens.tolist() == [5, 5]
    cache.update(k[:, :, :2], k[:, :, :2], 1)
    assert cache.moeb_lens.tolist() == [2, 2]


def test_models_with_other_layers_are_refused():
    linear = transformers.Qwen3NextConfig(**{**BASE, "num_hidden_layers": 4})
    with pytest.raises(ValueError, match="linear_attention"):
        integrate._head_dim(linear)
    with pytest.raises(ValueError, match="chunked_attention"):
        integrate.patch_hf_attention(_llama4())


def test_models_that_are_not_patched_refuse_the_cache(stand_in):
    """Their attention would see the newest keys alone. After unpatching, to_stock() goes on."""
    m = _qwen3(dtype=torch.float32).eval()
    ids = _ids(1, 9)
    cache = integrate.quantized_kv_cache(m, 1, 32, page_size=16)
    with torch.no_grad():
        want = m(ids).logits
        with pytest.raises(ValueError, match="patch_hf_attention"):
            m(ids[:, :5], past_key_values=cache)
        assert cache.get_seq_length() == 0
        integrate.patch_hf_attention(m)
        m(ids[:, :5], past_key_values=cache)
        integrate.unpatch_hf_attention(m)
        with pytest.raises(ValueError, match="to_stock"):
            m(ids[:, 5:6], past_key_values=cache)
        assert cache.get_seq_length() == 5
        got = m(ids[:, 5:], past_key_values=cache.to_stock()).logits
    assert (got - want[:, 5:]).norm() / want[:, 5:].norm() < 2e-2  # the stand-in's rows come back in bfloat16


def test_captured_calls_are_refused(stand_in, monkeypatch):
    m = _qwen3(dtype=torch.float32).eval()
    integrate.patch_hf_attention(m)
    cache = integrate.quantized_kv_cache(m, 1, 32, page_size=16)
    assert not integrate._capturing(torch.zeros(1))
    monkeypatch.setattr(integrate, "_capturing", lambda t: True)
    with torch.no_grad(), pytest.raises(RuntimeError, match="captured"):
        m(_ids(1, 5), past_key_values=cache)
    assert cache.moeb_seen == [0, 0]


def test_refused_calls_leave_the_cache_as_it_was(stand_in, monkeypatch):
    """A call in training mode, one with a mask of its own, one whose write fails: the next call goes on where the last good one
    ended."""
    m = _qwen3(dtype=torch.float32).eval()
    integrate.patch_hf_attention(m)
    ids = _ids(2, 12)
    with torch.no_grad():
        want = m(ids).logits
        cache = integrate.quantized_kv_cache(m, 2, 32, page_size=16)

        def no_launch():
            raise RuntimeError("no launch")

        def refused(n, error, **kw):
            seen = list(cache.moeb_seen)
            with pytest.raises(error):
                m(ids[:, :n], past_key_values=cache, **kw)
            assert cache.moeb_seen == seen

        for a, b in ((0, 5), (5, 11), (11, 12)):
            m.train()
            refused(4, ValueError)
            m.eval()
            refused(3, ValueError, attention_mask=torch.ones(2, 1, 3, a + 3, dtype=torch.bool))
            with monkeypatch.context() as patch:
                patch.setattr(integrate.ops, "kv_write", lambda *_: no_launch())
                refused(2, RuntimeError)
                left = [1]
                patch.setattr(integrate.ops, "kv_write", lambda *a: _write(*a) if left and left.pop() else no_launch())
                refused(2, RuntimeError)  # in the second layer
            got = m(ids[:, a:b], past_key_values=cache).logits
            assert (got - want[:, a:b]).norm() / want[:, a:b].norm() < 1e-4, (a, b)
