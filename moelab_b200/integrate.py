"""Model integration: run the sparse-MoE blocks of a Hugging Face transformers model through this library's layer
call.

This is the torch counterpart of the reference's mlx-lm patch (moelab/e2e.py:29-72 and its _patch_gptoss /
_patch_deepseek variants). That patch swaps the expert compute of every MoE block for a variant's `run` at
decode-sized calls (<= MAX_T tokens, e2e.py:26) and keeps the stock path above. Here each block's expert
weights are quantized once into the variant state, and the block's forward runs router + experts + combine as
one `layer` call for up to `max_tokens` tokens. Supported blocks:

- Qwen3MoeSparseMoeBlock, MixtralSparseMoeBlock. `experts.gate_up_proj` [E, 2f, d] and `experts.down_proj`
  [E, d, f], SiLU-gated. Router: softmax over all experts, top-k, renormalised when `norm_topk_prob`
  (Qwen3-MoE) or always (Mixtral). int4 affine g64 or MXFP4.
- GptOssMLP. `experts.gate_up_proj` [E, d, 2f] with gate and up columns interleaved, `down_proj` [E, f, d],
  per-expert biases, clamped SwiGLU (alpha 1.702, limit 7, (u + 1)). Router: linear with bias, softmax over
  the top-k logits (e2e.py:171-176). MXFP4, the format gpt-oss ships in. Returns (y, routing weights) like the
  stock block.
- DeepseekV2Moe with `topk_method == "greedy"`. The routed experts are laid out as in Qwen3-MoE. The
  `shared_experts` MLP (width n * f) runs as n always-on experts of weight 1 (e2e.py:146-147). Router: fp32
  softmax over all experts, top-k without renormalisation, times `routed_scaling_factor` (e2e.py:136-140).
  int4.

The attention of the same models (heads of 64 or 128 values; not DeepSeek's latent attention) can run over the 4-bit KV cache:
`patch_hf_attention` routes it through the library for calls that carry a `QuantizedKVCache`, which takes the place of the
model's cache in `model(...)` and `model.generate(...)`. gpt-oss's sliding windows and sink logits are arguments of the kernel.

The library computes router logits in fp32 from bf16 inputs. Where a stock block computes them in the model
dtype, near-ties can pick a different expert. `dequantize_into_stock` writes the variant's dequantized weights
back into the stock parameters, so a stock model runs on exactly the weights the kernels see; the tests compare
the two on that basis.
"""
import sys
import types

import torch

from . import ops
from .variants.cuda import b200_mxfp4_gptoss, b200_mxfp4_moe, b200_q4_moe

FAMILIES = {"Qwen3MoeSparseMoeBlock": "switch", "MixtralSparseMoeBlock": "switch", "GptOssMLP": "gptoss",
            "DeepseekV2Moe": "deepseek"}
KNOWN_BLOCKS = tuple(FAMILIES)
MAX_TOKENS = 256  # decode-sized calls use the library; larger ones keep the stock block (e2e.py:26)


def moe_blocks(model):
    """The model's sparse-MoE blocks this patch can take over, in module order."""
    return [m for m in model.modules() if type(m).__name__ in FAMILIES]


def _variant(fmt):
    if fmt == "q4":
        return b200_q4_moe
    if fmt == "mxfp4":
        return b200_mxfp4_moe
    raise ValueError(f"unknown format {fmt!r} (q4 or mxfp4)")


def _is_silu(act):
    return act is None or isinstance(act, torch.nn.SiLU) or type(act).__name__ in ("SiLU", "SiLUActivation")


def _bf16(t):
    return t.detach().to(torch.bfloat16).contiguous()


def _switch_weights(ex):
    E, f2, d = ex.gate_up_proj.shape
    f = f2 // 2
    assert ex.down_proj.shape == (E, d, f), "unexpected expert layout"
    assert _is_silu(getattr(ex, "act_fn", None)), "only SiLU-gated experts are supported"
    w = ex.gate_up_proj.detach()
    return w[:, :f], w[:, f:], ex.down_proj.detach()


def _prepare(b, fmt):
    """(variant module, state, forward kind, static call arguments) for one block."""
    fam = FAMILIES[type(b).__name__]
    if fam == "switch":
        mod = _variant(fmt)
        wg, wu, wd = _switch_weights(b.experts)
        assert wg.is_cuda, "moelab_b200 runs on CUDA devices only"
        st = mod.prepare(_bf16(wg), _bf16(wu), _bf16(wd))
        return mod, st, {"k": int(b.gate.top_k), "norm": bool(getattr(b.gate, "norm_topk_prob", True))}
    if fam == "gptoss":
        ex = b.experts
        assert ex.gate_up_proj.is_cuda, "moelab_b200 runs on CUDA devices only"
        assert float(ex.alpha) == 1.702 and float(ex.limit) == 7.0, "clamped SwiGLU constants differ"
        gu, bgu = ex.gate_up_proj.detach(), ex.gate_up_proj_bias.detach()
        wg, wu = gu[..., ::2].transpose(1, 2), gu[..., 1::2].transpose(1, 2)  # [E, f, d]
        wd = ex.down_proj.detach().transpose(1, 2)                               # [E, d, f]
        st = b200_mxfp4_gptoss.state(_bf16(wg), _bf16(wu), _bf16(wd), bgu[:, ::2], bgu[:, 1::2],
                                     ex.down_proj_bias.detach())
        return b200_mxfp4_gptoss, st, {"k": int(b.router.top_k)}
    # deepseek
    if fmt != "q4":
        raise ValueError("DeepSeek shared experts run on the int4 path")
    assert b.topk_method == "greedy", "only greedy top-k routing is supported"
    wg, wu, wd = _switch_weights(b.experts)
    assert wg.is_cuda, "moelab_b200 runs on CUDA devices only"
    sh = b.shared_experts
    assert sh.gate_proj.bias is None and _is_silu(getattr(sh, "act_fn", None)), "unsupported shared MLP"
    st = b200_q4_moe.prepare_shared(_bf16(wg), _bf16(wu), _bf16(wd), _bf16(sh.gate_proj.weight),
                                    _bf16(sh.up_proj.weight), _bf16(sh.down_proj.weight))
    return b200_q4_moe, st, {"k": int(b.top_k), "norm": False, "rscale": float(b.routed_scaling_factor)}


def patch_hf_moe(model, fmt="q4", max_tokens=MAX_TOKENS):
    """Quantize every known sparse-MoE block's experts and route its forward through the library for calls of up to
    `max_tokens` tokens. Returns the number of blocks patched. Idempotent (a patched block is re-quantized).
    gpt-oss blocks always use MXFP4."""
    if fmt not in ("q4", "mxfp4"):
        raise ValueError(f"unknown format {fmt!r} (q4 or mxfp4)")
    blocks = moe_blocks(model)
    for b in blocks:
        mod, st, kw = _prepare(b, fmt)
        if "_moeb_stock" not in b.__dict__:
            b._moeb_stock = b.forward
        b._moeb = {"family": FAMILIES[type(b).__name__], "mod": mod, "state": st, "kw": kw,
                   "max_tokens": int(max_tokens)}
        b.forward = types.MethodType(_forward, b)
    return len(blocks)


def unpatch_hf_moe(model):
    """Restore the stock forward of every patched block."""
    n = 0
    for b in moe_blocks(model):
        if "_moeb_stock" in b.__dict__:
            b.forward = b._moeb_stock
            del b._moeb_stock
            del b._moeb
            n += 1
    return n


def dequantize_into_stock(model):
    """Write each patched block's dequantized expert weights into its stock parameters (in their dtype), so the
    stock forward runs on the weights the kernels use."""
    for b in moe_blocks(model):
        cfg = b.__dict__.get("_moeb")
        if cfg is None:
            continue
        wg, wu, wd = cfg["mod"].dequant(cfg["state"])
        ex = b.experts
        with torch.no_grad():
            if cfg["family"] == "gptoss":
                gu = ex.gate_up_proj
                gu[..., ::2].copy_(wg.transpose(1, 2).to(gu.dtype))
                gu[..., 1::2].copy_(wu.transpose(1, 2).to(gu.dtype))
                ex.down_proj.copy_(wd.transpose(1, 2).to(ex.down_proj.dtype))
                continue
            E = ex.gate_up_proj.shape[0]
            ex.gate_up_proj.copy_(torch.cat([wg[:E], wu[:E]], dim=1).to(ex.gate_up_proj.dtype))
            ex.down_proj.copy_(wd[:E].to(ex.down_proj.dtype))
            if cfg["family"] == "deepseek":  # the shared MLP: experts E .. E + n - 1 of the state
                sh = b.shared_experts
                sh.gate_proj.weight.copy_(wg[E:].reshape(-1, wg.shape[-1]).to(sh.gate_proj.weight.dtype))
                sh.up_proj.weight.copy_(wu[E:].reshape(-1, wu.shape[-1]).to(sh.up_proj.weight.dtype))
                sh.down_proj.weight.copy_(torch.cat(list(wd[E:]), dim=1).to(sh.down_proj.weight.dtype))


def _forward(self, hidden_states):
    cfg = self._moeb
    shape = hidden_states.shape
    T = hidden_states.numel() // shape[-1]
    if T > cfg["max_tokens"] or self.training:
        return self._moeb_stock(hidden_states)
    x = hidden_states.reshape(T, shape[-1]).to(torch.bfloat16).contiguous()
    kw = cfg["kw"]
    if cfg["family"] == "gptoss":
        y, _, wts = cfg["mod"].layer(cfg["state"], x, _bf16(self.router.weight), kw["k"],
                                     gate_b=_bf16(self.router.bias), return_routing=True)
        return y.to(hidden_states.dtype).reshape(shape), wts.to(hidden_states.dtype)
    gate = self.gate.weight
    y = cfg["mod"].layer(cfg["state"], x, _bf16(gate), kw["k"], norm=kw["norm"], rscale=kw.get("rscale", 1.0))
    return y.to(hidden_states.dtype).reshape(shape)


def policy_for(T, block):
    """The expert kernel family the library picks for a T-token call of this block (for reports)."""
    st = block._moeb["state"]
    return ops.policy(T, st["E"], block._moeb["kw"]["k"])


# ------------------------------------------------------------------ attention over the 4-bit KV cache
ATTENTION, ATTENTION_SDPA = "moelab_b200_kv4", "moelab_b200_kv4_sdpa"


class _Length(int):
    """A mask's number of keys that comes from a 4-bit cache."""


class _Causal:
    """What a layer's attention gets in a mask's place with a 4-bit cache: causal, the last `window` keys (0: all)."""

    def __init__(self, window):
        self.window = window


def _kv_cache_class():
    """The cache class, made on first use (transformers is optional)."""
    global QuantizedKVCache
    if QuantizedKVCache is None:
        from transformers import DynamicCache

        class _QuantizedKVCache(DynamicCache):
            """Keys and values of every layer in 4 bits (ops.KVCache), `batch` sequences of equal length, up to `max_len`
            tokens each. Pass as past_key_values to a model patched with patch_hf_attention. Sequences advance together, so
            padded batches are refused (by the mask function), and so is what reorders or repeats them
            (beam search). crop() and reset() give tokens up."""

            def __init__(self, config, batch, max_len, fmt="q4", page_size=64, device="cuda"):
                super().__init__(config=config)
                cfg = self.moeb_config = config.get_text_config()
                dim = _head_dim(cfg)
                heads = getattr(cfg, "num_key_value_heads", None) or cfg.num_attention_heads
                per = -(-max_len // page_size)
                self.moeb_max, self.moeb_batch = int(max_len), int(batch)
                self.moeb_layers = [ops.KVCache(batch * per, heads, dim, page_size=page_size, fmt=fmt, device=device)
                                    for _ in range(cfg.num_hidden_layers)]
                dev = self.moeb_layers[0].device
                self.moeb_table = torch.arange(batch * per, dtype=torch.int32, device=dev).view(batch, per)
                self.moeb_lens = torch.zeros(batch, dtype=torch.int32, device=dev)
                self.moeb_seen, self.moeb_filled = [0] * cfg.num_hidden_layers, 0  # tokens of each layer; what moeb_lens holds

            def get_seq_length(self, layer_idx=0):
                return self.moeb_seen[layer_idx or 0]

            def get_mask_sizes(self, new, layer_idx=0):
                n = new if isinstance(new, int) else new.shape[0]
                return _Length(self.get_seq_length(layer_idx) + n), 0

            def crop(self, max_length):
                n = max_length if max_length >= 0 else self.get_seq_length() + max_length
                self.moeb_seen = [max(min(n, s), 0) for s in self.moeb_seen]

            def reset(self):
                self.crop(0)

            def _refuse(self, *_, **__):
                raise NotImplementedError("sequences of the 4-bit KV cache are not reordered, repeated or selected")

            reorder_cache = batch_repeat_interleave = batch_select_indices = _refuse

            def update(self, key_states, value_states, layer_idx, cache_kwargs=None):
                if self.moeb_config._attn_implementation not in (ATTENTION, ATTENTION_SDPA):
                    raise ValueError("the model's attention does not read the 4-bit KV cache: call patch_hf_attention(model) first, "
                                     "or go on with to_stock()")
                if _capturing(key_states):
                    raise RuntimeError("the 4-bit cache of a model counts its tokens on the host: a captured call would write the "
                                       "same places in every replay. Capture ops.kv_write and ops.kv_attention, which read lens")
                B, H, n, D = key_states.shape
                if B != self.moeb_batch:
                    raise ValueError(f"a batch of {B} sequences, the cache is for {self.moeb_batch}")
                seen = self.moeb_seen[layer_idx] + n
                if seen > self.moeb_max:
                    raise ValueError(f"{seen} tokens, the cache holds {self.moeb_max}")
                if seen != self.moeb_filled:  # by the first layer of a call that has attention
                    self.moeb_lens.fill_(seen)
                    self.moeb_filled = seen
                try:
                    ops.kv_write(self.moeb_layers[layer_idx], _rows(key_states), _rows(value_states), self.moeb_table,
                                 self.moeb_lens)
                except Exception:
                    self.moeb_undo(n)
                    raise
                self.moeb_seen[layer_idx] = seen
                key = key_states.view_as(key_states)  # a tensor of its own to mark
                key._moeb_kv = (self, layer_idx)
                return key, value_states

            def moeb_undo(self, n):
                """A call of n tokens ended early: the layers that had taken them give them up."""
                self.moeb_seen = [s - n if s == self.moeb_filled else s for s in self.moeb_seen]

            def to_stock(self):
                """A DynamicCache with the stored values in bf16, to continue on the stock attention."""
                out = DynamicCache()
                for i, c in enumerate(self.moeb_layers):
                    n = self.moeb_seen[i]
                    kv = ops.kv_read(c, self.moeb_table, None, self.moeb_batch * n)
                    out.update(*(t.view(self.moeb_batch, n, c.kv_heads, c.head_dim).transpose(1, 2) for t in kv), i)
                return out

        QuantizedKVCache = _QuantizedKVCache
    return QuantizedKVCache


QuantizedKVCache = None


def quantized_kv_cache(model, batch, max_len, fmt="q4", page_size=64):
    """A 4-bit cache for `model` (its layers' heads and widths): `batch` sequences of up to `max_len` tokens."""
    return _kv_cache_class()(model.config, batch, max_len, fmt, page_size, next(model.parameters()).device)


def _head_dim(cfg):
    if getattr(cfg, "kv_lora_rank", None):
        raise ValueError("latent attention (DeepSeek) has no per-head cache: not supported")
    other = set(getattr(cfg, "layer_types", None) or ()) - {"full_attention", "sliding_attention"}
    if other:
        raise ValueError(f"layers of full and sliding attention are supported, this model has {', '.join(sorted(other))}")
    if getattr(cfg, "attn_logit_softcapping", None) is not None:
        raise ValueError("capped attention scores (attn_logit_softcapping) are not supported by the 4-bit KV cache attention")
    dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
    if dim not in (64, 128):
        raise ValueError(f"heads of 64 or 128 values are supported, this model has {dim}")
    return dim


def _capturing(t):
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


def _rows(t):
    """[B, H, n, D] -> bf16 [B * n, H, D] (a view where the strides allow one)."""
    B, H, n, D = t.shape
    return t.detach().to(torch.bfloat16).transpose(1, 2).reshape(B * n, H, D)


class _NoBackward(torch.autograd.Function):
    """The first argument, as a function of the others whose backward pass is an error and not a missing term."""

    @staticmethod
    def forward(ctx, y, *inputs):
        return y.view_as(y)

    @staticmethod
    def backward(ctx, grad):
        raise NotImplementedError("the 4-bit KV cache has no backward pass: call the model without it, or under torch.no_grad()")


# What models hand to their attention function that the kernel has an argument for, or that changes nothing about a call's result.
_KNOWN = frozenset(("scaling", "sliding_window", "s_aux", "dropout", "is_causal", "position_ids", "cache_position", "use_cache",
                    "output_attentions", "output_hidden_states", "output_router_logits", "return_dict", "logits_to_keep",
                    "num_items_in_batch"))


def _cached_window(module, attention_mask, kw):
    """The window of a layer's call with a 4-bit cache; refuses what the kernel has no argument for."""
    if module.training:
        raise ValueError("the 4-bit KV cache has no backward pass: call model.eval() first")
    unknown = sorted(k for k, v in kw.items() if k not in _KNOWN and v is not None and v is not False)
    if unknown or kw.get("dropout") or kw.get("is_causal") is False or getattr(module, "is_causal", True) is False:
        raise ValueError(f"the 4-bit KV cache attention is causal, without dropout, and does not know {unknown or 'other kinds'}")
    window = int(kw.get("sliding_window") or 0)
    if isinstance(attention_mask, _Causal):
        if window and window != attention_mask.window:
            raise ValueError(f"a layer with a window of {window} and a mask with one of {attention_mask.window}")
        return attention_mask.window
    if attention_mask is not None:
        raise ValueError("attention masks of the caller's own are not supported by the 4-bit KV cache attention")
    return window


def _attention(module, query, key, value, attention_mask=None, **kw):
    B, H, n, D = query.shape
    tag = getattr(key, "_moeb_kv", None)
    if tag is not None:
        cache, layer = tag
        try:
            window = _cached_window(module, attention_mask, kw)
        except ValueError:
            cache.moeb_undo(n)  # a refused call leaves the cache as it was
            raise
        sinks = kw.get("s_aux")
        y = ops.kv_attention(_rows(query), cache.moeb_layers[layer], cache.moeb_table, cache.moeb_lens, scale=kw.get("scaling"),
                             window=window, sink_logits=None if sinks is None else sinks.detach().float())
        y = y.view(B, n, H, D).to(query.dtype)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (query, key, value, sinks)):
            y = _NoBackward.apply(y, query, key, value, sinks)
        return y, None
    return _stock_attention(module, query, key, value, attention_mask, **kw)


def _stock_attention(module, query, key, value, attention_mask, **kw):
    """A call without the 4-bit cache: the attention that the model ran before the patch (or the nearest, see _without)."""
    if isinstance(attention_mask, _Causal):
        raise ValueError(f"{type(module).__name__} does not hand the keys of the 4-bit KV cache to its attention as they are")
    if module.config._attn_implementation == ATTENTION_SDPA:
        from transformers import AttentionInterface
        return AttentionInterface()["sdpa"](module, query, key, value, attention_mask, **kw)
    if attention_mask is not None and attention_mask.dtype == torch.bool:  # the eager attention adds its mask
        attention_mask = torch.zeros_like(attention_mask, dtype=query.dtype).masked_fill(~attention_mask, torch.finfo(query.dtype).min)
    for c in type(module).__mro__:  # each model's file has its own
        eager = getattr(sys.modules.get(c.__module__), "eager_attention_forward", None)
        if eager is not None:
            return eager(module, query, key, value, attention_mask, **kw)
    raise ValueError(f"{type(module).__name__} has no eager attention to run a call without the 4-bit KV cache")


def _attention_mask(*args, **kw):
    return _mask("eager", *args, **kw)


def _attention_mask_sdpa(*args, **kw):
    return _mask("sdpa", *args, **kw)


def _same(f, g):
    """Whether two functions are the same code over equal values."""
    if not (callable(f) and callable(g)):
        if isinstance(f, tuple) and isinstance(g, tuple):
            return len(f) == len(g) and all(_same(x, y) for x, y in zip(f, g))
        return type(f) is type(g) is int and f == g
    if f is g:
        return True
    cells = [[c.cell_contents for c in getattr(x, "__closure__", None) or ()] for x in (f, g)]
    return getattr(f, "__code__", f) is getattr(g, "__code__", g) and _same(*map(tuple, cells))


def _window(mask_function, local_size):
    """The window of a mask function (0: plainly causal); any other (chunks, packed sequences, both directions) is refused."""
    from transformers import masking_utils as m
    if mask_function is None or _same(mask_function, m.causal_mask_function):
        return 0
    if local_size and _same(mask_function, m.sliding_window_causal_mask_function(local_size)):
        return int(local_size)
    raise ValueError("masks other than the causal one and its sliding window are not supported by the 4-bit KV cache attention")


def _mask(stock, *args, kv_length=None, attention_mask=None, **kw):
    """With a 4-bit cache no mask tensor: causality and the window are the kernel's; what it has no argument for and padded
    batches are refused here, in every call: a mask may come with single tokens too. Without one the mask of the stock attention."""
    if not isinstance(kv_length, _Length):
        from transformers import AttentionMaskInterface
        return AttentionMaskInterface()[stock](*args, kv_length=kv_length, attention_mask=attention_mask, **kw)
    if attention_mask is not None and not bool(attention_mask.bool().all()):  # waits for the device, as generate() does per token
        raise ValueError("padded batches are not supported by the 4-bit KV cache attention")
    return _Causal(_window(kw.get("mask_function"), kw.get("local_size")))


def _without(model, stock):
    """The name under which a model is patched: calls without the 4-bit cache keep its eager or sdpa attention; what ran on
    another kernel (flash, flex) runs on sdpa where the model has it."""
    return ATTENTION_SDPA if stock != "eager" and getattr(model, "_supports_sdpa", False) else ATTENTION


def patch_hf_attention(model):
    """Route the model's attention through the library for calls with a quantized_kv_cache (others run the stock attention).
    Returns the name of the implementation that unpatch_hf_attention restores."""
    from transformers import AttentionInterface, AttentionMaskInterface
    _head_dim(model.config.get_text_config())
    for name, mask in ((ATTENTION, _attention_mask), (ATTENTION_SDPA, _attention_mask_sdpa)):
        AttentionInterface.register(name, _attention)
        AttentionMaskInterface.register(name, mask)
    stock = model.config._attn_implementation
    if stock not in (ATTENTION, ATTENTION_SDPA):
        model._moeb_attention_stock = stock
        model.set_attn_implementation(_without(model, stock))
    return model._moeb_attention_stock


def unpatch_hf_attention(model):
    """Restore the stock attention. Returns whether the model was patched."""
    stock = model.__dict__.pop("_moeb_attention_stock", None)
    if stock is not None:
        model.set_attn_implementation(stock)
    return stock is not None
