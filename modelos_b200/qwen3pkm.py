"""Qwen3 with product-key memory layers (the consumer of the PKM path).

The reference's ``modeling_qwen3pkm.py`` builds a Qwen3 decoder whose layers
listed in ``config.pkm_layers`` replace the feed-forward block with a
``HashingMemory`` read (``modeling_qwen3pkm.py:318-333``): after the
post-attention RMSNorm the layer computes ``pkm(hidden)[0]`` instead of
``mlp(hidden)`` and adds it to the residual (``:699-707``).  Its memory is
built as ``HashingMemory(hidden, hidden, mem_k_dim=pkm_k_dim,
mem_v_dim=pkm_v_dim, mem_heads=pkm_heads, mem_knn=pkm_topk,
mem_n_keys=pkm_n_subkeys, mem_share_values=False,
mem_query_rmsnorm=pkm_query_rmsnorm)`` and re-initialised with
``reset_parameters`` (``:733-737``).

This module assembles the same network from transformers' own Qwen3 blocks
(``Qwen3ForCausalLM``) with this package's ``HashingMemory`` in those
positions, so the benchmark machine (which has transformers but not the
reference tree) can run the model: a training step, a prefill and a decode
loop.  ``reference_state_dict_names`` maps parameter names between this
assembly and the reference model (``layers.i.pkm.*`` there,
``layers.i.mlp.pkm.*`` here), which is how the CPU test checks the two give
the same logits from the same weights.

``attn_implementation="modelos_b200"`` runs the decoder's attention on this
package's kernels (``modelos_b200.attention``): training, prompts and single
tokens, full or sliding-window layers (the configuration's ``layer_types`` and
``sliding_window``), with ``attention_sinks`` first tokens that stay visible to
windowed layers.  ``QuantizedCache`` holds the keys and values of a generation
in 4 bits, as a cache of transformers.
"""
from __future__ import annotations

from typing import Iterable, Optional

import torch
from torch import nn

from . import _native
from .attention import MAX_ROWS, KVCache4, window_attention
from .pkm.memory import HashingMemory

ATTENTION = "modelos_b200"  # the attention implementation's name in transformers

# Benchmark config 3: a Qwen3-0.6B-shaped decoder with PKM layers of the
# config-2 geometry at layers 6, 12 and 18.
CONFIG3 = dict(vocab_size=151936, hidden_size=1024, intermediate_size=3072, num_hidden_layers=28,
               num_attention_heads=16, num_key_value_heads=8, head_dim=128, rms_norm_eps=1e-6,
               rope_theta=1_000_000.0, max_position_embeddings=40960, tie_word_embeddings=True)
PKM3 = dict(pkm_layers=(6, 12, 18), pkm_k_dim=512, pkm_v_dim=1024, pkm_heads=4, pkm_topk=32, pkm_n_subkeys=512,
            pkm_query_rmsnorm=True)


class PKMFeedForward(nn.Module):
    """The feed-forward slot of a PKM layer: ``HashingMemory(hidden)[0]``; the
    memory's indices of the last call stay in ``last_pkm_indices``."""

    def __init__(self, hidden: int, pkm_k_dim: int, pkm_v_dim: int, pkm_heads: int, pkm_topk: int,
                 pkm_n_subkeys: int, pkm_query_rmsnorm: bool):
        super().__init__()
        self.pkm = HashingMemory(input_dim=hidden, output_dim=hidden, mem_k_dim=pkm_k_dim, mem_v_dim=pkm_v_dim,
                                 mem_heads=pkm_heads, mem_knn=pkm_topk, mem_n_keys=pkm_n_subkeys,
                                 mem_share_values=False, mem_query_rmsnorm=pkm_query_rmsnorm)
        self.last_pkm_indices = None

    def forward(self, x):
        out, idx = self.pkm(x)
        self.last_pkm_indices = idx
        return out


def attention_bounds(attention_mask: torch.Tensor, kv_length: int, kv_offset: Optional[int] = None) -> torch.Tensor:
    """``[2, B]`` int32: the first real token of each row of a padding mask
    ``[B, tokens]`` among ``kv_length`` columns from ``kv_offset`` on (None: the
    last), and one past the last (equal where a row has none).  Real tokens must
    be consecutive: padding between them (a right-padded prompt that goes on) is
    refused, which waits for the mask; within a capture ``_native.check_device_errors``
    reports it after a replay."""
    first = attention_mask.shape[1] - kv_length if kv_offset is None else kv_offset
    m = (attention_mask[:, max(first, 0):first + kv_length] != 0).to(torch.int32)
    first = m.argmax(1)
    last = m.shape[1] - m.flip(1).argmax(1)
    last = torch.where(m.any(1), last, first)
    holes = (last - first != m.sum(1)).any()
    if m.is_cuda and torch.cuda.is_current_stream_capturing():
        _native.err_word(m.device).bitwise_or_(holes.to(torch.int32) * _native.DEVERR_MASK)
    elif holes:
        raise ValueError(_native.MASK_HOLES)
    return torch.stack((first, last)).to(torch.int32)


def _alike(f, g) -> bool:
    """Whether two mask functions are the same code over functions that are
    alike (numbers that they hold, as a window, may differ)."""
    def inner(h):
        for cell in h.__closure__ or ():
            held = cell.cell_contents
            yield from (x for x in (held if isinstance(held, (tuple, list)) else (held,)) if callable(x))

    if getattr(f, "__code__", None) is None or f.__code__ is not g.__code__:
        return False
    a, b = list(inner(f)), list(inner(g))
    return len(a) == len(b) and all(map(_alike, a, b))


def _attention_mask(batch_size, q_length, kv_length, q_offset=0, kv_offset=0, mask_function=None, attention_mask=None,
                    allow_is_causal_skip=True, use_vmap=False, config=None, **kwargs):
    """What transformers hands to ``_attention`` as the mask: None or the
    rows' bounds; causality, window and sinks are the kernels' own."""
    from transformers.masking_utils import causal_mask_function, sliding_window_causal_mask_function

    # (chunked, bidirectional and a caller's own masks arrive as a function only)
    known = mask_function is None or any(
        _alike(mask_function, f) for f in (causal_mask_function, sliding_window_causal_mask_function(1)))
    if use_vmap or not allow_is_causal_skip or not known:
        raise ValueError("modelos_b200 attention: only causal and sliding-window masks with padding are implemented "
                         "(no packed sequences, no chunked, bidirectional or overlaid masks, no static cache)")
    if kv_offset and getattr(config, "attention_sinks", 0):
        raise ValueError("modelos_b200 attention: this cache has dropped the first tokens, which attention_sinks needs; "
                         "pass past_key_values=QuantizedCache(...) or a cache without sliding layers")
    if attention_mask is None:
        return None
    # a column of the mask is a position; it may have columns for tokens to come
    # (without a cache kv_length is the mask's width, whatever the keys' number)
    kv_length = min(kv_length, q_offset + q_length - kv_offset)
    if attention_mask.shape[1] < kv_offset + kv_length:
        raise ValueError(f"modelos_b200 attention: the mask has {attention_mask.shape[1]} columns for "
                         f"{kv_offset + kv_length} tokens")
    bounds = attention_bounds(attention_mask, kv_length, kv_offset)
    # where all queries are padding, nothing is visible (KVCache4.attend takes no ends)
    bounds[0].masked_fill_(bounds[1] <= kv_length - q_length, kv_length)
    return bounds


# arguments of other models' attention that change its result (score caps, a
# sink's logit, biases, packed lengths); what else comes along, as position_ids, does not
_CHANGES = ("softcap", "s_aux", "position_bias", "head_mask", "cu_seq_lens_q", "cu_seq_lens_k")


def _attention(module, query, key, value, attention_mask, scaling=None, dropout=0.0, sliding_window=None,
               is_causal=None, **kwargs):
    """transformers' attention interface: ``(output [B, T, heads, D], None)``."""
    if dropout:
        raise ValueError("modelos_b200 attention: attention dropout is not implemented")
    for name in _CHANGES:
        if kwargs.get(name) is not None:
            raise ValueError(f"modelos_b200 attention: {name} is not implemented")
    # (one query sees all keys either way)
    if query.shape[2] > 1 and not (getattr(module, "is_causal", True) if is_causal is None else is_causal):
        raise ValueError("modelos_b200 attention: only causal attention is implemented (is_causal is False)")
    sinks = getattr(module.config, "attention_sinks", 0) if sliding_window else 0
    if attention_mask is not None and (attention_mask.dim() != 2 or attention_mask.dtype != torch.int32):
        raise ValueError("modelos_b200 attention: masks written out are not implemented; pass a padding mask [batch, tokens]")
    starts, ends = (None, None) if attention_mask is None else attention_mask.unbind()
    if isinstance(key, KVCache4):
        out = key.attend(query, window=sliding_window, sinks=sinks, scale=scaling, starts=starts)
        if ends is not None and query.shape[2] > 1:  # (a token alone: its starts say so)
            at = key.lengths[:, None] - query.shape[2] + torch.arange(query.shape[2], device=query.device)
            out = out.masked_fill((at >= ends[:, None])[:, None, :, None], 0)
    else:
        out = window_attention(query, key, value, window=sliding_window, sinks=sinks, scale=scaling, starts=starts,
                               ends=ends)
    return out.transpose(1, 2), None


def register_attention():
    """Make ``ATTENTION`` known to transformers (``build_qwen3_pkm`` does it)."""
    from transformers import AttentionInterface, AttentionMaskInterface

    AttentionInterface.register(ATTENTION, _attention)
    AttentionMaskInterface.register(ATTENTION, _attention_mask)


def _quantized_cache_types():
    from transformers.cache_utils import Cache, CacheLayerMixin

    class Layer(CacheLayerMixin):
        """One layer's keys and values in 4 bits; every row at the same length
        (padding is part of a row, as in transformers' other caches)."""

        is_sliding = False

        def __init__(self, max_len: int):
            super().__init__()
            self.max_len, self.cache, self.tokens = max_len, None, 0

        def lazy_initialization(self, key_states, value_states):
            B, H, _, D = key_states.shape
            self.dtype, self.device = key_states.dtype, key_states.device
            self.cache = KVCache4(B, H, self.max_len, D, dtype=self.dtype, device=self.device)
            self.is_initialized = True

        def update(self, key_states, value_states, *args, **kwargs):
            if not self.is_initialized:
                self.lazy_initialization(key_states, value_states)
            first, n = self.tokens == 0, key_states.shape[2]
            if self.tokens + n > self.max_len:
                raise ValueError(f"QuantizedCache holds {self.max_len} tokens, {self.tokens + n} needed")
            self.cache.append(key_states, value_states)
            self.tokens += n
            if first:  # a prompt attends over its own keys and values
                return key_states, value_states
            if n <= self.short:  # the attention reads the codes
                return self.cache, self.cache
            return self.cache.read(0, self.tokens)

        short = 1  # tokens to a call that attend over the codes; more read the values back

        def get_mask_sizes(self, query_length):
            return self.tokens + query_length, 0

        def get_seq_length(self):
            return self.tokens

        def get_max_cache_shape(self):
            return self.max_len

        def crop(self, max_length):
            n = max_length if max_length >= 0 else max(self.tokens + max_length, 0)
            if n < self.tokens:
                self.tokens = n
                self.cache.lengths.fill_(n)

        def reset(self):
            self.crop(0)

        def _pick(self, pick):
            if self.is_initialized:
                c = self.cache
                self.cache = KVCache4.wrap(*(pick(t).contiguous() for t in (c.k_codes, c.k_params, c.v_codes,
                                                                            c.v_params, c.lengths)))

        def reorder_cache(self, beam_idx):
            self._pick(lambda t: t.index_select(0, beam_idx.to(t.device)))

        def batch_repeat_interleave(self, repeats):
            self._pick(lambda t: t.repeat_interleave(repeats, dim=0))

        def batch_select_indices(self, indices):
            self._pick(lambda t: t[indices])

    return Cache, Layer


def QuantizedCache(config, max_len: int):
    """A transformers cache (``past_key_values``) for a model built with
    ``attn_implementation="modelos_b200"``: ``max_len`` tokens of every layer's
    keys and values in 4 bits (``KVCache4``: 0.31 of a 16-bit cache).  The
    prompt attends over its own 16-bit keys and values, later tokens over the
    cache's.  Every layer keeps all tokens, windowed or not, so that sinks stay;
    a windowed layer reads only what its window and sinks show."""
    Cache, Layer = _quantized_cache_types()
    layers = [Layer(max_len) for _ in range(config.num_hidden_layers)]
    for layer in layers:
        layer.short = MAX_ROWS // (config.num_attention_heads // config.num_key_value_heads)
    return Cache(layers=layers)


def build_qwen3_pkm(model_kw: Optional[dict] = None, pkm_kw: Optional[dict] = None,
                    attn_implementation: str = "sdpa", dtype=torch.bfloat16, device=None, seed: int = 0,
                    attention_sinks: int = 0):
    """A ``Qwen3ForCausalLM`` (random init) whose ``pkm_layers`` carry a
    ``PKMFeedForward`` in place of the MLP, re-initialised like the
    reference (``reset_parameters`` of every memory).

    ``attn_implementation="modelos_b200"`` uses this package's attention;
    ``attention_sinks`` first tokens then stay visible to sliding-window
    layers (``model_kw``: ``use_sliding_window``, ``sliding_window``,
    ``max_window_layers`` or ``layer_types``)."""
    from transformers import Qwen3Config, Qwen3ForCausalLM

    if attn_implementation == ATTENTION:
        register_attention()
    elif attention_sinks:
        raise ValueError(f"attention_sinks needs attn_implementation={ATTENTION!r}")
    mk = dict(CONFIG3)
    mk.update(model_kw or {})
    pk = dict(PKM3)
    pk.update(pkm_kw or {})
    layers: Iterable[int] = pk.pop("pkm_layers")
    cfg = Qwen3Config(**mk)
    cfg._attn_implementation = attn_implementation
    cfg.attention_sinks = int(attention_sinks)
    torch.manual_seed(seed)
    model = Qwen3ForCausalLM(cfg)
    for i in layers:
        ff = PKMFeedForward(mk["hidden_size"], **pk)
        ff.pkm.reset_parameters()
        model.model.layers[i].mlp = ff
    return model.to(device=device, dtype=dtype)


def reference_state_dict_names(name: str) -> str:
    """This assembly's parameter name for a name of the reference model
    (``model.layers.i.pkm.*`` -> ``model.layers.i.mlp.pkm.*``)."""
    parts = name.split(".")
    if len(parts) > 3 and parts[0] == "model" and parts[1] == "layers" and parts[3] == "pkm":
        return ".".join(parts[:3] + ["mlp"] + parts[3:])
    return name
