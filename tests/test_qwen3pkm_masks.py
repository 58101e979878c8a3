"""What transformers may hand to this package's attention as mask and
arguments: right, or refused.  Without a GPU (stand-ins of the kernels), but for
what a capture does."""
from __future__ import annotations

import pytest
import torch

import attnref
import fake_native
from modelos_b200 import qwen3pkm

BF = torch.bfloat16
MODEL = dict(vocab_size=96, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=2, head_dim=64, max_position_embeddings=512, tie_word_embeddings=False)
WINDOW = dict(use_sliding_window=True, sliding_window=6, max_window_layers=1)  # the first layer sees everything


@pytest.fixture(autouse=True)
def stand_in(monkeypatch, request):
    if request.node.get_closest_marker("gpu"):
        return
    fake_native.install(monkeypatch)
    attnref.install(monkeypatch)


def model(kw, **extra):
    return qwen3pkm.build_qwen3_pkm(dict(MODEL, **kw), dict(pkm_layers=[]), qwen3pkm.ATTENTION, dtype=BF, device="cpu",
                                    **extra).eval()


def ids(B, T):
    return torch.randint(0, 96, (B, T), generator=torch.Generator().manual_seed(1))


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("kw", [{}, WINDOW])
@pytest.mark.parametrize("quantized", [False, True])
def test_a_mask_wider_than_the_keys_so_far(kw, quantized):
    """A prompt in chunks, each called with the whole batch's mask: columns are
    key positions."""
    m = model(kw)
    x, mask = ids(2, 12), torch.ones(2, 12, dtype=torch.long)
    mask[1, :5] = 0
    cache = qwen3pkm.QuantizedCache(m.config, 16) if quantized else None
    with torch.no_grad():
        want = m(x[:, :8], attention_mask=mask[:, :8], use_cache=False).logits
        out = m(x[:, :8], attention_mask=mask, past_key_values=cache, use_cache=True)
        real = mask[:, :8].bool()
        assert torch.equal(out.logits[real], want[real])
        out = m(x[:, 8:10], attention_mask=mask, past_key_values=out.past_key_values)
        want = m(x[:, :10], attention_mask=mask[:, :10], use_cache=False).logits[:, 8:]
    # one chunk or two, the same roundings up to their order; 4 bits lose 0.08 of keys and of values in two layers:
    # 0.08 * 4 ** 0.5
    assert rel(out.logits, want) < (0.16 if quantized else 2.0 ** -6)


def test_a_mask_of_fewer_columns_than_keys_is_refused():
    with pytest.raises(ValueError, match="columns"):
        qwen3pkm._attention_mask(2, 1, 9, q_offset=8, attention_mask=torch.ones(2, 1, dtype=torch.long))


def test_bounds_count_columns_from_the_first_key():
    m = torch.tensor([[0, 0, 1, 1, 1, 1], [1, 1, 1, 1, 1, 0], [0, 0, 0, 0, 0, 1]])
    assert qwen3pkm.attention_bounds(m, 4, 0).tolist() == [[2, 0, 0], [4, 4, 0]]
    assert qwen3pkm.attention_bounds(m, 3, 1).tolist() == [[1, 0, 0], [3, 3, 0]]


def test_masks_with_holes_are_refused():
    """A right-padded prompt that goes on: the padding lies between real tokens."""
    m = model({})
    x, mask = ids(2, 6), torch.tensor([[1, 1, 1, 1, 1, 1], [1, 1, 0, 0, 0, 1]])
    with torch.no_grad():
        out = m(x[:, :5], attention_mask=mask[:, :5], use_cache=True)
        with pytest.raises(ValueError, match="between"):
            m(x[:, 5:], attention_mask=mask, past_key_values=out.past_key_values)
        with pytest.raises(ValueError, match="between"):
            m(x, attention_mask=mask, use_cache=False)
        # behind the last query, and before the first key, they are not seen
        mask[1] = torch.tensor([1, 1, 1, 0, 0, 1])
        m(x[:, :5], attention_mask=mask, use_cache=False)
    holes = torch.tensor([[1, 0, 1, 1]])
    assert qwen3pkm._attention_mask(1, 1, 2, q_offset=3, kv_offset=2, attention_mask=holes).tolist() == [[0], [2]]
    with pytest.raises(ValueError, match="between"):
        qwen3pkm._attention_mask(1, 1, 3, q_offset=2, kv_offset=0, attention_mask=holes)
    # what is not 0 is real
    assert qwen3pkm._attention_mask(1, 3, 3, attention_mask=torch.tensor([[0, 2, 255]])).tolist() == [[1], [3]]


@pytest.mark.gpu
def test_a_captured_mask_with_holes_is_reported():
    """A capture cannot wait for the mask: its replays report it."""
    from modelos_b200 import _native
    mask = torch.ones(2, 6, dtype=torch.long, device="cuda")
    _native.check_device_errors()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bounds = qwen3pkm._attention_mask(2, 6, 6, attention_mask=mask)
    graph.replay()
    _native.check_device_errors()
    assert bounds.tolist() == [[0, 0], [6, 6]]
    mask[1, 2] = 0
    graph.replay()
    with pytest.raises(ValueError, match="between"):
        _native.check_device_errors()
    _native.check_device_errors()


def test_masks_that_are_not_causal_are_refused():
    """transformers' other masks arrive as a function, not as a tensor."""
    from transformers import masking_utils as mu
    m = model(WINDOW)
    x = torch.zeros(2, 8, 64, dtype=BF)
    kw = dict(inputs_embeds=x, attention_mask=None, past_key_values=None)
    assert mu.create_causal_mask(m.config, **kw) is None
    assert mu.create_sliding_window_causal_mask(m.config, **kw) is None
    m.config.attention_chunk_size = 4
    with pytest.raises(ValueError, match="only causal"):
        mu.create_chunked_causal_mask(m.config, **kw)
    for f in (mu.bidirectional_mask_function, mu.chunked_causal_mask_function(4, torch.zeros(2, dtype=torch.long)),
              mu.and_masks(mu.causal_mask_function, lambda b, h, q, k: k != 3),
              mu.or_masks(mu.causal_mask_function, mu.causal_mask_function),
              lambda b, h, q, k: k <= q):
        with pytest.raises(ValueError, match="only causal"):
            qwen3pkm._attention_mask(2, 8, 8, mask_function=f)
    for f in (mu.causal_mask_function, mu.sliding_window_causal_mask_function(3)):
        assert qwen3pkm._attention_mask(2, 8, 8, mask_function=f) is None
    with pytest.raises(ValueError, match="only causal"):
        mu.create_bidirectional_mask(m.config, inputs_embeds=x, attention_mask=torch.ones(2, 8))


def test_written_out_masks_are_refused():
    m = model({})
    with pytest.raises(ValueError, match="padding mask"):
        m(ids(2, 8), attention_mask=torch.zeros(2, 1, 8, 8, dtype=BF), use_cache=False)


@pytest.mark.parametrize("what", [dict(softcap=30.0), dict(s_aux=torch.zeros(4)), dict(is_causal=False),
                                  dict(position_bias=torch.zeros(1)), dict(head_mask=torch.ones(4)),
                                  dict(cu_seq_lens_q=torch.tensor([0, 4, 8])), dict(cu_seq_lens_k=torch.tensor([0, 4, 8]))])
def test_arguments_that_change_the_result_are_refused(what):
    """Score caps, a sink's logit, biases, packed lengths, an encoder's attention."""
    class Module:
        config = None
        is_causal = True

    q, k = torch.zeros(1, 4, 8, 64, dtype=BF), torch.zeros(1, 2, 8, 64, dtype=BF)
    with pytest.raises(ValueError, match=next(iter(what))):
        qwen3pkm._attention(Module, q, k, k, None, **what)
    none = {name: None for name in what}
    out, _ = qwen3pkm._attention(Module, q, k, k, None, position_ids=torch.zeros(1, 8), use_cache=True, **none)
    assert out.shape == (1, 8, 4, 64)


def test_modules_that_are_not_causal_are_refused():
    class Module:
        config = None
        is_causal = False

    q = torch.zeros(1, 4, 8, 64, dtype=BF)
    with pytest.raises(ValueError, match="is_causal"):
        qwen3pkm._attention(Module, q, q, q, None)
    qwen3pkm._attention(Module, q, q, q, None, is_causal=True)
    qwen3pkm._attention(Module, q[:, :, :1], q, q, None)  # one query sees all keys either way


@pytest.mark.parametrize("kw", [{}, WINDOW])
def test_rows_whose_tokens_are_all_padding_over_the_4_bit_cache(kw):
    """A row without real tokens, and one that has ended: as over the 16-bit cache,
    their tokens see nothing."""
    m = model(kw)
    x, mask = ids(3, 12), torch.ones(3, 12, dtype=torch.long)
    mask[1] = 0
    mask[2, 8:] = 0
    logits = []
    with torch.no_grad():
        for cache in (None, qwen3pkm.QuantizedCache(m.config, 16)):
            out = m(x[:, :8], attention_mask=mask[:, :8], past_key_values=cache, use_cache=True)
            steps = []
            for a, b in ((8, 9), (9, 12)):
                out = m(x[:, a:b], attention_mask=mask[:, :b], past_key_values=out.past_key_values)
                steps.append(out.logits[1:])
            logits.append(torch.cat(steps, 1))
    assert torch.equal(*logits)  # (the attention's output is 0 in every layer)


def test_padding_behind_a_few_tokens_over_the_4_bit_cache():
    """Some of a few tokens are padding: they see nothing, as over the 16-bit cache,
    so that their logits come from themselves alone."""
    m = model(WINDOW)
    x, mask = ids(3, 12), torch.ones(3, 12, dtype=torch.long)
    mask[1, 10:] = 0
    mask[2, 11:] = 0
    logits = []
    with torch.no_grad():
        for cache in (None, qwen3pkm.QuantizedCache(m.config, 16)):
            out = m(x[:, :8], attention_mask=mask[:, :8], past_key_values=cache, use_cache=True)
            logits.append(m(x[:, 8:], attention_mask=mask, past_key_values=out.past_key_values).logits)
    padding = ~mask[:, 8:].bool()
    assert torch.equal(logits[0][padding], logits[1][padding])
    assert rel(logits[1], logits[0]) < 0.16  # 4 bits in two layers: 0.08 * 4 ** 0.5
