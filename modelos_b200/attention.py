"""Windowed attention with sink tokens, and a key/value cache held in 4 bits.

The attention half of the Qwen3-PKM decoder layers (the reference takes it
from transformers' attention interface, ``modeling_qwen3pkm.py:302-333``) on
the library's kernels:

* ``window_attention``: causal attention in which a query sees the last
  ``window`` tokens and the sequence's first ``sinks`` tokens; forward and
  backward pass, prompts, chunks of prompts and single tokens;
* ``KVCache4``: keys and values quantised to 4 bits as they are written, read
  back, and attended over without being unpacked in memory.

There is no CPU path.  bf16 and fp16; statistics and sums in fp32.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native

GROUP = 32  # channels that share a step and an offset in the 4-bit cache
MAX_ROWS = 64  # query rows (tokens x grouped heads) to a KV head in KVCache4.attend


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError("modelos_b200 attention: " + what)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: Optional[int] = None,
                     sinks: int = 0, scale: Optional[float] = None, starts: Optional[torch.Tensor] = None,
                     ends: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over the last ``window`` keys and the first ``sinks``.

    ``q`` [B, heads, Tq, D], ``k`` and ``v`` [B, kv_heads, Tk, D]; bf16 or
    fp16, any strides, D a multiple of 8 up to 128, ``heads`` a multiple of
    ``kv_heads``, ``Tk >= Tq``.  Query ``i`` stands at row ``p = i + Tk - Tq``;
    key ``j`` is visible to it when ``starts[b] <= j <= p < ends[b]`` and
    ``window`` is 0 or None, or ``j > p - window``, or ``j < starts[b] +
    sinks``.  ``starts`` / ``ends`` (integers [B], default 0 / Tk) are the rows
    each sequence occupies in a padded batch; padding rows may hold anything,
    their output is 0 and their gradients are 0.  ``scale`` defaults to
    ``D ** -0.5``.

    Returns [B, heads, Tq, D], laid out in memory as ``q`` is ([B, T, heads,
    D] or contiguous).  Differentiable once in q, k and v, backwards (tensors
    with a forward-mode tangent are refused); results are deterministic.  May be
    captured into a graph, also with its backward pass: refused
    (``RuntimeError``) while an eager graph of the default stream holds leaves
    among q, k and v, whose gradients would be accumulated there.
    """
    return _native.attention().window_attention(q, k, v, window or 0, sinks, scale, starts, ends)


class KVCache4:
    """Keys and values of ``batch`` sequences, at most ``max_len`` tokens each,
    held in 4 bits.

    Each side has ``codes`` uint8 [batch, kv_heads, max_len, head_dim/2]
    (channel 2i in the low half of byte i) and ``params`` [batch, kv_heads,
    max_len, head_dim/32, 2] in ``dtype``: the step and the offset of each
    group of 32 channels of one token and head.  offset = min, step =
    (max - min) / 15 rounded to ``dtype``, code = (x - offset) / step rounded
    to the nearest integer, value = code * step + offset rounded to ``dtype``.
    A group holding a NaN or an infinity reads back as NaN.

    ``lengths`` (int32 [batch], on the device) are the tokens that each
    sequence holds.  No call synchronises; a token whose row lies outside the
    cache is dropped and reported by ``_native.check_device_errors`` (as an
    ``IndexError``).
    """

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device: Union[str, torch.device] = "cuda"):
        def side():
            return (torch.zeros((batch, kv_heads, max_len, head_dim // 2), dtype=torch.uint8, device=device),
                    torch.zeros((batch, kv_heads, max_len, head_dim // GROUP, 2), dtype=dtype, device=device))

        _need(head_dim in (64, 128), "the 4-bit cache takes head_dim 64 or 128")
        self._set(*side(), *side(), torch.zeros(batch, dtype=torch.int32, device=device))

    @classmethod
    def wrap(cls, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor,
             lengths: Optional[torch.Tensor] = None) -> "KVCache4":
        """A cache over the caller's own tensors.  Without ``lengths`` it can be
        written and read at given rows, not appended to or attended over."""
        self = cls.__new__(cls)
        self._set(k_codes, k_params, v_codes, v_params, lengths)
        return self

    def _set(self, k_codes, k_params, v_codes, v_params, lengths):
        _need(k_codes.dim() == 4 and k_codes.dtype == torch.uint8 and k_codes.shape[3] in (32, 64),
              "codes must be uint8 [batch, kv_heads, max_len, head_dim/2], head_dim 64 or 128")
        B, H, cap, half = k_codes.shape
        want = (B, H, cap, 2 * half // GROUP, 2)
        _need(v_codes.shape == k_codes.shape and v_codes.dtype == torch.uint8, "k and v codes must match")
        _need(k_params.shape == want and v_params.shape == want,
              "params must be [batch, kv_heads, max_len, head_dim/32, 2]")
        _need(k_params.dtype == v_params.dtype and k_params.dtype in (torch.bfloat16, torch.float16),
              "params must be bf16 or fp16")
        for t in (k_codes, k_params, v_codes, v_params):
            _need(t.is_contiguous() and t.data_ptr() % 16 == 0, "cache tensors must be contiguous and 16-byte aligned")
            _need(t.device == k_codes.device, "cache tensors must be on one device")
        if lengths is not None:
            _need(lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.device == k_codes.device
                  and lengths.is_contiguous(), "lengths must be int32 [batch] on the cache's device")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.lengths = lengths

    batch = property(lambda self: self.k_codes.shape[0])
    kv_heads = property(lambda self: self.k_codes.shape[1])
    max_len = property(lambda self: self.k_codes.shape[2])
    head_dim = property(lambda self: 2 * self.k_codes.shape[3])
    dtype = property(lambda self: self.k_params.dtype)
    device = property(lambda self: self.k_codes.device)

    @property
    def nbytes(self) -> int:
        """Bytes of the codes and params of both sides."""
        return sum(t.numel() * t.element_size() for t in self._tensors())

    def _tensors(self):
        return self.k_codes, self.k_params, self.v_codes, self.v_params

    def write(self, k: torch.Tensor, v: torch.Tensor, at: Union[int, torch.Tensor]):
        """Quantise ``k`` and ``v`` [batch, kv_heads, T, head_dim] into rows
        ``at .. at + T - 1`` of every sequence (``at``: one row number, or one
        a sequence as integers [batch] on the device).  ``lengths`` stay."""
        rows = at if isinstance(at, torch.Tensor) else None
        _native.attention().kv4_write(k, v, rows, -1 if rows is not None else at, self.k_codes, self.k_params,
                                      self.v_codes, self.v_params)

    def append(self, k: torch.Tensor, v: torch.Tensor):
        """``write`` behind each sequence's tokens, and count them."""
        _need(self.lengths is not None, "append needs lengths")
        self.write(k, v, self.lengths)
        self.lengths.add_(k.shape[2]).clamp_(max=self.max_len)

    def read(self, at: Union[int, torch.Tensor], count: int):
        """``(k, v)`` [batch, kv_heads, count, head_dim]: the values of rows
        ``at .. at + count - 1`` (``at`` as in ``write``)."""
        rows = at if isinstance(at, torch.Tensor) else None
        return _native.attention().kv4_read(self.k_codes, self.k_params, self.v_codes, self.v_params, rows,
                                            -1 if rows is not None else at, count)

    def attend(self, q: torch.Tensor, *, window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None,
               starts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``window_attention`` of ``q`` [batch, heads, Tq, head_dim] over the
        cache's values, query ``i`` of a sequence at its row ``length - Tq +
        i`` (append the queries' own keys first).  ``starts`` as in
        ``window_attention``; rows behind a sequence's length are not read.
        ``Tq * heads / kv_heads`` is at most 64: ``read`` the cache and call
        ``window_attention`` for longer runs of queries.  Not differentiable."""
        _need(self.lengths is not None, "attend needs lengths")
        return _native.attention().kv4_attend(q, self.k_codes, self.k_params, self.v_codes, self.v_params, window or 0,
                                              sinks, scale, starts, self.lengths)
