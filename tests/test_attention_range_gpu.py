"""Gradients of fp16 attention whose intermediate values leave fp16's range
though the gradients do not, against 64 bits."""
from __future__ import annotations

import pytest
import torch

import attnref

pytestmark = pytest.mark.gpu
DEV = "cuda"
HF = torch.float16


def gradients(q, k, v, dout, scale, window=0, sinks=0):
    from modelos_b200.attention import window_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(window_attention(*leaves, window=window, sinks=sinks, scale=scale), leaves, dout)


def randn(*shape, seed, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(HF)


def test_sinks_whose_sums_pass_the_range_on_the_way():
    """The first keys' dv: some queries add about 400,000, as many take it away
    again."""
    T, D = 1300, 64
    q, k, v = (randn(1, 1, T, D, seed=i, size=0.5) for i in (9, 10, 11))
    dout = randn(1, 1, T, D, seed=12, size=0.01)
    dout[:, :, 300:800] += 30000
    dout[:, :, 800:] -= 30000
    r = attnref.reference(q, k, v, 33, 4, 1e-3, None, None, dout)
    assert r["dv"].abs().max() < 6e4
    for name, x in zip(("dq", "dk", "dv"), gradients(q, k, v, dout, 1e-3, 33, 4)):
        attnref.within(x, r[name], r[name + "_tol"], name)
