"""Few query rows over 16-bit keys: the output is off by its own rounding, not
by the probabilities' (which take part with their remainders)."""
from __future__ import annotations

import pytest
import torch

import attnref
from test_attention_gpu import make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (HF, 128), (HF, 64), (BF, 40)])
@pytest.mark.parametrize("shape", [(2, 4, 2, 1, 30), (2, 4, 2, 1, 300), (3, 8, 2, 3, 50), (1, 4, 2, 4, 900),
                                   (1, 16, 1, 1, 70)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (25, 3)])
def test_output(dtype, D, shape, window, sinks):
    from modelos_b200.attention import window_attention
    q, k, v, _ = make(*shape, D, dtype, seed=D + shape[-1])
    scale = D ** -0.5
    out = window_attention(q, k, v, window=window, sinks=sinks)
    see = attnref.visible(shape[0], shape[3], shape[4], window, sinks, None, None, device=DEV)
    ks, vs = attnref.spread(k.double(), shape[1]), attnref.spread(v.double(), shape[1])
    want, _, p = attnref.forward(q.double(), ks, vs, see, scale)
    u = torch.finfo(dtype).eps / 2
    # a score in 32 bits: D products, the scaling and the maximum's subtraction; the exponential's own error (2^-22)
    size = (q.double().abs() @ ks.abs().transpose(-1, -2)) * scale
    E = 2.0 ** -20 + (D + 8) * attnref.F32 * (size * see).amax().item()
    n = see.sum(-1).amax().item()
    a = p @ vs.abs()
    # the first part of a probability is rounded down, by up to 2 u of it, and the
    # remainder to the nearest, by u of that; below fp16's normal range half its smallest step
    least = torch.finfo(dtype).smallest_normal * u
    tol = u * want.abs() * (1 + u) + (2.02 * u * u + 2 * E + (n + 16) * attnref.F32) * a
    tol += 2 * least * (see.double() @ vs.abs())  # (a remainder of 0 is held as the smallest number, two halves of a step)
    attnref.within(out, want, tol, "out")
