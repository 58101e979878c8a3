"""What the forward pass keeps for the backward pass: the output and what its
rounding left are together the output without that rounding."""
from __future__ import annotations

import ctypes

import pytest
import torch

import attnref
from test_attention_gpu import ints, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def forward(q, k, v, scale, window, sinks, starts, ends):
    from modelos_b200 import _native

    def p(t):
        return None if t is None else ctypes.c_void_p(t.data_ptr())

    def s(t):
        return (ctypes.c_int64 * 3)(*t.stride()[:3])

    L = _native.lib()
    sizes = (*q.shape[:2], k.shape[1], q.shape[2], k.shape[2], q.shape[3])
    out, lo = torch.empty_like(q), torch.empty_like(q)
    lse = torch.empty(q.shape[:3], device=DEV)
    n = ctypes.c_size_t(0)
    assert L.pkm_attn_fwd_workspace(*sizes, window, sinks, ctypes.byref(n)) == 0
    ws = torch.empty(n.value + 16, dtype=torch.uint8, device=DEV)
    assert L.pkm_attn_fwd(p(q), s(q), p(k), s(k), p(v), s(v), _native.DT[q.dtype], *sizes, scale, window, sinks,
                          p(starts), p(ends), p(out), s(out), p(lo), p(lse), p(ws), n.value, None,
                          torch.cuda.current_stream().cuda_stream) == 0
    return out, lo


# tiles; keys shared by several blocks; few rows, alone and over a cluster
SHAPES = [(2, 4, 2, 300, 300), (1, 2, 1, 130, 1500), (2, 4, 2, 5, 40), (1, 4, 2, 3, 900)]
TYPES = [(BF, 128), (HF, 64), (BF, 72)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_output_and_its_remainder(shape, dtype, D, window, sinks):
    q, k, v, _ = make(*shape, D, dtype, seed=shape[-1])
    starts = ints(*([0] + [11] * (shape[0] - 1)))
    out, lo = forward(q, k, v, 0.2, window, sinks, starts, None)
    r = attnref.reference(q, k, v, window, sinks, 0.2, starts)
    u = torch.finfo(dtype).eps / 2
    # the bound without the output's rounding; the remainder's own is u of the remainder
    tol = r["out_tol"] - (u - 1.01 * u * u) * r["out"].abs()
    got = out.double() + lo.double()
    assert ((got - r["out"]).abs() <= tol + 2.0 ** -25).all()
    # it is a remainder: at most half a step, and not nothing
    assert (lo.double().abs() <= u * out.double().abs() * (1 + 2 * u) + 2.0 ** -25).all()
    assert (lo != 0).float().mean() > 0.5


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,D", TYPES)
def test_remainder_of_a_mean(shape, dtype, D):
    """All scores 0: the probabilities are exact, and only sums in 32 bits (with
    the weights of a split's parts, the exponentials of a difference of two
    logarithms in 32 bits, some 2^-20) and the remainder's rounding are left."""
    q, k, v, _ = make(*shape, D, dtype, seed=shape[-1])
    out, lo = forward(torch.zeros_like(q), k, v, 0.2, 0, 0, None, None)
    see = attnref.visible(*q.shape[:1], *shape[3:], 0, 0, None, None, device=DEV).double()
    vs = attnref.spread(v.double(), q.shape[1])
    p = see / see.sum(-1, keepdim=True)
    u = torch.finfo(dtype).eps / 2
    tol = ((shape[-1] + 32) * attnref.F32 + 2.0 ** -19) * (p @ vs.abs()) + 1.01 * u * u * (p @ vs).abs() + 2.0 ** -25
    assert ((out.double() + lo.double() - p @ vs).abs() <= tol).all()
