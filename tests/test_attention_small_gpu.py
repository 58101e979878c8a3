"""Small calls over few keys, bound by launches: outputs and gradients are off by their own
rounding, not by those of the probabilities and their gradients (which take part
with their remainders)."""
from __future__ import annotations

import pytest
import torch

import attnref
from test_attention_gpu import garbage, ints, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def bounds(q, k, v, dout, window, sinks, scale, starts, ends):
    """Results in 64 bits and bounds on the kernels' error: what is held in the
    operands' type is held with its remainder, good to u * u of it (probabilities
    2 u * u: their first part is rounded down, and a remainder of 0 is held as the
    type's smallest number, 2 ``least``); scores, sums and statistics are in 32 bits,
    the exponential is good to 2^-22."""
    u, f32 = torch.finfo(q.dtype).eps / 2, attnref.F32
    least = torch.finfo(q.dtype).smallest_normal * u
    B, Hq, Tq, D = q.shape
    Hk, Tk = k.shape[1], k.shape[2]
    rows = attnref.real_rows(B, Tk, starts, ends, DEV)
    q, do = (attnref.clean(t.double(), rows[:, Tk - Tq:]) for t in (q, dout))
    ks, vs = (attnref.spread(attnref.clean(t.double(), rows), Hq) for t in (k, v))
    see = attnref.visible(B, Tq, Tk, window, sinks, starts, ends, device=DEV)
    out, _, p = attnref.forward(q, ks, vs, see, scale)
    seen = see.double().expand_as(p)
    size = (q.abs() @ ks.abs().transpose(-1, -2)) * abs(scale)
    n, m = see.sum(-1).amax().item(), Tq * (Hq // Hk)
    one = 2.02 * u * u + 2 * (2.0 ** -20 + (D + 8) * f32 * (size * see).amax().item()) + (n + 16) * f32
    ep = p * one + 2 * least * seen
    r = dict(out=(out, u * out.abs() * (1 + u) + ep @ vs.abs()))
    dp = do @ vs.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    e_dp = (D + 4) * f32 * (do.abs() @ vs.abs().transpose(-1, -2))
    e_out = ep @ vs.abs() + 1.01 * u * u * out.abs()
    e_delta = (do.abs() * e_out).sum(-1, keepdim=True) + (D + 4) * f32 * (do * out).abs().sum(-1, keepdim=True)
    e_ds = abs(scale) * (p * ((dp - delta).abs() * one + e_dp + e_delta) * 1.01 + least * seen)

    def heads(x):
        return x.view(B, Hk, Hq // Hk, Tk, D).sum(2)

    dq, dk = ds @ ks, heads(ds.transpose(-1, -2) @ q)
    dv = heads(p.transpose(-1, -2) @ do)
    r["dq"] = dq, u * dq.abs() * (1 + u) + e_ds @ ks.abs() + (n + 8) * f32 * (ds.abs() @ ks.abs())
    r["dk"] = dk, (u * dk.abs() * (1 + u) + heads(e_ds.transpose(-1, -2) @ q.abs())
                   + (m + 8) * f32 * heads(ds.abs().transpose(-1, -2) @ q.abs()))
    r["dv"] = dv, (u * dv.abs() * (1 + u) + heads(ep.transpose(-1, -2) @ do.abs())
                   + (m + 8) * f32 * heads(p.transpose(-1, -2) @ do.abs()))
    return r


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (BF, 40), (HF, 64), (HF, 120)])
@pytest.mark.parametrize("shape,window,sinks,pad", [
    (shape, *mask) for shape in ((2, 2, 1, 24, 24), (1, 2, 1, 17, 100), (2, 4, 2, 101, 101), (1, 6, 2, 60, 128),
                                 (3, 3, 3, 128, 128))
    for mask in ((0, 0, 0), (8, 2, 3), (100, 0, 7))
] + [((1, 2, 1, 450, 600), 20, 4, 0), ((2, 4, 2, 300, 300), 1, 0, 5), ((2, 3, 1, 513, 513), 31, 1, 9)])
def test_output_and_gradients(dtype, D, shape, window, sinks, pad):
    from modelos_b200 import _native
    from modelos_b200.attention import window_attention
    B, Tq, Tk = shape[0], shape[3], shape[4]
    q, k, v, dout = make(*shape, D, dtype, seed=D + Tk)
    starts = ints(*(pad * b for b in range(B))) if pad else None
    ends = ints(*(Tk - pad * (b % 2) for b in range(B))) if pad else None
    if pad:
        keep = attnref.real_rows(B, Tk, starts, ends, DEV)
        q, dout = (garbage(t, keep[:, Tk - Tq:]) for t in (q, dout))
        k, v = garbage(k, keep), garbage(v, keep)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, window=window, sinks=sinks, starts=starts, ends=ends)
    got = (out, *torch.autograd.grad(out, leaves, dout))
    r = bounds(q, k, v, dout, window, sinks, D ** -0.5, starts, ends)
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        attnref.within(x, *r[name], name)
    _native.check_device_errors()
