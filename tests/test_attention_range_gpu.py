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


def bounds(q, k, v, dout, scale, window=0, sinks=0):
    """The gradients in 64 bits and bounds on the kernels' error where all scores
    are 0 (q or k is): P = 1 / n, the forward pass adds exact probabilities of 1
    and delta comes from the output with its remainder, so that what is left are
    the roundings of P and of dS.  They are held times powers of two, P times 2^14
    and dS times at least 2^13 / N, N the largest norm of a dout row times that of a
    v row: below fp16's normal range a rounding is off by 2^-25 of the held value,
    2^-39 of P and N 2^-38 of dS."""
    B, Hq, Tq, D = q.shape
    Hk, Tk = k.shape[1], k.shape[2]
    u, f32 = 2.0 ** -11, attnref.F32
    see = attnref.visible(B, Tq, Tk, window, sinks, None, None, device=DEV).double()
    q, do = q.double(), dout.double()
    ks, vs = attnref.spread(k.double(), Hq), attnref.spread(v.double(), Hq)
    p = (see / see.sum(-1, keepdim=True)).expand(B, Hq, Tq, Tk)
    dp = do @ vs.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    # dp and delta in 32 bits (and the remainder's own rounding, u^2); P's exponential
    size = (do.abs() @ vs.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    N = do.norm(dim=-1).amax() * vs.norm(dim=-1).amax()
    e_ds = ds.abs() * (1.01 * u + 2 * attnref.EXP)
    e_ds += p * abs(scale) * size * ((2 * D + Tk + 16) * f32 + 2 * u * u) + N * 2.0 ** -38 * abs(scale) * see
    e_p = p * (1.01 * u + 2 * attnref.EXP) + 2.0 ** -39 * see

    def heads(x):
        return x.view(B, Hk, Hq // Hk, Tk, D).sum(2)

    m = (Tq * (Hq // Hk) + 8) * f32
    dq, dk = ds @ ks, heads(ds.transpose(-1, -2) @ q)
    dv = heads(p.transpose(-1, -2) @ do)
    return dict(
        ds=ds, dq=dq, dq_tol=u * dq.abs() + e_ds @ ks.abs() + (Tk + 8) * f32 * (ds.abs() @ ks.abs()),
        dk=dk, dk_tol=(u * dk.abs() + heads(e_ds.transpose(-1, -2) @ q.abs())
                       + m * heads(ds.abs().transpose(-1, -2) @ q.abs())),
        dv=dv, dv_tol=(u * dv.abs() + heads(e_p.transpose(-1, -2) @ do.abs())
                       + m * heads(p.transpose(-1, -2) @ do.abs())))


def randn(*shape, seed, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(HF)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
@pytest.mark.parametrize("zero", ["q", "k"])
def test_small_output_gradients(D, window, sinks, zero):
    """dout of 2^-15 over some thousand keys: P (dP - delta) lies near 2^-23,
    where fp16 holds a bit or none."""
    T = 2048
    q, k = randn(1, 2, T, D, seed=1, size=8.0), randn(1, 1, T, D, seed=2, size=8.0)
    (q if zero == "q" else k).zero_()
    v, dout = randn(1, 1, T, D, seed=3), randn(1, 2, T, D, seed=4, size=2.0 ** -15)
    r = bounds(q, k, v, dout, 1.0, window, sinks)
    for name, x in zip(("dq", "dk", "dv"), gradients(q, k, v, dout, 1.0, window, sinks)):
        attnref.within(x, r[name], r[name + "_tol"], name)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
@pytest.mark.parametrize("zero", ["q", "k"])
def test_large_output_gradients(D, window, sinks, zero):
    """dout of 2^12 (a scaled loss) and values of 8: P (dP - delta) passes 65504,
    the gradients do not."""
    T = 600
    q, k = randn(1, 2, T, D, seed=5), randn(1, 1, T, D, seed=6)
    (q if zero == "q" else k).zero_()
    v, dout = randn(1, 1, T, D, seed=7, size=8.0), randn(1, 2, T, D, seed=8, size=2.0 ** 12)
    scale = 1 / 64
    r = bounds(q, k, v, dout, scale, window, sinks)
    assert r["ds"].abs().max() / scale > 65504
    assert all(r[n].abs().max() < 6e4 for n in ("dq", "dk", "dv"))
    for name, x in zip(("dq", "dk", "dv"), gradients(q, k, v, dout, scale, window, sinks)):
        attnref.within(x, r[name], r[name + "_tol"], name)


def test_many_keys():
    """P of 1 / 70000, where fp16 itself holds 8 bits."""
    q, k = torch.zeros(1, 2, 130, 64, dtype=HF, device=DEV), randn(1, 1, 70_000, 64, seed=16)
    v, dout = randn(1, 1, 70_000, 64, seed=17), randn(1, 2, 130, 64, seed=18, size=100.0)
    r = bounds(q, k, v, dout, 1.0)
    for name, x in zip(("dq", "dk", "dv"), gradients(q, k, v, dout, 1.0)):
        attnref.within(x, r[name], r[name + "_tol"], name)


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


def test_gradients_of_zeros():
    q, k, v = (randn(1, 1, 200, 64, seed=i) for i in (13, 14, 15))
    for x in gradients(q, k, v, torch.zeros_like(q), 0.125):
        assert (x == 0).all()
    dq, dk, dv = gradients(q, k, torch.zeros_like(v), q, 0.125)
    assert (dq == 0).all() and (dk == 0).all() and torch.isfinite(dv).all()
