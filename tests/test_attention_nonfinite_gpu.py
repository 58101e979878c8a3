"""NaN and infinities in rows that are seen, on the GPU kernels: the output, the
softmax's logarithm and the gradients are what the definition gives, and never
a finite number in place of a NaN."""
from __future__ import annotations

import pytest
import torch

import attnref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def make(B, Hq, Hk, Tq, Tk, D, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def t(H, T):
        return torch.randn(B, T, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2)

    return t(Hq, Tq), t(Hk, Tk), t(Hk, Tk), t(Hq, Tq)


def expected(q, k, v, window, sinks, scale, starts=None, lengths=None):
    """``(out, lse, tol)`` in 64 bits.  A score of -inf is a probability of 0, one
    of +inf or NaN makes the row NaN, as a row is whose scores are all -inf."""
    Hq, Tq = q.shape[1:3]
    see = attnref.visible(q.shape[0], Tq, k.shape[2], window, sinks, starts, None, lengths, DEV)
    ks, vs = attnref.spread(k.double(), Hq), attnref.spread(v.double(), Hq)
    s = torch.stack([q[b].double() @ ks[b].transpose(-1, -2) for b in range(len(q))]) * scale
    s = s.masked_fill(~see, -INF)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    none = ~see.any(-1, keepdim=True)
    p = torch.where(none, torch.zeros_like(p), p)
    # hidden keys take no part, whatever they hold
    out = torch.where(see[..., None], p[..., None] * vs[:, :, None], torch.zeros((), dtype=p.dtype, device=DEV)).sum(-2) \
        if vs.isnan().any() else p @ vs
    # as attnref.reference has it; the scores' size from the finite keys alone
    u = torch.finfo(q.dtype).eps / 2
    least = torch.finfo(q.dtype).smallest_normal * u
    size = (torch.nan_to_num(q.double(), 0, 0, 0).abs() @ torch.nan_to_num(ks, 0, 0, 0).abs().transpose(-1, -2)) * scale
    E = attnref.EXP + 2 * (q.shape[-1] + 4) * attnref.F32 * (size * see).amax().item()
    n = see.sum(-1).amax().item()
    va = torch.nan_to_num(vs, 0, 0, 0).abs()
    a = torch.nan_to_num(p, 0, 0, 0) @ va
    tol = u * torch.nan_to_num(out, 0, 0, 0).abs() + (u + 2 * E + (n + 8) * attnref.F32) * a * 1.01 + least * (
        see.double() @ va)
    return out, lse, tol


def compare(got, want, tol, what):
    bad = want.isnan()
    assert bad.any(), what
    assert torch.equal(got.isnan(), bad), f"{what}: {int((got.isnan() != bad).sum())} of {bad.numel()} are NaN wrongly"
    attnref.within(got[~bad], want[~bad], tol[~bad], what)  # (none where every row sees the bad key)


# tiles of 128 rows; keys shared by several blocks; few rows, alone and over a cluster
SHAPES = [(2, 4, 2, 300, 300), (1, 2, 1, 130, 1500), (2, 4, 2, 5, 40), (1, 4, 2, 3, 900)]


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64), (BF, 72)])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("what", ["k nan", "k inf", "q nan", "q inf"])
def test_scores_that_are_not_finite(shape, dtype, D, what):
    from modelos_b200.attention import window_attention
    B, Hq, Hk, Tq, Tk = shape
    q, k, v, _ = make(B, Hq, Hk, Tq, Tk, D, dtype, seed=Tk)
    value = NAN if "nan" in what else INF
    if what[0] == "k":
        # one key early among the last queries' own, and (where they are not) one of the first block
        k[0, 0, Tk - Tq + 1, 3] = value
        k[-1, -1, 7 if Tk > Tq else Tk - 2, 3] = value
    else:
        q[0, 1, Tq // 2, 3] = value
    for window, sinks in ((0, 0), (max(2, Tk // 4), 3)):
        want, _, tol = expected(q, k, v, window, sinks, D ** -0.5)
        got = window_attention(q, k, v, window=window, sinks=sinks)
        compare(got, want, tol, (what, window))


@pytest.mark.parametrize("shape", SHAPES)
def test_a_value_that_is_not_finite(shape):
    """In the rows that see it, and there in its channel alone."""
    from modelos_b200.attention import window_attention
    B, Hq, Hk, Tq, Tk = shape
    q, k, v, _ = make(B, Hq, Hk, Tq, Tk, 64, BF, seed=Tk)
    v[0, 0, 7 if Tk > Tq else 0, 3] = NAN  # all rows see it
    want, _, tol = expected(q, k, v, 0, 0, 0.125)
    compare(window_attention(q, k, v), want, tol, "v")


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_whose_scores_are_all_minus_infinity(shape):
    """0 / 0, not the 0 of a row that sees nothing; rows outside the sequence
    stay 0, whatever they hold."""
    from modelos_b200.attention import window_attention
    B, Hq, Hk, Tq, Tk = shape
    q, k, v, _ = make(B, Hq, Hk, Tq, Tk, 64, BF, seed=Tk)
    q[:, :, :, 5], k[:, :, :, 5] = 1.0, -INF
    first = Tk - Tq + 1  # the first query is padding
    starts = torch.full((B,), first, dtype=torch.int32, device=DEV)
    out = window_attention(q, k, v, starts=starts)
    assert (out[:, :, 0] == 0).all() and out[:, :, 1:].isnan().all()


def test_log_of_the_softmax_sum_and_gradients():
    """A bad query: its lse and dq are NaN, and dk and dv of the keys that it
    sees; other queries' dq are right."""
    from test_attention_gpu import attn_fwd

    from modelos_b200.attention import window_attention
    for Tq, Tk in ((260, 260), (3, 900), (130, 1500)):
        q, k, v, dout = make(1, 2, 1, Tq, Tk, 64, BF, seed=Tk)
        clean = q.clone()
        q[0, 1, 2, 3] = NAN
        _, lse = attn_fwd(q, k, v, 0.125, 0, 0, None, None)
        assert lse[0, 1, 2].isnan() and int(lse.isnan().sum()) == 1
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        dq, dk, dv = torch.autograd.grad(window_attention(*leaves), leaves, dout)
        r = attnref.reference(clean, k, v, 0, 0, 0.125, None, None, dout)
        real = torch.ones(1, 2, Tq, dtype=torch.bool, device=DEV)
        real[0, 1, 2] = False
        assert dq[~real].isnan().all()
        attnref.within(dq[real], r["dq"][real], r["dq_tol"][real], "dq")
        seen = Tk - Tq + 3
        assert dk[:, :, :seen].isnan().all() and dv[:, :, :seen].isnan().all()


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("side", ["k", "v"])
def test_groups_of_the_4_bit_cache_that_read_back_as_nan(dtype, D, side):
    from modelos_b200.attention import KVCache4
    B, Hk, cap = 3, 2, 700
    c = KVCache4(B, Hk, cap, D, dtype=dtype, device=DEV)
    _, k, v, _ = make(B, 4, Hk, cap, cap, D, dtype, seed=D)
    bad = k if side == "k" else v
    bad[0, 0, 40, 33] = NAN
    bad[1, 1, 299, 1] = INF
    c.write(k, v, 0)
    lengths = torch.tensor([700, 300, 65], dtype=torch.int32, device=DEV)
    c.lengths.copy_(lengths)
    for Tq in (1, 3):
        q = make(B, 4, Hk, Tq, cap, D, dtype, seed=9)[0]
        for window, sinks in ((0, 0), (700, 1)):
            rk, rv = c.read(0, cap)
            want, _, tol = expected(q, rk, rv, window, sinks, D ** -0.5, lengths=lengths)
            if side == "v":  # hidden by a few tokens' causality, a NaN may still reach the rows beside
                want[1, :, :-1] = 0
            got = c.attend(q, window=window, sinks=sinks)
            if side == "v":
                got = got.clone()
                got[1, :, :-1] = 0
            compare(got, want, tol, (side, Tq, window))


@pytest.mark.parametrize("shape", SHAPES + [(2, 2, 1, 24, 24), (1, 40, 1, 100, 128)])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64), (BF, 72)])
def test_an_infinite_value(shape, dtype, D):
    """inf in its channel for the rows that see it (also where probabilities take
    part in two products), and in dv's channel for an infinite output gradient."""
    from modelos_b200.attention import window_attention
    B, Hq, Hk, Tq, Tk = shape
    q, k, v, dout = make(B, Hq, Hk, Tq, Tk, D, dtype, seed=Tk)
    key = 7 if Tk > Tq else 0  # all rows see it
    v[0, 0, key, 3], v[-1, -1, key, 5] = INF, -INF
    out = window_attention(q, k, v)
    want = torch.zeros_like(out)
    G = Hq // Hk
    want[0, :G, :, 3], want[-1, -G:, :, 5] = INF, -INF
    assert torch.equal(out.isinf(), want.isinf()) and not out.isnan().any()
    assert torch.equal(out[want.isinf()], want[want.isinf()])
    # the last query sees all keys
    leaves = [t.detach().requires_grad_() for t in make(B, Hq, Hk, Tq, Tk, D, dtype, seed=Tk)[:3]]
    dout[0, 0, -1, 3] = INF
    _, _, dv = torch.autograd.grad(window_attention(*leaves), leaves, dout)
    assert (dv[0, 0, :, 3] == INF).all() and torch.isfinite(dv[0, 0, :, :3]).all()
