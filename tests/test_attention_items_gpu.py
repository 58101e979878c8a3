"""Attention over several times as many tiles as the GPU has multiprocessors:
what a persistent block carries from one item to the next (ring and barrier
phases, accumulators, store boxes), with partial, empty and single tiles in
turn."""
from __future__ import annotations

import pytest
import torch

import attnref
from test_attention_gpu import check, garbage, ints, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def enough(B, Hq, Hk, Tq, Tk):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles = (Tq + 127) // 128 * (Hq // Hk)
    for n in ((tiles + 1) // 2, tiles, (Tk + 127) // 128):  # forward, dq, dk and dv
        assert n * B * Hk > 2 * sms


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 5), (90, 150)])
def test_ragged_batches(dtype, D, window, sinks):
    B, Hq, Hk, T = 8, 16, 8, 700
    enough(B, Hq, Hk, T, T)
    starts = ints(0, 130, 0, 699, 257, 5, 700, 300)
    ends = ints(700, 700, 513, 700, 258, 129, 700, 300)  # the last two are empty
    q, k, v, dout = make(B, Hq, Hk, T, T, D, dtype, seed=D + window)
    keep = attnref.real_rows(B, T, starts, ends, DEV)
    q, k, v, dout = (garbage(t, keep) for t in (q, k, v, dout))
    out, grads = check(q, k, v, dout, window, sinks, starts, ends)
    for t in (out, *grads):
        assert (t.transpose(1, 2)[~keep] == 0).all()


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 40)])
@pytest.mark.parametrize("Hq,Hk,Tq,Tk", [(9, 9, 640, 901), (15, 5, 1030, 1030)])
def test_odd_numbers_of_tiles(dtype, D, Hq, Hk, Tq, Tk):
    """Pairs of tiles of which the last is alone; queries behind a cache."""
    B = 12
    enough(B, Hq, Hk, Tq, Tk)
    ends = ints(*(Tk - 37 * b for b in range(B)))
    check(*make(B, Hq, Hk, Tq, Tk, D, dtype, seed=Tq), 300, 3, None, ends)
