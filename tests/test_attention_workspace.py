"""The backward pass's workspace, from the C entry point (no kernel runs; the number
of multiprocessors counts)."""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

from modelos_b200 import _native

pytestmark = pytest.mark.gpu


def bwd(B, Hq, Hk, Tq, Tk, D, window, sinks):
    n = ctypes.c_size_t(0)
    assert _native.lib().pkm_attn_bwd_workspace(B, Hq, Hk, Tq, Tk, D, window, sinks, ctypes.byref(n)) == 0
    return n.value


def limit(D):
    """Partial dk and dv of 128 rows each, at most twelve times as many as the GPU
    has multiprocessors."""
    return 12 * torch.cuda.get_device_properties(0).multi_processor_count * 128 * 2 * 4 * D


@pytest.mark.parametrize("window,sinks", [(512, 4), (512, 8192), (256, 32767), (1, 32767), (128, 500)])
def test_sinks_do_not_take_gigabytes(window, sinks):
    sizes = (1, 16, 8, 32768, 32768, 128)
    assert bwd(*sizes, window, sinks) - bwd(*sizes, window, 0) <= limit(128)


def test_sinks_over_the_range():
    r = random.Random(1)
    shared = 0
    for _ in range(2000):
        B, Hk, G, D = r.choice([1, 2, 5, 16]), r.choice([1, 2, 8, 32]), r.choice([1, 2, 7]), r.choice([8, 64, 128])
        Tk = int(2 ** r.uniform(4, 18))
        Tq = r.choice([Tk, max(1, Tk // 3)])
        window, sinks = int(2 ** r.uniform(0, 15)), int(2 ** r.uniform(0, 17))
        extra = bwd(B, Hk * G, Hk, Tq, Tk, D, window, sinks) - bwd(B, Hk * G, Hk, Tq, Tk, D, window, 0)
        assert 0 <= extra <= limit(D), (B, Hk, G, D, Tq, Tk, window, sinks)
        shared += extra > 0
    assert shared > 100  # the range reaches what it is about
