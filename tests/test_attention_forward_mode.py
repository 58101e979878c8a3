"""Forward-mode derivatives are refused, not dropped (no GPU needed: the check
comes before the one on devices)."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from modelos_b200.attention import KVCache4, window_attention


@pytest.mark.parametrize("which", [0, 1, 2])
def test_dual_tensors(which):
    x = [torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16) for _ in range(3)]
    with fwAD.dual_level():
        x[which] = fwAD.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            window_attention(*x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            window_attention(*x)
        with pytest.raises(RuntimeError, match="CUDA"):  # what carries no tangent is as it was
            window_attention(*(fwAD.unpack_dual(t).primal for t in x))


def test_dual_queries_over_the_4_bit_cache():
    c = KVCache4(1, 2, 8, 64, device="cpu")
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            c.attend(dual)
        for k, v in ((dual, x), (x, dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                c.write(k, v, 0)
