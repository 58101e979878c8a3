"""KVCache4's tensors are its attributes: replaced by ones that do not fit (a
snapshot of another batch), a call is refused before any kernel reads past them."""
from __future__ import annotations

import pytest
import torch

from modelos_b200.attention import KVCache4

BF = torch.bfloat16


def attempts(c):
    x = torch.zeros(2, 2, 1, 64, dtype=BF)
    return (lambda: c.write(x, x, 0), lambda: c.read(0, 1), lambda: c.attend(x), lambda: c.append(x, x))


@pytest.mark.parametrize("name,bad", [
    ("v_codes", torch.zeros(1, 2, 8, 32, dtype=torch.uint8)), ("v_codes", torch.zeros(2, 2, 4, 32, dtype=torch.uint8)),
    ("v_codes", torch.zeros(2, 2, 8, 32, dtype=torch.int8)), ("k_codes", torch.zeros(2, 2, 16, 32, dtype=torch.uint8)),
    ("k_codes", torch.zeros(2, 2, 8, 64, dtype=torch.uint8)[..., :32]), ("k_codes", torch.zeros(2, 8, 32, dtype=torch.uint8)),
    ("k_params", torch.zeros(2, 2, 8, 1, 2, dtype=BF)), ("v_params", torch.zeros(2, 2, 8, 2, 2, dtype=torch.float16)),
    ("v_params", torch.zeros(2, 2, 8, 2, dtype=BF)),
])
def test_codes_and_params(name, bad):
    c = KVCache4(2, 2, 8, 64, device="cpu")
    setattr(c, name, bad)
    for call in attempts(c):
        with pytest.raises(ValueError, match="do not fit"):
            call()


@pytest.mark.parametrize("bad", [torch.zeros(1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32),
                                 torch.zeros(2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)[::2],
                                 torch.zeros(2, 1, dtype=torch.int32), torch.zeros((), dtype=torch.int32)])
def test_lengths(bad):
    c = KVCache4(2, 2, 8, 64, device="cpu")
    c.lengths = bad
    with pytest.raises(ValueError, match="lengths must be"):
        c.attend(torch.zeros(2, 2, 1, 64, dtype=BF))
