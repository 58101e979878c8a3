"""Which exception a device error word becomes when several bits are set: a wait
that gave up (whose results mean nothing) is not hidden by a skipped row."""
from __future__ import annotations

import pytest

from modelos_b200 import _native


@pytest.mark.parametrize("bits,error,what", [
    (1, IndexError, "embedding index"), (2, RuntimeError, "timed out"), (4, IndexError, "4-bit cache"),
    (8, ValueError, "padding mask"), (2 | 4, RuntimeError, "timed out"), (2 | 8, RuntimeError, "timed out"),
    (1 | 2, IndexError, "embedding index"), (4 | 8, IndexError, "4-bit cache"),
])
def test_order(monkeypatch, bits, error, what):
    monkeypatch.setattr(_native, "read_device_errors", lambda dev=None, reset=True: bits)
    with pytest.raises(error, match=what):
        _native.check_device_errors()
