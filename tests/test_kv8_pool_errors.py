"""Calls that change a pool's counts are made once, whatever becomes of them (no GPU needed)."""
import pytest
import torch

import metalops_amd as mo
from metalops_amd import _lib
from metalops_amd import pool as module

I32 = torch.int32


class _Native:
    """A native call path whose launches fail."""

    def kv8_fork(self, *args):
        return _lib.MCQ4_ERR_HIP

    kv8_resize = kv8_fork


class _Counting:
    """The library, counting the calls that the Python functions make of it."""

    def __init__(self):
        self.calls = 0

    def mcq4_last_error(self):
        return b"no launch"

    def mcq4_status_string(self, status):
        return b"HIP error"

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0
        return call


def test_a_launch_that_failed_is_not_made_again(monkeypatch):
    pool = mo.KV8Pool.empty(1, 5, 1, 16, 16, "cpu")
    t, n = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32)
    library = _Counting()
    monkeypatch.setattr(module, "_native", _Native())
    monkeypatch.setattr(module, "_require_device", lambda *a: None)
    monkeypatch.setattr(_lib, "lib", library)
    for call, name in ((lambda: mo.kv8_fork(pool, t, n, n), "kv8_fork"), (lambda: mo.kv8_resize(pool, t, n, n), "kv8_resize")):
        with pytest.raises(_lib.Mcq4Error, match=f"mcq4_{name}.*no launch") as e:
            call()
        assert e.value.status == _lib.MCQ4_ERR_HIP
    assert library.calls == 0
