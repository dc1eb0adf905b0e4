"""Sizes at the limits of the 8-bit cache's calls, at the C ABI (no GPU needed, nothing is launched)."""
import ctypes

import pytest

from metalops_amd import _lib

L = _lib.lib
X, W, S, Y = 0x10000, 0x20000, 0x30000, 0x40000      # never dereferenced


def _cache(**kw):
    f = dict(k_codes=X, v_codes=W, k_scales=S, v_scales=Y, num_pages=1 << 20, kv_heads=8, head_dim=128, page_size=64)
    return ctypes.byref(_lib.Kv8CacheStruct(**{**f, **kw}))


def _batch(width, T, batch=1):
    return ctypes.byref(_lib.Kv8BatchStruct(block_table=X, table_stride=width, batch=batch, width=width, lens=W, cu_seqlens=None, T=T))


def test_page_of_two_gib_is_refused():
    b = _batch(4, 1)
    assert L.mcq4_kv8_read(_cache(kv_heads=32768, page_size=256, head_dim=256), b, X, Y, 1, None) == _lib.MCQ4_ERR_SHAPE
    assert b"too large" in L.mcq4_last_error()
    # One head less passes that check: what is refused then is the output's alignment.
    assert L.mcq4_kv8_read(_cache(kv_heads=32767, page_size=256, head_dim=256), b, X + 4, Y, 1, None) == _lib.MCQ4_ERR_ALIGNMENT


@pytest.mark.parametrize("T,width,kv_heads", [(131072, 16384, 8), (1 << 20, 1 << 20, 8), (16384, 1 << 24, 1)])
def test_long_prompts_over_wide_tables(T, width, kv_heads):
    """New tokens times the table's tokens pass 2^31 many times; the calls are taken."""
    c, context = _cache(kv_heads=kv_heads), width * 64
    assert 0 <= L.mcq4_kv8_attention_workspace_bytes(c, _batch(width, T), 4 * kv_heads, 1, 0, context) < 1 << 34
    args = (S, 128, 128, 4 * kv_heads, 1, Y + 4, None, 1.0, 1, 0, context, None, 0, None)
    assert L.mcq4_kv8_attention(c, _batch(width, T), *args) == _lib.MCQ4_ERR_ALIGNMENT
    assert L.mcq4_kv8_attention(c, _batch(width, (1 << 24) + 1), *args) == _lib.MCQ4_ERR_SHAPE


def test_workspace_does_not_grow_with_the_table():
    need = [L.mcq4_kv8_attention_workspace_bytes(_cache(), _batch(w, 1024, 1024), 32, 1, 0, w * 64) for w in (1 << 10, 1 << 14)]
    assert 0 < need[0] == need[1] < 64 << 20


@pytest.mark.parametrize("window", [(1 << 30) + 1, 1 << 31, (1 << 32) + 5, 1 << 70])
def test_window_beyond_32_bits_is_refused(window):
    """Not cut to its lower bits."""
    import torch

    import metalops_amd as mo
    cache = mo.KV8Cache.empty(3, 2, 64, 16, "cpu")
    table, lens = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="window must be 0 to"):
        mo.kv8_attention(torch.zeros(1, 2, 64, dtype=torch.float16), cache, table, lens, window=window)
