"""What kv8_shared_attention refuses, in Python and at the C ABI (no GPU needed, nothing is launched)."""
import ctypes

import pytest
import torch

import metalops_amd as mo
from metalops_amd import _lib

I32 = torch.int32
INVALID, SHAPE, ALIGN, WS = (_lib.MCQ4_ERR_INVALID_ARG, _lib.MCQ4_ERR_SHAPE, _lib.MCQ4_ERR_ALIGNMENT, _lib.MCQ4_ERR_WORKSPACE)
A, B, C, Q = 0x10000, 0x20000, 0x30000, 0x40000      # never dereferenced


def _args(**kw):
    a = dict(q=torch.zeros(4, 4, 64).half(), cache=mo.KV8Cache.empty(9, 2, 64, 16, "cpu"), prefix_table=torch.zeros(2, 3, dtype=I32),
             prefix_lens=torch.zeros(2, dtype=I32), block_table=torch.zeros(4, 2, dtype=I32), context_lens=torch.zeros(4, dtype=I32))
    a.update(kw)
    return a


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_cpu_tensors_rejected_no_fallback():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mo.kv8_shared_attention(**_args())


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(4, 4, 64)), "float16 or bfloat16"), (dict(q=torch.zeros(4, 3, 64).half()), "multiple of the cache's"),
    (dict(q=torch.zeros(4, 4, 32).half()), r"q must be \[T, heads, 64\]"), (dict(prefix_table=torch.zeros(2, 3)), "prefix_table"),
    (dict(prefix_table=torch.zeros(3, dtype=I32)), "prefix_table"), (dict(prefix_lens=torch.zeros(3, dtype=I32)), "prefix_lens"),
    (dict(prefix_lens=torch.zeros(2)), "prefix_lens"), (dict(groups=torch.zeros(2, dtype=I32)), "groups"), (dict(groups=torch.zeros(3)), "groups"),
    (dict(prefix_table=torch.zeros(3, 3, dtype=I32), prefix_lens=torch.zeros(3, dtype=I32)), "multiple of the 3 prefixes"),
    (dict(block_table=torch.zeros(4, 2)), "block_table"), (dict(context_lens=torch.zeros(3, dtype=I32)), "context_lens"),
    (dict(cu_seqlens=torch.zeros(4, dtype=I32)), "cu_seqlens"), (dict(block_table=torch.zeros(3, 2, dtype=I32), context_lens=torch.zeros(3, dtype=I32)), "multiple of the 3 sequences"),
    (dict(max_prefix=-1), "max_prefix"), (dict(max_context=-1), "max_context")])
def test_python(kw, match, monkeypatch):
    from metalops_amd import kv8
    monkeypatch.setattr(kv8, "_require_device", lambda *a: None)
    with pytest.raises(RuntimeError, match=match):
        mo.kv8_shared_attention(**_args(**kw))


def test_capi():
    L = _lib.lib

    def go(query=False, cache=None, prefix=None, batch=None, **kw):
        c = dict(k_codes=A, v_codes=A, k_scales=B, v_scales=B, num_pages=9, kv_heads=2, head_dim=64, page_size=64)
        p = dict(block_table=A, table_stride=3, prefixes=2, width=3, lens=B, groups=None)
        b = dict(block_table=A, table_stride=2, batch=4, width=2, lens=B, cu_seqlens=None, T=4)
        for d, u in ((c, cache), (p, prefix), (b, batch)):
            d.update(u or {})
        f = dict(q=Q, token=256, head=64, heads=4, dtype=1, out=C, lse=None, scale=1.0, max_prefix=192, max_context=128, ws=A, ws_bytes=1 << 30)
        f.update(kw)
        s = [ctypes.byref(t) for t in (_lib.Kv8CacheStruct(**c), _lib.Kv8PrefixesStruct(**p), _lib.Kv8BatchStruct(**b))]
        if query:
            return L.mcq4_kv8_shared_attention_workspace_bytes(*s, f["heads"], f["max_prefix"], f["max_context"])
        return L.mcq4_kv8_shared_attention(*s, *f.values(), None)
    need = go(True)
    assert need > 0
    assert go(ws=None) == WS and go(ws_bytes=need - 1) == WS and go(ws=A + 8) == ALIGN
    assert go(q=None) == INVALID and go(out=None) == INVALID and go(dtype=0) == INVALID
    for kw in (dict(q=Q + 8), dict(token=260), dict(head=60), dict(out=C + 8), dict(lse=C + 2)):
        assert go(**kw) == ALIGN
    for kw in (dict(token=-8), dict(head=-8), dict(heads=3), dict(heads=0), dict(max_prefix=-1), dict(max_context=-1)):
        assert go(**kw) == SHAPE
    for kw in (dict(block_table=None), dict(lens=None)):
        assert go(prefix=kw) == INVALID and go(batch=kw) == INVALID
    for kw in (dict(prefixes=0), dict(prefixes=1 << 21), dict(prefixes=3), dict(width=0), dict(width=1 << 25), dict(table_stride=2)):
        assert go(prefix=kw) == SHAPE and go(True, prefix=kw) == 0
    assert go(prefix=dict(prefixes=3, groups=B), ws_bytes=0) == WS
    for kw in (dict(block_table=A + 2), dict(lens=B + 1), dict(groups=B + 2)):
        assert go(prefix=kw) == ALIGN
    assert go(batch=dict(T=5)) == SHAPE and go(batch=dict(T=0)) == SHAPE and go(batch=dict(batch=0)) == SHAPE
    # More pieces than the kernel counts.
    many = dict(prefix=dict(prefixes=1, width=1 << 20, table_stride=1 << 20), batch=dict(T=1 << 20, batch=1 << 20))
    assert go(**many) == SHAPE and go(True, **many) == 0
    # More rows of records: 2^20 sequences and prefixes, 64 heads, 16 rows to a prefix's record.
    many = dict(cache=dict(kv_heads=64, head_dim=16, page_size=16), prefix=dict(prefixes=1 << 20, width=1, table_stride=1),
                batch=dict(T=1 << 20, batch=1 << 20, width=1, table_stride=1), heads=64)
    assert go(**many) == SHAPE and go(True, **many) == 0
    assert go(cache=dict(head_dim=72)) == SHAPE and go(True, cache=dict(page_size=8)) == 0
