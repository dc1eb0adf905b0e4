"""What the MXFP4 and 8-bit cache calls refuse, in Python and at the C ABI (no GPU needed, nothing is launched)."""
import ctypes

import pytest
import torch

import metalops_amd as mo
from metalops_amd import _lib

U8, I32 = torch.uint8, torch.int32


def test_k_assertions():
    with pytest.raises(AssertionError, match=r"K \(33\) must be divisible by 32"):
        mo.quantize_mxfp4(torch.zeros(4, 33))
    with pytest.raises(AssertionError, match=r"K \(48\) must be divisible by 32"):
        mo.dequantize_mxfp4(torch.zeros(4, 24, dtype=U8), torch.zeros(4, 1, dtype=U8))
    w = torch.zeros(8, 32, dtype=U8), torch.zeros(8, 2, dtype=U8)
    with pytest.raises(AssertionError, match=r"X K dim \(96\) must match weight K \(64\)"):
        mo.matmul_mxfp4(torch.zeros(2, 96), *w)
    with pytest.raises(AssertionError, match=r"X K dim \(32\) must match weight K \(64\)"):
        mo.matmul_mxfp4_mxfp4(torch.zeros(2, 16, dtype=U8), torch.zeros(2, 1, dtype=U8), *w)


def test_packed_shapes_and_types():
    p, s = torch.zeros(8, 32, dtype=U8), torch.zeros(8, 2, dtype=U8)
    for bad in ((p, s[:, :1]), (p, s[:7]), (p, s.float()), (p.int(), s), (torch.zeros((), dtype=U8), s)):
        with pytest.raises(RuntimeError):
            mo.dequantize_mxfp4(*bad)
        with pytest.raises(RuntimeError):
            mo.matmul_mxfp4(torch.zeros(2, 64), *bad)
    with pytest.raises(RuntimeError, match="scalar|dimension"):
        mo.quantize_mxfp4(torch.tensor(1.0))
    with pytest.raises(RuntimeError, match=r"\[N, K/2\]"):
        mo.matmul_mxfp4(torch.zeros(2, 64), p[None], s[None])


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_cpu_tensors_rejected_no_fallback():
    p, s = torch.zeros(8, 32, dtype=U8), torch.zeros(8, 2, dtype=U8)
    cache = mo.KV8Cache.empty(3, 2, 64, 16, "cpu")
    k, t, n = torch.zeros(1, 2, 64), torch.zeros(1, 3, dtype=I32), torch.zeros(1, dtype=I32)
    for call in (lambda: mo.quantize_mxfp4(torch.zeros(8, 64)), lambda: mo.dequantize_mxfp4(p, s),
                 lambda: mo.matmul_mxfp4(torch.zeros(2, 64), p, s), lambda: mo.matmul_mxfp4_mxfp4(p, s, p, s),
                 lambda: mo.kv8_append(cache, k, k, t, n), lambda: mo.kv8_read(cache, t, n),
                 lambda: mo.kv8_attention(k.half(), cache, t, n)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_cache_shapes():
    def make(P=3, H=2, page=16, D=64, v=None, s=None, dtype=U8):
        return mo.KV8Cache(torch.zeros(P, H, page, D, dtype=dtype), torch.zeros(v or (P, H, D, page), dtype=dtype),
                           torch.zeros(P, H, dtype=dtype), torch.zeros(s or (P, H), dtype=dtype))
    c = make()
    assert (c.num_pages, c.kv_heads, c.page_size, c.head_dim) == (3, 2, 16, 64) and "page_size=16" in repr(c)
    for bad in (dict(page=48), dict(page=8), dict(page=512), dict(D=72), dict(D=272), dict(P=0), dict(v=(3, 2, 16, 64)),
                dict(s=(3, 1)), dict(dtype=torch.int8)):
        with pytest.raises(RuntimeError):
            make(**bad)
    with pytest.raises(RuntimeError, match="contiguous"):
        mo.KV8Cache(c.k_codes, c.k_codes.transpose(2, 3), c.k_scales, c.v_scales)
    with pytest.raises(AttributeError):
        c.k_codes = c.k_codes.clone()


def test_cache_call_arguments():
    c = mo.KV8Cache.empty(3, 2, 64, 16, "cpu")
    k, t, n = torch.zeros(4, 2, 64), torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32)
    cu = torch.tensor([0, 1, 4], dtype=I32)
    for bad in ((k[:, :1], k[:, :1], t, n), (k, k[:3], t, n), (k, k.half(), t, n), (k.int(), k.int(), t, n), (k, k, t.long(), n),
                (k, k, t[0], n), (k, k, t, n.long()), (k, k, t, n[:1]), (k, k, t, n, cu[:2]), (k, k, t, n, cu.long()),
                (k[:3], k[:3], t, n), (k[..., :32], k[..., :32], t, n)):
        with pytest.raises(RuntimeError) as e:
            mo.kv8_append(c, *bad)
        assert "no CPU fallback" not in str(e.value)
    q = torch.zeros(4, 4, 64, dtype=torch.float16)
    for bad, kw in (((q.float(), c, t, n), {}), ((q[:, :3], c, t, n), {}), ((q[..., :48], c, t, n), {}), ((q[0], c, t, n), {}),
                    ((q, c, t, n), dict(window=-1)), ((q, c, t, n), dict(max_context=-2)), ((q[:, :0], c, t, n), {}),
                    ((q[:3], c, t, n), {}), ((q, c, t, n, cu[:2]), {})):
        with pytest.raises(RuntimeError) as e:
            mo.kv8_attention(*bad, **kw)
        assert "no CPU fallback" not in str(e.value)
    with pytest.raises(RuntimeError, match="dtype"):
        mo.kv8_read(c, t, n, torch.float64)


INVALID, SHAPE, ALIGN, WS = (_lib.MCQ4_ERR_INVALID_ARG, _lib.MCQ4_ERR_SHAPE, _lib.MCQ4_ERR_ALIGNMENT, _lib.MCQ4_ERR_WORKSPACE)
X, W, S, Y = 0x10000, 0x20000, 0x30000, 0x40000      # never dereferenced


def test_capi_conversions():
    L = _lib.lib
    q = L.mcq4_quantize_mxfp4
    assert q(None, 0, 64, 1, 4, 64, W, S, None) == INVALID
    assert q(X, 3, 64, 1, 4, 64, W, S, None) == INVALID
    assert q(X, 0, 64, 1, 4, 48, W, S, None) == SHAPE
    assert q(X, 0, 64, 1, 0, 64, W, S, None) == SHAPE
    assert q(X, 0, -64, 1, 4, 64, W, S, None) == SHAPE
    assert q(X, 0, 64, 1, 1 << 30, 1 << 10, W, S, None) == SHAPE
    assert q(X + 2, 0, 64, 1, 4, 64, W, S, None) == ALIGN
    assert q(X, 0, 64, 1, 4, 64, W + 8, S, None) == ALIGN
    d = L.mcq4_dequantize_mxfp4
    assert d(W, S, 4, 64, None, 1, None) == INVALID
    assert d(W, S, 4, 64, Y, 9, None) == INVALID
    assert d(W, S, 4, 40, Y, 1, None) == SHAPE
    assert d(W, S, 4, 64, Y + 4, 1, None) == ALIGN


def test_capi_products():
    L = _lib.lib
    m = L.mcq4_matmul_mxfp4
    ok = [X, 1, 64, W, S, Y, 8, 2, 64, 8, None, 0, None]

    def with_(i, v):
        return m(*[v if j == i else a for j, a in enumerate(ok)])
    for i in (0, 3, 4, 5):
        assert with_(i, None) == INVALID
    assert with_(1, 5) == INVALID
    assert with_(2, 32) == SHAPE and with_(6, 4) == SHAPE and with_(7, 0) == SHAPE and with_(8, 60) == SHAPE and with_(9, 0) == SHAPE
    assert with_(0, X + 8) == ALIGN and with_(2, 68) == ALIGN and with_(3, W + 4) == ALIGN and with_(5, Y + 1) == ALIGN
    m2 = L.mcq4_matmul_mxfp4_mxfp4
    assert m2(X, None, W, S, Y, 1, 8, 2, 64, 8, None, 0, None) == INVALID
    assert m2(X, S, W, S, Y, 4, 8, 2, 64, 8, None, 0, None) == INVALID
    assert m2(X + 8, S, W, S, Y, 1, 8, 2, 64, 8, None, 0, None) == ALIGN
    assert L.mcq4_matmul_mxfp4_workspace_bytes(1, 48, 8, 1) == 0 and L.mcq4_matmul_mxfp4_mxfp4_workspace_bytes(0, 64, 8) == 0
    for M, K, N, dt in ((1, 4096, 4096, 1), (16, 14336, 4096, 2), (300, 4128, 1001, 0), (64, 14336, 512, 1)):
        need = L.mcq4_matmul_mxfp4_workspace_bytes(M, K, N, dt)
        if need:
            assert m(X, dt, K, W, S, Y, N, M, K, N, None, 0, None) == WS
            assert m(X, dt, K, W, S, Y, N, M, K, N, 0x50000, need - 1, None) == WS


def _cache(**kw):
    f = dict(k_codes=X, v_codes=W, k_scales=S, v_scales=Y, num_pages=9, kv_heads=2, head_dim=64, page_size=64)
    return _lib.Kv8CacheStruct(**{**f, **kw})


def _batch(**kw):
    f = dict(block_table=X, table_stride=4, batch=2, width=4, lens=W, cu_seqlens=None, T=2)
    return _lib.Kv8BatchStruct(**{**f, **kw})


BAD_CACHES = [(dict(k_codes=None), INVALID), (dict(v_scales=None), INVALID), (dict(page_size=24), SHAPE), (dict(page_size=512), SHAPE),
              (dict(head_dim=40), SHAPE), (dict(head_dim=0), SHAPE), (dict(head_dim=288), SHAPE), (dict(kv_heads=0), SHAPE),
              (dict(num_pages=0), SHAPE), (dict(v_codes=W + 8), ALIGN)]
BAD_BATCHES = [(dict(block_table=None), INVALID), (dict(lens=None), INVALID), (dict(batch=0), SHAPE), (dict(width=0), SHAPE),
               (dict(table_stride=3), SHAPE), (dict(width=1 << 25, table_stride=1 << 25), SHAPE), (dict(lens=W + 2), ALIGN)]


def test_capi_cache():
    L, ref = _lib.lib, ctypes.byref
    good = ref(_cache()), ref(_batch())

    def append(c, b, k=X, dt=1, stride=128):
        return L.mcq4_kv8_append(c, b, k, stride, 64, W, 128, 64, dt, None)

    def read(c, b, k=X, dt=1):
        return L.mcq4_kv8_read(c, b, k, W, dt, None)

    def attend(c, b, q=X, dt=1, heads=4, window=0, most=256, ws=None, n=0, stride=256, out=Y):
        return L.mcq4_kv8_attention(c, b, q, stride, 64, heads, dt, out, None, 1.0, 1, window, most, ws, n, None)

    for kw, want in BAD_CACHES:
        c = ref(_cache(**kw))
        assert [f(c, good[1]) for f in (append, read, attend)] == [want] * 3, kw
    for kw, want in BAD_BATCHES:
        b = ref(_batch(**kw))
        assert [f(good[0], b) for f in (append, read, attend)] == [want] * 3, kw
    for kw in (dict(T=3), dict(T=0)):
        assert [f(good[0], ref(_batch(**kw))) for f in (append, attend)] == [SHAPE] * 2
    assert append(*good, k=None) == INVALID and append(*good, dt=7) == INVALID and append(*good, stride=-1) == SHAPE
    assert append(*good, k=X + 1) == ALIGN and read(*good, k=X + 8) == ALIGN and read(*good, dt=3) == INVALID
    assert attend(*good, dt=0) == INVALID and attend(*good, heads=3) == SHAPE and attend(*good, window=-1) == SHAPE
    assert attend(*good, most=-1) == SHAPE and attend(*good, q=X + 8) == ALIGN and attend(*good, stride=252) == ALIGN
    assert attend(*good, out=Y + 4) == ALIGN and attend(*good, q=None) == INVALID
    # A long context is divided and needs what the query says.
    c, b = ref(_cache(num_pages=1000)), ref(_batch(width=500, table_stride=500))
    need = L.mcq4_kv8_attention_workspace_bytes(c, b, 4, 1, 0, 32000)
    assert need > 256 * 1024
    assert attend(c, b, most=32000) == WS and attend(c, b, most=32000, ws=0x50000, n=need - 1) == WS
    assert attend(c, b, most=32000, ws=0x50008, n=need) == ALIGN
    assert L.mcq4_kv8_attention_workspace_bytes(c, b, 3, 1, 0, 32000) == 0
