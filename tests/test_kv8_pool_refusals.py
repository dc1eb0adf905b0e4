"""What the pool's calls refuse, in Python and at the C ABI (no GPU needed, nothing is launched)."""
import ctypes

import pytest
import torch

import metalops_amd as mo
from metalops_amd import _lib

I32 = torch.int32
INVALID, SHAPE, ALIGN, WS = (_lib.MCQ4_ERR_INVALID_ARG, _lib.MCQ4_ERR_SHAPE, _lib.MCQ4_ERR_ALIGNMENT, _lib.MCQ4_ERR_WORKSPACE)
A, B, C = 0x10000, 0x20000, 0x30000      # never dereferenced


def test_pool():
    pool = mo.KV8Pool.empty(2, 5, 1, 16, 16, "cpu")
    assert pool.refs.tolist() == [0] * 5 and "layers=2" in repr(pool) and pool.table(2, 3).tolist() == [[-1] * 3] * 2
    with pytest.raises(AttributeError):
        pool.refs = torch.zeros(5, dtype=I32)
    c = pool.caches[0]
    for bad in ([], [c, mo.KV8Cache.empty(6, 1, 16, 16, "cpu")], [c, mo.KV8Cache.empty(5, 2, 16, 16, "cpu")], [c, mo.KV8Cache.empty(5, 1, 16, 32, "cpu")]):
        with pytest.raises(RuntimeError):
            mo.KV8Pool(bad)
    for refs in (torch.zeros(4, dtype=I32), torch.zeros(5), torch.zeros(10, dtype=I32)[::2]):
        with pytest.raises(RuntimeError, match="refs"):
            mo.KV8Pool([c], refs)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_cpu_tensors_rejected_no_fallback():
    pool, t, n = mo.KV8Pool.empty(1, 5, 1, 16, 16, "cpu"), torch.zeros(1, 2, dtype=I32), torch.zeros(1, dtype=I32)
    for call in (lambda: mo.kv8_fork(pool, t, n, n), lambda: mo.kv8_resize(pool, t, n, n), lambda: mo.kv8_compact(pool, t),
                 lambda: mo.kv8_copy_pages(pool, n, n)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_python(monkeypatch):
    from metalops_amd import pool as module
    monkeypatch.setattr(module, "_require_device", lambda *a: None)
    pool = mo.KV8Pool.empty(1, 5, 1, 16, 16, "cpu")
    t, n = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32)
    for bad in (t.long(), t[0], t.float()):
        for call in (lambda: mo.kv8_fork(pool, bad, n, n), lambda: mo.kv8_resize(pool, bad, n, n), lambda: mo.kv8_compact(pool, bad)):
            with pytest.raises(RuntimeError, match="block_table"):
                call()
    for bad in (torch.zeros(3, 2, dtype=I32).t(), torch.zeros(1, 3, dtype=I32).expand(2, 3)):
        for call in (lambda: mo.kv8_resize(pool, bad, n, n), lambda: mo.kv8_compact(pool, bad)):
            with pytest.raises(RuntimeError, match="in place"):
                call()
    for bad in (n.long(), n[:1], n[None]):
        with pytest.raises(RuntimeError, match="lens"):
            mo.kv8_fork(pool, t, bad, n)
        with pytest.raises(RuntimeError, match="lens"):
            mo.kv8_resize(pool, t, bad, n)
        with pytest.raises(RuntimeError, match="new_lens"):
            mo.kv8_resize(pool, t, n, bad)
    with pytest.raises(RuntimeError, match="parents"):
        mo.kv8_fork(pool, t, n, n.long())
    for src, dst in ((n.long(), n), (n, n[:1]), (n, n.float()), (t, n)):
        with pytest.raises(RuntimeError, match="src|dst"):
            mo.kv8_copy_pages(pool, src, dst)


def _pool(**kw):
    f = dict(tensors=A, refs=B, num_pages=9, layers=2, kv_heads=2, head_dim=64, page_size=64)
    f.update(kw)
    return ctypes.byref(_lib.Kv8PoolStruct(**f))


def test_capi():
    L = _lib.lib
    need_r, need_c = L.mcq4_kv8_resize_workspace_bytes(_pool(), 3), L.mcq4_kv8_compact_workspace_bytes(_pool())
    assert need_r and need_c

    def fork(p=None, **kw):
        f = dict(block_table=A, stride=4, batch=3, width=4, lens=B, parents=B, rows=5, out=C, out_lens=C, release=0)
        f.update(kw)
        return L.mcq4_kv8_fork(p or _pool(), *f.values(), None)

    def resize(p=None, **kw):
        f = dict(block_table=A, stride=4, batch=3, width=4, lens=B, new_lens=B, missing=C, ws=A, ws_bytes=need_r)
        f.update(kw)
        return L.mcq4_kv8_resize(p or _pool(), *f.values(), None)

    def compact(p=None, **kw):
        f = dict(names=A, live=B, ws=C, ws_bytes=need_c)
        f.update(kw)
        return L.mcq4_kv8_compact(p or _pool(), *f.values(), None)

    def copy(p=None, **kw):
        f = dict(src=A, dst=B, n=3)
        f.update(kw)
        return L.mcq4_kv8_copy_pages(p or _pool(), *f.values(), None)

    def rename(**kw):
        f = dict(block_table=A, stride=4, batch=3, width=4, names=B, num_pages=9)
        f.update(kw)
        return L.mcq4_kv8_rename(*f.values(), None)
    for call in (fork, resize, compact, copy):
        for kw in (dict(tensors=None), dict(refs=None)):
            assert call(_pool(**kw)) == INVALID
        for kw in (dict(num_pages=0), dict(num_pages=1 << 31), dict(layers=0), dict(layers=1 << 17), dict(kv_heads=0), dict(kv_heads=70000),
                   dict(head_dim=72), dict(head_dim=272), dict(page_size=48), dict(page_size=512), dict(kv_heads=65535, head_dim=256, page_size=256)):
            assert call(_pool(**kw)) == SHAPE
        assert call(_pool(tensors=A + 4)) == ALIGN and call(_pool(refs=B + 2)) == ALIGN
    assert L.mcq4_kv8_fork(None, A, 4, 3, 4, B, B, 5, C, C, 0, None) == INVALID
    for call in (fork, resize, rename):
        assert call(block_table=None) == INVALID and call(block_table=A + 2) == ALIGN
        assert call(stride=3) == SHAPE and call(batch=0) == SHAPE and call(batch=1 << 21) == SHAPE and call(width=0) == SHAPE
        assert call(width=1 << 29, stride=1 << 29) == SHAPE
    for name in ("lens", "parents", "out", "out_lens"):
        assert fork(**{name: None}) == INVALID and fork(**{name: A + 2}) == ALIGN
    assert fork(rows=0) == SHAPE and fork(rows=1 << 21) == SHAPE
    for name in ("lens", "new_lens", "missing"):
        assert resize(**{name: None}) == INVALID and resize(**{name: A + 2}) == ALIGN
    assert resize(ws=None) == WS and resize(ws_bytes=need_r - 1) == WS and resize(ws=A + 8) == ALIGN
    for name in ("names", "live"):
        assert compact(**{name: None}) == INVALID and compact(**{name: A + 2}) == ALIGN
    assert compact(ws=None) == WS and compact(ws_bytes=need_c - 1) == WS and compact(ws=A + 8) == ALIGN
    for name in ("src", "dst"):
        assert copy(**{name: None}) == INVALID and copy(**{name: A + 2}) == ALIGN
    assert copy(n=0) == SHAPE and copy(n=1 << 31) == SHAPE
    assert rename(names=None) == INVALID and rename(names=B + 2) == ALIGN and rename(num_pages=0) == SHAPE
    assert L.mcq4_kv8_resize_workspace_bytes(_pool(layers=0), 3) == 0 and L.mcq4_kv8_resize_workspace_bytes(_pool(), 0) == 0
    assert L.mcq4_kv8_compact_workspace_bytes(_pool(page_size=8)) == 0
