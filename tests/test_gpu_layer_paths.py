"""linear_mxfp4, qk_norm_rope, the pool and kv8_shared_attention by the native call path and by ctypes: the same bits."""
import pytest
import torch

import metalops_amd as mo
from metalops_amd import kv8, mxfp4, pool, rope

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(mxfp4._native is None, reason="the native call path is not built")]
I32 = torch.int32


def _same(a, b):
    a, b = ([t] if torch.is_tensor(t) else list(t) for t in (a, b))
    assert len(a) == len(b) and all(x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y) for x, y in zip(a, b))


class _Seen:
    """The extension, noting which functions gave a result."""

    def __init__(self, native):
        self.native, self.took = native, []

    def __getattr__(self, name):
        def call(*args):
            out = getattr(self.native, name)(*args)
            if out is not None:
                self.took.append(name)
            return out
        return call


def _both(monkeypatch, module, name, fn):
    seen = _Seen(module._native)
    with monkeypatch.context() as m:
        m.setattr(module, "_native", seen)
        a = fn()
    assert name in seen.took
    with monkeypatch.context() as m:
        m.setattr(module, "_native", None)
        b = fn()
    _same(a, b)
    return a


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_linear(dev, dtype, monkeypatch):
    W = mo.quantize_mxfp4(torch.randn(200, 256, device=dev))
    for M in (1, 33):
        X, m, r = (torch.randn(M, n, device=dev).to(dtype) for n in (256, 200, 200))
        for act in (None, "relu", "silu", "gelu", "gelu_tanh"):
            for bias in (None, torch.randn(200, device=dev), torch.randn(200, device=dev).to(dtype)):
                _both(monkeypatch, mxfp4, "mx_linear", lambda: mo.linear_mxfp4(X, *W, bias, act, m, r))
        _both(monkeypatch, mxfp4, "mx_linear", lambda: mo.linear_mxfp4(X, *W))


def test_rope(dev, monkeypatch):
    q, k = torch.randn(9, 4, 64, device=dev).bfloat16(), torch.randn(9, 2, 64, device=dev).bfloat16()
    f, w = torch.rand(24, device=dev), torch.randn(64, device=dev)
    pos = torch.randint(0, 5000, (3, 9), dtype=I32, device=dev)
    _both(monkeypatch, rope, "qk_norm_rope", lambda: mo.qk_norm_rope(q, k, pos[0], f, w, None, 1e-5))
    _both(monkeypatch, rope, "qk_norm_rope", lambda: mo.qk_norm_rope(q, k, pos, f, None, w, sections=(8, 10, 6), interleaved=True))


def test_pool(dev, monkeypatch):
    def life():
        p = mo.KV8Pool.empty(2, 30, 2, 32, 16)
        for c in p.caches:
            c.k_codes.view(torch.uint8).copy_(torch.arange(c.k_codes.numel(), device=dev).view(c.k_codes.shape) % 120)
        t, zero, lens = p.table(2, 5), torch.zeros(2, dtype=I32, device=dev), torch.tensor([20, 40], dtype=I32, device=dev)
        out = [mo.kv8_resize(p, t, zero, lens)]
        t, lens = mo.kv8_fork(p, t, lens, torch.tensor([1, 0, 1], dtype=I32, device=dev), True)
        more = lens + 7
        out += [mo.kv8_resize(p, t, lens, more), t, lens, p.refs] + [c.k_codes.view(torch.uint8) for c in p.caches]
        return out
    _both(monkeypatch, pool, "kv8_fork", life)
    _both(monkeypatch, pool, "kv8_resize", life)


@pytest.mark.parametrize("n", [1, 60])
def test_shared(dev, n, monkeypatch):
    c = mo.KV8Cache.empty(40, 2, 64, 16)
    for t in (c.k_codes, c.v_codes):
        t.view(torch.uint8).copy_(torch.randint(0, 110, t.shape, dtype=torch.uint8, device=dev))
    c.k_scales.fill_(120), c.v_scales.fill_(121)
    ids = torch.randperm(40, device=dev).to(I32)
    pt, t = ids[:8].view(2, 4), ids[8:36].view(4, 7)
    pl, cl = torch.tensor([50, 9], dtype=I32, device=dev), torch.tensor([100, 60, 77, 61], dtype=I32, device=dev)
    cu, groups = torch.tensor([0, n, 2 * n, 3 * n, 4 * n], dtype=I32, device=dev), torch.tensor([0, 3, 4], dtype=I32, device=dev)
    q = torch.randn(4 * n, 8, 64, device=dev).half()
    for kw in ({}, dict(cu_seqlens=cu, groups=groups, return_lse=True), dict(max_prefix=50, max_context=100, scale=0.3)):
        _both(monkeypatch, kv8, "kv8_shared_attention", lambda: mo.kv8_shared_attention(q, c, pt, pl, t, cl, **kw))
