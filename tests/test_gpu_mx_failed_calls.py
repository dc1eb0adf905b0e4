"""A call of the MXFP4 products or of the cache's attention that fails leaves the counters of the stream's workspace,
which all products share, at zero, whatever it left there."""
import pytest
import torch

from metalops_amd import _lib, kv8, mxfp4
from metalops_amd.quantization import _native, _workspace

pytestmark = pytest.mark.gpu

COUNTERS = 256 * 1024


class _Failing:
    """The library, but for one call that dirties its workspace's counters and fails."""

    def __init__(self, name, at, dirty):
        self._name, self._at, self._dirty = name, at, dirty

    def __getattr__(self, name):
        if name != self._name:
            return getattr(_LIB, name)

        def call(*args):
            self._dirty(args[self._at])
            return _lib.MCQ4_ERR_HIP
        return call


_LIB = _lib.lib


def _cache(dev):
    import metalops_amd as mo
    cache = mo.KV8Cache.empty(600, 2, 64, 64, dev)
    table = torch.arange(600, dtype=torch.int32, device=dev)[None]
    return lambda: mo.kv8_attention(torch.ones(1, 4, 64, dtype=torch.float16, device=dev), cache, table,
                                    torch.full((1,), 38000, dtype=torch.int32, device=dev))


def _products(dev):
    import metalops_amd as mo
    w = mo.quantize_mxfp4(torch.ones(64, 4096, device=dev))
    x = torch.ones(4, 4096, dtype=torch.float16, device=dev)
    xp = mo.quantize_mxfp4(x)
    return lambda: mo.matmul_mxfp4(x, *w), lambda: mo.matmul_mxfp4_mxfp4(*xp, *w)


@pytest.mark.parametrize("name,at", [("mcq4_matmul_mxfp4", 10), ("mcq4_matmul_mxfp4_mxfp4", 10), ("mcq4_kv8_attention", 13)])
def test_the_python_path(dev, monkeypatch, name, at):
    monkeypatch.setenv("MCQ4_MX_PATH", "7")
    monkeypatch.setenv("MCQ4_MX_SPLIT", "2")
    fn = {"mcq4_matmul_mxfp4": 0, "mcq4_matmul_mxfp4_mxfp4": 1}.get(name)
    fn = _cache(dev) if fn is None else _products(dev)[fn]
    want = fn()
    for mod in (kv8, mxfp4):
        monkeypatch.setattr(mod, "_native", None)
    stream = torch.cuda.current_stream(dev).cuda_stream
    ws = _workspace.get(dev if dev.index is not None else torch.device("cuda", 0), stream, COUNTERS)

    def dirty(ptr):
        assert ptr == ws.data_ptr()
        ws[:COUNTERS].fill_(1)
    fn()
    monkeypatch.setattr(_lib, "lib", _Failing(name, at, dirty))
    with pytest.raises(RuntimeError):
        fn()
    monkeypatch.setattr(_lib, "lib", _LIB)
    left = ws[:COUNTERS].clone()
    ws[:COUNTERS].zero_()
    assert not bool(left.any())
    assert torch.equal(fn(), want)


@pytest.mark.skipif(_native is None, reason="the native call path is not built")
@pytest.mark.parametrize("packed", [False, True])
def test_the_native_path(dev, monkeypatch, packed):
    """Too many rows: refused after the workspace was fetched, before any launch."""
    monkeypatch.setenv("MCQ4_MX_PATH", "1")
    monkeypatch.setenv("MCQ4_MX_SPLIT", "2")
    M, K, N = (1 << 20) + 1, 256, 16
    u8 = dict(dtype=torch.uint8, device=dev)
    w = torch.zeros(N, K // 2, **u8), torch.zeros(N, K // 32, **u8)
    if packed:
        call = lambda: _native.mx_matmul_mx(torch.zeros(M, K // 2, **u8), torch.zeros(M, K // 32, **u8), *w, torch.float16)
    else:
        call = lambda: _native.mx_matmul(torch.zeros(M, K, dtype=torch.float16, device=dev), *w)
    s = torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        need = max(_LIB.mcq4_matmul_mxfp4_mxfp4_workspace_bytes(M, K, N), _LIB.mcq4_matmul_mxfp4_workspace_bytes(M, K, N, 1))
        assert need > COUNTERS
        ws = _native.workspace(0, s.cuda_stream, need)
        ws[:COUNTERS].fill_(1)
        assert call() is None
        left = ws[:COUNTERS].clone()
        ws[:COUNTERS].zero_()
    torch.cuda.synchronize()
    assert not bool(left.any())
