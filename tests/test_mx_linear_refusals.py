"""What linear_mxfp4 refuses, in Python and at the C ABI (no GPU needed, nothing is launched)."""
import ctypes

import pytest
import torch

import metalops_amd as mo
from metalops_amd import _lib

U8 = torch.uint8
X, W, S, Y = 0x10000, 0x20000, 0x30000, 0x40000      # never dereferenced
INVALID, SHAPE, ALIGN, WS = (_lib.MCQ4_ERR_INVALID_ARG, _lib.MCQ4_ERR_SHAPE, _lib.MCQ4_ERR_ALIGNMENT, _lib.MCQ4_ERR_WORKSPACE)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_cpu_tensors_rejected_no_fallback():
    p, s = torch.zeros(8, 32, dtype=U8), torch.zeros(8, 2, dtype=U8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mo.linear_mxfp4(torch.zeros(2, 64), p, s)


def test_python(monkeypatch):
    from metalops_amd import mxfp4
    monkeypatch.setattr(mxfp4, "_require_device", lambda *a: None)
    p, s = torch.zeros(8, 32, dtype=U8), torch.zeros(8, 2, dtype=U8)
    x, y = torch.zeros(2, 64), torch.zeros(2, 8)
    with pytest.raises(AssertionError, match=r"X K dim \(96\) must match weight K \(64\)"):
        mo.linear_mxfp4(torch.zeros(2, 96), p, s)
    for kw, match in ((dict(activation="swish"), "activation must be one of"), (dict(activation="SILU"), "activation"),
                      (dict(bias=torch.zeros(7)), r"bias must be \(8,\)"), (dict(bias=torch.zeros(1, 8)), "bias"),
                      (dict(bias=torch.zeros(8).half()), "bias"), (dict(multiply=y[:1]), "multiply must be"), (dict(multiply=y.half()), "multiply"),
                      (dict(residual=torch.zeros(2, 9)), "residual must be"), (dict(residual=torch.zeros(2, 1, 8)), "residual")):
        with pytest.raises(RuntimeError, match=match):
            mo.linear_mxfp4(x, p, s, **kw)
    with pytest.raises(RuntimeError, match="float16, bfloat16 or float32"):
        mo.linear_mxfp4(x.double(), p, s)
    with pytest.raises(RuntimeError, match="K must be at least 32"):
        mo.linear_mxfp4(torch.zeros(2, 0), torch.zeros(8, 0, dtype=U8), torch.zeros(8, 0, dtype=U8))
    with pytest.raises(RuntimeError, match=r"\[N, K/2\]"):
        mo.linear_mxfp4(x, p[None], s[None])


def test_capi():
    call = _lib.lib.mcq4_linear_mxfp4

    def go(i=None, v=None, **kw):
        f = dict(bias=Y, multiply=X, residual=X, ld_multiply=8, ld_residual=8, bias_dtype=1, activation=2)
        f.update(kw)
        e = _lib.EpilogueStruct(**f)
        a = [X, 1, 64, W, S, ctypes.byref(e), Y, 8, 2, 64, 8, None, 0, None]
        return call(*[v if j == i else b for j, b in enumerate(a)])
    for i in (0, 3, 4, 5, 6):
        assert go(i, None) == INVALID
    assert go(1, 5) == INVALID
    assert go(2, 32) == SHAPE and go(7, 4) == SHAPE and go(8, 0) == SHAPE and go(9, 48) == SHAPE and go(10, 0) == SHAPE
    assert go(0, X + 8) == ALIGN and go(3, W + 4) == ALIGN and go(6, Y + 1) == ALIGN
    assert go(activation=5) == INVALID and go(activation=-1) == INVALID and go(bias_dtype=2) == INVALID and go(bias_dtype=7) == INVALID
    assert go(ld_multiply=7) == SHAPE and go(ld_residual=7) == SHAPE
    assert go(bias=Y + 1) == ALIGN and go(bias=Y + 2, bias_dtype=0) == ALIGN and go(multiply=X + 1) == ALIGN and go(residual=X + 1) == ALIGN
    M, K, N = 64, 14336, 512
    need = _lib.lib.mcq4_matmul_mxfp4_workspace_bytes(M, K, N, 1)
    assert need
    e = _lib.EpilogueStruct(ld_multiply=N, ld_residual=N)
    assert call(X, 1, K, W, S, ctypes.byref(e), Y, N, M, K, N, None, 0, None) == WS
    assert call(X, 1, K, W, S, ctypes.byref(e), Y, N, M, K, N, 0x50000, need - 1, None) == WS
