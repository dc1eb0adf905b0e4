"""What qk_norm_rope refuses, in Python and at the C ABI (no GPU needed, nothing is launched)."""
import ctypes

import pytest
import torch

import metalops_amd as mo
from metalops_amd import _lib

INVALID, SHAPE, ALIGN = _lib.MCQ4_ERR_INVALID_ARG, _lib.MCQ4_ERR_SHAPE, _lib.MCQ4_ERR_ALIGNMENT
X, Y, P, F = 0x10000, 0x20000, 0x30000, 0x40000      # never dereferenced


def _args(**kw):
    a = dict(q=torch.zeros(5, 4, 64), k=torch.zeros(5, 2, 64), positions=torch.zeros(5, dtype=torch.int32), inv_freq=torch.zeros(32))
    a.update(kw)
    return a


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_cpu_tensors_rejected_no_fallback():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mo.qk_norm_rope(**_args())


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 256)), r"q must be \[T, heads, D\]"), (dict(k=torch.zeros(5, 2, 64).half()), "both be"),
    (dict(q=torch.zeros(5, 4, 64).double(), k=torch.zeros(5, 2, 64).double()), "both be"), (dict(k=torch.zeros(4, 2, 64)), "one T and D"),
    (dict(k=torch.zeros(5, 2, 32)), "one T and D"), (dict(k=torch.zeros(5, 0, 64)), "must have heads"),
    (dict(q=torch.zeros(5, 4, 60), k=torch.zeros(5, 2, 60)), "multiple of 8"), (dict(q=torch.zeros(5, 4, 520), k=torch.zeros(5, 2, 520)), "up to 512"),
    (dict(inv_freq=torch.zeros(30)), "multiple of 4"), (dict(inv_freq=torch.zeros(36)), "multiple of 4"), (dict(inv_freq=torch.zeros(0)), "multiple of 4"),
    (dict(inv_freq=torch.zeros(32).half()), "float32"), (dict(inv_freq=torch.zeros(1, 32)), "1-dimensional"),
    (dict(positions=torch.zeros(5)), "int32"), (dict(positions=torch.zeros(5, dtype=torch.int64)), "int32"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), "positions must be"), (dict(positions=torch.zeros(5, 1, dtype=torch.int32)), "positions must be"),
    (dict(sections=(16, 15)), "add up to 32"), (dict(sections=(16, 16)), "positions must be"), (dict(sections=()), "1 to 4"),
    (dict(sections=(8, 8, 8, 4, 4)), "1 to 4"), (dict(sections=(40, -8)), "1 to 4"),
    (dict(q_weight=torch.zeros(32)), "q_weight"), (dict(k_weight=torch.zeros(64).double()), "k_weight"), (dict(out=(torch.zeros(5, 4, 64),)), "two tensors")])
def test_python(kw, match):
    with pytest.raises(RuntimeError, match=match):
        mo.qk_norm_rope(**_args(**kw))


def test_outputs(monkeypatch):
    from metalops_amd import rope
    monkeypatch.setattr(rope, "_require_device", lambda *a: None)
    a = _args()
    for bad, match in ((torch.zeros(5, 4, 32), "output of q"), (torch.zeros(5, 4, 64).half(), "output of q"),
                       (torch.zeros(5, 64, 4).transpose(1, 2), "neighbouring"), (torch.zeros(1, 4, 64).expand(5, 4, 64), "broadcast")):
        with pytest.raises(RuntimeError, match=match):
            mo.qk_norm_rope(**a, out=(bad, a["k"]))


def test_capi():
    def go(side=None, **kw):
        heads = dict(x=X, out=Y, weight=None, token_stride=256, head_stride=64, out_token_stride=256, out_head_stride=64, heads=4, weight_dtype=0)
        q, k = dict(heads), dict(heads)
        if side:
            (q if side == "q" else k).update(kw)
            kw = {}
        f = dict(positions=P, inv_freq=F, axis_stride=5, T=5, sections=(32, 0, 0, 0), axes=1, head_dim=64, rotary_dim=64, interleaved=0, dtype=1,
                 eps=1e-6)
        f.update(kw)
        f["sections"] = (ctypes.c_int32 * 4)(*f["sections"])
        return _lib.lib.mcq4_qk_norm_rope(ctypes.byref(_lib.RopeStruct(q=_lib.RopeHeadsStruct(**q), k=_lib.RopeHeadsStruct(**k), **f)), None)
    assert _lib.lib.mcq4_qk_norm_rope(None, None) == INVALID
    assert go(positions=None) == INVALID and go(inv_freq=None) == INVALID and go(dtype=4) == INVALID
    for side in "qk":
        assert go(side, x=None) == INVALID and go(side, out=None) == INVALID and go(side, weight=X, weight_dtype=5) == INVALID
        assert go(side, heads=0) == SHAPE and go(side, heads=70000) == SHAPE and go(side, token_stride=-1) == SHAPE and go(side, out_head_stride=-8) == SHAPE
        assert go(side, x=X + 1) == ALIGN and go(side, out=Y + 1) == ALIGN and go(side, weight=X + 2, weight_dtype=0) == ALIGN
    assert go(head_dim=60) == SHAPE and go(head_dim=520) == SHAPE and go(head_dim=0) == SHAPE and go(rotary_dim=72) == SHAPE
    assert go(rotary_dim=60) == SHAPE and go(rotary_dim=0) == SHAPE and go(rotary_dim=56) == SHAPE and go(T=0) == SHAPE and go(T=1 << 25) == SHAPE
    assert go(axes=0) == SHAPE and go(axes=5) == SHAPE and go(axes=2, sections=(16, 15, 0, 0)) == SHAPE and go(axes=2, sections=(40, -8, 0, 0)) == SHAPE
    assert go(axes=2, sections=(16, 16, 0, 0), axis_stride=4) == SHAPE
    assert go(positions=P + 2) == ALIGN and go(inv_freq=F + 4) == ALIGN
