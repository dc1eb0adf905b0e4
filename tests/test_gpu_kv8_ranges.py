"""The 8-bit cache over the whole range of its element types, and attention over many parts, against the oracle.
Codes and scales are compared byte for byte; attention has the bounds of test_gpu_kv8."""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref
from test_gpu_kv8 import DT, Both, _check, _i32, _np, _rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stride", [1, 257, 4097])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_finite_value(dev, dtype, stride):
    """All bit patterns that are finite, in order (a page holds neighbours) and dealt out over the pages (a page holds all
    magnitudes); the values behind them get the patterns from the other end."""
    import metalops_amd as mo
    bits = ((np.arange(65536) * stride) % 65536).astype(np.uint16)
    k = torch.from_numpy(bits.view(np.int16)).view(DT[dtype])
    k = torch.where(k.isfinite(), k, torch.zeros_like(k)).view(4096, 1, 16)
    v = k.flip(0)
    both = Both(dev, _rng("every", dtype), 1, 256, 1, 16, 16)
    for i, x in enumerate((k, v)):
        both.ref.append(i, _np(x), both.table, [0], [0, 4096])
    mo.kv8_append(both.gpu, k.to(dev), v.to(dev), _i32(both.table, dev), _i32([0], dev))
    both.same()


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_not_finite(dev, dtype, odd):
    """Infinities and NaN in some pages and heads and not in others, with rows at aligned and at odd addresses."""
    import metalops_amd as mo
    rng = _rng("odd", dtype)
    both = Both(dev, rng, 2, 3, 2, 64, 64)
    x = torch.from_numpy(rng.normal(size=(2, 180, 2, 64))).to(DT[dtype])
    x[0, 3, 1, 5], x[0, 100, 0, :], x[1, 7, 0, 9], x[1, 179, 1, 63] = float("inf"), float("nan"), -float("inf"), float("nan")
    for i in range(2):
        both.ref.append(i, _np(x[i]), both.table, [5, 0], [0, 90, 180])
    g = x.to(dev)
    if odd:
        g = torch.cat([g.new_zeros(2, 180, 2, 1), g], 3)[..., 1:]
    mo.kv8_append(both.gpu, g[0], g[1], _i32(both.table, dev), _i32([5, 0], dev), _i32([0, 90, 180], dev))
    for codes in (both.gpu.k_codes, both.gpu.v_codes, *both.ref.codes):      # NaN's sign bit is not fixed by the definition
        codes[(codes & 127) == 127] = 127
    both.same()


@pytest.mark.parametrize("H,G,D,page", [(1, 1, 16, 64), (1, 16, 256, 128), (2, 3, 80, 16), (1, 4, 128, 256)])
def test_many_parts(dev, monkeypatch, H, G, D, page):
    """A part for each piece of 64 tokens: contexts of 71 pieces, of one, of two, and an empty one."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_KV8_ROWS", "16")
    monkeypatch.setenv("MCQ4_KV8_SPAN", "1")
    rng, ctx = _rng("parts", D), [4500, 64, 65, 0]
    both = Both(dev, rng, 4, -(-4500 // page), H, D, page)
    q = torch.from_numpy(rng.normal(size=(4, H * G, D))).half()
    want, lse, terms = ref.attention(_np(q), both.ref, both.table, ctx, [0, 1, 2, 3, 4], D ** -0.5)
    args = q.to(dev), both.gpu, _i32(both.table, dev), _i32(ctx, dev)
    first = mo.kv8_attention(*args)
    _check(first, want, terms, 4500, D, "f16")
    for _ in range(3):
        out, got = mo.kv8_attention(*args, return_lse=True)
        assert torch.equal(out, first)
    assert np.array_equal(np.isinf(_np(got)), np.isinf(lse)) and np.allclose(_np(got)[:3], lse[:3], atol=1e-3)
