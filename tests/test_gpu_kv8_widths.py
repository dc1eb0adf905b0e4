"""Attention over the 8-bit cache at every width of a head, through both kernels, against the 64-bit oracle.
Bounds: test_gpu_kv8."""
import pytest
import torch

from oracle import mx_ref as ref
from test_gpu_kv8 import DT, Both, _check, _cum, _i32, _np, _rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("rows", ["16", "128"])
@pytest.mark.parametrize("D", range(16, 257, 16))
def test_every_width(dev, monkeypatch, D, rows, page):
    """Contexts of several pieces of 64 tokens, whole and in parts, with rows of one wave and of several."""
    import metalops_amd as mo
    print(f"width {D} rows {rows} page {page}", flush=True)
    monkeypatch.setenv("MCQ4_KV8_ROWS", rows)
    rng, new, context = _rng("width", D, page), [2, 75], [150, 260]
    both = Both(dev, rng, 2, -(-260 // page), 1, D, page)
    q = torch.from_numpy(rng.normal(size=(77, 2, D)))
    for dt in ("f16", "bf16"):
        x = q.to(DT[dt])
        want, _, terms = ref.attention(_np(x), both.ref, both.table, context, _cum(new), D ** -0.5)
        for span in ("1", "64"):
            monkeypatch.setenv("MCQ4_KV8_SPAN", span)
            out = mo.kv8_attention(x.to(dev), both.gpu, _i32(both.table, dev), _i32(context, dev), _i32(_cum(new), dev))
            _check(out, want, terms, 260, D, dt)
