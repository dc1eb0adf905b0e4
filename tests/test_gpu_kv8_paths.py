"""Both attention kernels over the 8-bit cache, and contexts in one part and in many, each forced,
against the 64-bit oracle.  The bounds are those of test_gpu_kv8."""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref
from test_gpu_kv8 import DT, Both, _check, _cum, _i32, _np, _rng

pytestmark = pytest.mark.gpu

CASES = [  # new tokens, contexts, H, G, D, page, causal, window
    ([1], [1], 1, 1, 16, 16, True, 0),
    ([1, 1, 1], [63, 65, 700], 2, 4, 128, 64, True, 0),
    ([3, 3], [200, 4], 2, 2, 96, 64, True, 0),
    ([5, 1, 0, 40], [5, 300, 77, 60], 2, 3, 128, 64, True, 0),
    ([20, 33], [20, 500], 2, 4, 64, 16, False, 0),
    ([12], [7], 2, 2, 64, 64, True, 0),
    ([140, 70], [300, 70], 1, 2, 160, 64, True, 0),
    ([150], [150], 1, 1, 192, 256, True, 50),
    ([130, 65], [130, 400], 1, 5, 80, 16, True, 0),
    ([100], [260], 2, 1, 256, 32, False, 0),
    ([33], [600], 1, 16, 224, 128, True, 200),
    ([64, 1], [1000, 900], 3, 7, 48, 32, True, 333),
]


@pytest.mark.parametrize("span", ["1", "3", "64"])
@pytest.mark.parametrize("rows", ["16", "128"])
@pytest.mark.parametrize("new,context,H,G,D,page,causal,window", CASES)
def test_each_kernel(dev, monkeypatch, new, context, H, G, D, page, causal, window, rows, span):
    import metalops_amd as mo
    print(f"kv8 rows {rows} span {span} {new} {context} H={H} G={G} D={D} page={page} {causal} {window}", flush=True)
    monkeypatch.setenv("MCQ4_KV8_ROWS", rows)
    monkeypatch.setenv("MCQ4_KV8_SPAN", span)
    rng = _rng(new, context)
    both = Both(dev, rng, len(new), -(-max(context) // page), H, D, page)
    T, cu = sum(new), _cum(new)
    for dtype in ("f16", "bf16"):
        q = torch.from_numpy(rng.normal(size=(T, H * G, D))).to(DT[dtype])
        want, lse, terms = ref.attention(_np(q), both.ref, both.table, context, cu, D ** -0.5, causal, window)
        gcu = None if len(set(new)) == 1 else _i32(cu, dev)
        out, got = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32(context, dev), gcu, causal=causal, window=window,
                                    return_lse=True)
        _check(out, want, terms, max(context), D, dtype)
        inf = np.isinf(lse)
        assert np.array_equal(np.isinf(_np(got)), inf) and not _np(out)[inf].any()
        ds = (D + 4) * 2.0 ** -24 * terms["sabs"][..., 0] + 2.0 ** -20 + max(context) * 2.0 ** -24
        np.testing.assert_array_less(np.abs(_np(got)[~inf] - lse[~inf]), (ds + np.abs(np.where(inf, 0, lse)) * 2.0 ** -22)[~inf])


@pytest.mark.parametrize("span", ["1", "64"])
@pytest.mark.parametrize("rows", ["16", "128"])
def test_rising_scores(dev, monkeypatch, rows, span):
    """Scores that grow along the context, by a little and by a lot from piece to piece, and fall again."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_KV8_ROWS", rows)
    monkeypatch.setenv("MCQ4_KV8_SPAN", span)
    rng = _rng("rise")
    H, D, page, L, new = 1, 64, 64, 640, 40
    for step in (0, 2, 9):
        both = Both(dev, rng, 1, L // page, H, D, page)
        for i in range(L // page):                        # K's scale grows, then falls
            b = 110 + step * min(i, L // page - i) // 2
            both.ref.bytes[0][both.table[0, i]] = b
            both.gpu.k_scales[int(both.table[0, i])] = b
        q = torch.from_numpy(rng.normal(size=(new, 2 * H, D))).half()
        want, _, terms = ref.attention(_np(q), both.ref, both.table, [L], [0, new], 0.125)
        out = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32([L], dev), scale=0.125)
        _check(out, want, terms, L, D, "f16")


@pytest.mark.parametrize("rows", ["16", "128"])
def test_nan_of_v_in_each_kernel(dev, monkeypatch, rows):
    """A NaN that some rows see and others do not, in a first, middle and last piece."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_KV8_ROWS", rows)
    rng = _rng("nan v")
    H, G, D, page, L, new = 2, 2, 96, 32, 300, 180
    both = Both(dev, rng, 1, 10, H, D, page)
    q = torch.from_numpy(rng.normal(size=(new, H * G, D))).half().to(dev)
    table, ctx = _i32(both.table, dev), _i32([L], dev)
    clean = mo.kv8_attention(q, both.gpu, table, ctx)
    for t in (5, 120, 121, 200, 255, 299):
        pg, slot = int(both.table[0, t // page]), t % page
        kept = both.gpu.v_codes[pg, 1, 70, slot].clone()
        both.gpu.v_codes[pg, 1, 70, slot] = 255
        out = mo.kv8_attention(q, both.gpu, table, ctx)
        both.gpu.v_codes[pg, 1, 70, slot] = kept
        hit = torch.zeros(new, H * G, D, dtype=torch.bool, device=dev)
        hit[max(0, t - (L - new)):, G:, 70] = True
        assert torch.equal(out.isnan(), hit)
        assert torch.equal(out[~hit], clean[~hit])
