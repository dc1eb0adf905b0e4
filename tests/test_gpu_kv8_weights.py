"""Attention over the 8-bit cache where the weights of a row, or the scales of its pages, lie far apart, against the
64-bit oracle, through both kernels and with contexts in one part and in many.

A row's output may be off by the output's rounding (half a step) and by
  * P in fp16: 2^-11 of each weight.  A weight is rounded relative to the row's largest product of a weight and its
    page's scale, which stands at 2^14 at least in the kernel of few rows and at 2^PROMPT_LOG / 2 at least in that of
    prompts: where it is subnormal in fp16 it is off by half a step of 2^-24, so by 2^-25 / 2^14 (2^PROMPT_LOG / 2) of
    that product, times 448, the largest code;
  * scores in fp32: D + 4 roundings of 2^-24 of sum |q||k| scale, of a weight and of the weights' sum; exp2's 2^-22;
  * sums in fp32: one rounding of 2^-24 for each token, of the weighted sum of |v|."""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref
from test_gpu_kv8 import DT, Both, _cum, _i32, _np, _rng

pytestmark = pytest.mark.gpu

PROMPT_LOG = 7


def _terms(q, cache, table, context, cu, scale, causal, window):
    """(out, lse, sum of weights times |v|, largest weight times 448 page scales, sum |q||k| scale), rows that see
    nothing left at 0."""
    T, heads, D = q.shape
    G = heads // cache.H
    out, av = np.zeros((T, heads, D)), np.zeros((T, heads, D))
    lse, top, sabs = np.full((T, heads), -np.inf), np.zeros((T, heads, 1)), np.zeros((T, heads, 1))
    for b, L in enumerate(context):
        n = cu[b + 1] - cu[b]
        k, here = cache.values(0, table, b, L)
        v, _ = cache.values(1, table, b, L)
        pages = [cache._id(table, b, t // cache.page) for t in range(L)]
        vs = np.array([np.zeros(cache.H) if p is None else ref.scale_value(cache.bytes[1][p]) for p in pages])
        key = np.arange(L)
        for i in range(n):
            pos = L - n + i
            see = here & (key <= pos if causal else True) & (key > pos - window if window else True)
            t = cu[b] + i
            if not see.any():
                continue
            for hq in range(heads):
                kk, vv, qq = k[see, hq // G], v[see, hq // G], q[t, hq].astype(np.float64)
                s = kk @ qq * scale
                p = np.exp(s - s.max())
                out[t, hq], av[t, hq] = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
                lse[t, hq] = s.max() + np.log(p.sum())
                top[t, hq] = (p * vs[see, hq // G]).max() * 448 / p.sum()
                sabs[t, hq] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
    return out, lse, av, top, sabs


def _check(both, dev, q, context, cu, dt, rows, causal=True, window=0, scale=None):
    import metalops_amd as mo
    D, L = q.shape[2], max(context)
    scale = D ** -0.5 if scale is None else scale
    want, lse, av, top, sabs = _terms(_np(q), both.ref, both.table, context, cu, scale, causal, window)
    out, got = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32(context, dev), _i32(cu, dev), scale=scale,
                                causal=causal, window=window, return_lse=True)
    eps = torch.finfo(DT[dt]).eps
    ds = (D + 4) * 2.0 ** -24 * sabs + 2.0 ** -21
    least = 2.0 ** (14 if rows == "16" else PROMPT_LOG - 1)
    bound = av * (2.0 ** -11 + 2 * ds + (L + 8) * 2.0 ** -24) + L * 2.0 ** -25 / least * top
    bound = bound * (1 + eps) + np.abs(want) * eps / 2 + (2.0 ** -25 if dt == "f16" else 2.0 ** -134)
    err = np.abs(_np(out) - want)
    assert (err <= bound).all(), f"worst {np.nanmax(err / np.maximum(bound, 1e-300))} of the bound, {np.abs(err / want).max()} of the value"
    inf = np.isinf(lse)
    assert np.array_equal(np.isinf(_np(got)), inf)
    tol = ds[..., 0] + 2.0 ** -20 + L * 2.0 ** -24 + np.abs(np.where(inf, 0, lse)) * 2.0 ** -22
    np.testing.assert_array_less(np.abs(_np(got)[~inf] - lse[~inf]), tol[~inf])
    return out


@pytest.fixture(params=[(rows, span) for rows in ("16", "128") for span in ("1", "64")], ids=lambda p: f"rows{p[0]}-span{p[1]}")
def kernel(request, monkeypatch):
    monkeypatch.setenv("MCQ4_KV8_ROWS", request.param[0])
    monkeypatch.setenv("MCQ4_KV8_SPAN", request.param[1])
    return request.param[0]


@pytest.mark.parametrize("gap", [9, 14, 17])
@pytest.mark.parametrize("at", [0, 77, 1200])
def test_a_token_that_takes_the_weight(dev, kernel, gap, at):
    """One token `gap` nats above the others, whose value is 0: the output is what the others make."""
    print(f"sink {kernel} gap {gap} at {at}", flush=True)
    rng, L, D, page, new = _rng("sink", gap, at), 1300, 64, 64, 40
    both = Both(dev, rng, 1, -(-L // page), 1, D, page)
    # Channel 0 alone tells the sink from the others: q is positive there, the others' scores differ by about a nat.
    q = torch.from_numpy(np.abs(rng.normal(size=(new, 2, D))) * 0.05 + 0.5).to(torch.float16)
    k, v = rng.normal(size=(L, 1, D)) * 0.25, rng.normal(size=(L, 1, D)) * 0.5 + 1
    k[:, :, 0] = 0
    k[at] = 0
    k[at, :, 0] = 1.75 * 16 * gap / 14      # score 0.5 * 28 * gap / 14 at least
    v[at] = 0
    for i, x in enumerate((k, v)):
        both.ref.append(i, x, both.table, [0], [0, L])
        (both.gpu.k_codes, both.gpu.v_codes)[i].copy_(torch.from_numpy(np.ascontiguousarray(both.ref.codes[i] if i == 0 else both.ref.codes[i].swapaxes(2, 3))))
        (both.gpu.k_scales, both.gpu.v_scales)[i].copy_(torch.from_numpy(both.ref.bytes[i]))
    _check(both, dev, q, [L], [0, new], "f16", kernel, scale=1.0)
    _check(both, dev, q.bfloat16(), [L], [0, new], "bf16", kernel, causal=False, scale=1.0)


def _with_value_scales(dev, rng, scales, H, D, page):
    """One sequence whose pages have these scale bytes for their values (a byte, or one for each head)."""
    both = Both(dev, rng, 1, len(scales), H, D, page)
    for i, b in enumerate(scales):
        p = int(both.table[0, i])
        both.ref.bytes[1][p] = b
        both.gpu.v_scales[p] = torch.tensor(np.broadcast_to(b, (H,)).copy(), dtype=torch.uint8)
    return both


@pytest.mark.parametrize("scales", [[0], [0, 0, 0, 0, 0], [0, 120, 0, 0, 118], [120, 0, 1, 0, 2]])
@pytest.mark.parametrize("new", [1, 40])
def test_byte_0_is_the_smallest_scale(dev, kernel, new, scales):
    """Pages whose values have byte 0, alone (values around 2^-120) and beside others."""
    print(f"byte 0 {kernel} {new} {scales}", flush=True)
    rng = _rng("byte 0", new, scales)
    both = _with_value_scales(dev, rng, scales, 2, 64, 64)
    q = torch.from_numpy(rng.normal(size=(new, 4, 64)))
    for dt in ("bf16", "f16"):
        _check(both, dev, q.to(DT[dt]), [64 * len(scales)], [0, new], dt, kernel)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 40), (False, 40)])
def test_pages_that_a_row_does_not_see(dev, kernel, page, causal, window):
    """A page whose values are 2^40 larger, in each place in turn: rows that do not see it are what the others make,
    to the bit what they were without it."""
    import metalops_amd as mo
    print(f"unseen {kernel} page {page} {causal} {window}", flush=True)
    rng, L, new = _rng("unseen", page), 192, 150
    q = torch.from_numpy(rng.normal(size=(new, 2, 64))).bfloat16()      # where the page is seen, beyond fp16's range
    for big in range(0, L // page, max(1, 48 // page)):
        scales = [110] * (L // page)
        both = _with_value_scales(dev, rng, scales, 1, 64, page)
        args = q.to(dev), both.gpu, _i32(both.table, dev), _i32([L], dev), _i32([0, new], dev), 0.125, causal, window
        without = mo.kv8_attention(*args)
        p = int(both.table[0, big])
        both.ref.bytes[1][p] = 150
        both.gpu.v_scales[p] = 150
        out = _check(both, dev, q, [L], [0, new], "bf16", kernel, causal, window)
        pos, lo, hi = np.arange(L - new, L), big * page, (big + 1) * page
        sees = (pos >= lo if causal else np.full(new, True)) & (pos - window + 1 < hi if window else True)
        assert torch.equal(out[~sees], without[~sees]), big


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [1, 40])
def test_pages_without_weight(dev, kernel, new, page):
    """Pages whose values are 2^40 larger and whose tokens have 2^-60 of the weight, first, last and between."""
    print(f"light pages {kernel} {new} page {page}", flush=True)
    rng, L, D = _rng("light", page), 256, 64
    for big in (0, 1, L // page // 2, L // page - 1):
        both = _with_value_scales(dev, rng, [150 if i == big else 110 for i in range(L // page)], 1, D, page)
        q = torch.from_numpy(np.abs(rng.normal(size=(new, 2, D))) * 0.05 + 0.5)
        for i in range(L // page):      # channel 0: 0, or -448 * 2^-2 where q is 0.5 or more
            p = int(both.table[0, i])
            both.ref.bytes[0][p], both.ref.codes[0][p, :, :, 0] = 125 if i == big else 118, 0xFE if i == big else 0
            both.gpu.k_scales[p] = int(both.ref.bytes[0][p, 0])
            both.gpu.k_codes[p, :, :, 0] = 0xFE if i == big else 0
            both.ref.codes[0][p, :, :, 1:] = 0x20
            both.gpu.k_codes[p, :, :, 1:] = 0x20
        _check(both, dev, q.half(), [L], [0, new], "f16", kernel, scale=1.0)
        _check(both, dev, q.bfloat16(), [L], [0, new], "bf16", kernel, causal=False, scale=1.0)


def _large_scores(dev, new, byte):
    """Whatever of the weights is lost, outputs stay between the values, and lse is the largest score to 2^-16 of it."""
    import metalops_amd as mo
    rng, L, D = _rng("large", byte), 320, 64
    both = _with_value_scales(dev, rng, [118, 121, 118, 90, 119], 1, D, 64)
    for i in range(5):
        both.ref.bytes[0][both.table[0, i]] = byte
        both.gpu.k_scales[int(both.table[0, i])] = byte
    for sign in (1.0, -1.0):
        q = torch.from_numpy(rng.normal(size=(new, 4, D))).half()
        _, lse, _, _, _ = _terms(_np(q), both.ref, both.table, [L], [0, new], sign, True, 0)
        out, got = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32([L], dev), scale=sign, return_lse=True)
        v = np.abs(both.ref.values(1, both.table, 0, L)[0]).max()
        assert out.isfinite().all() and out.abs().max().item() <= v * (1 + 2.0 ** -9)
        assert (np.abs(_np(got) - lse) <= np.abs(lse) * 2.0 ** -16 + 1).all()


@pytest.mark.parametrize("byte", [137, 141, 143, 145, 146])
@pytest.mark.parametrize("new", [1, 40])
def test_large_scores(dev, kernel, new, byte):
    """Scores of 2^20 to 2^29."""
    print(f"large scores {kernel} {new} {byte}", flush=True)
    _large_scores(dev, new, byte)


@pytest.mark.parametrize("byte", [147, 148, 150, 152, 155, 160, 200])
@pytest.mark.parametrize("new", [1, 40])
def test_larger_scores_in_the_kernel_of_few_rows(dev, monkeypatch, new, byte):
    """Scores of up to 2^83, which that of prompts does not take."""
    monkeypatch.setenv("MCQ4_KV8_ROWS", "16")
    for span in ("1", "64"):
        monkeypatch.setenv("MCQ4_KV8_SPAN", span)
        print(f"larger scores {new} {byte} span {span}", flush=True)
        _large_scores(dev, new, byte)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_byte_255_is_nan(dev, kernel, page, window, D):
    """A page's scale that is NaN: rows that see one of its tokens are NaN in that head, others what they were."""
    import metalops_amd as mo
    print(f"byte 255 {kernel} page {page} {window} D={D}", flush=True)
    rng, L, new = _rng("byte 255", page), 500, 230
    both = Both(dev, rng, 1, -(-L // page), 2, D, page)
    q = torch.from_numpy(rng.normal(size=(new, 4, D))).half().to(dev)
    args = q, both.gpu, _i32(both.table, dev), _i32([L], dev)
    without, lse = mo.kv8_attention(*args, window=window, return_lse=True)
    pos = np.arange(L - new, L)
    for j in range(0, -(-L // page), max(1, 64 // page)):
        p = int(both.table[0, j])
        sees = (pos >= j * page) & ((pos - window + 1 < (j + 1) * page) if window else True)
        sees = torch.from_numpy(sees).to(dev)
        for which, scales in (("k", both.gpu.k_scales), ("v", both.gpu.v_scales)):
            kept = scales[p, 1].clone()
            scales[p, 1] = 255
            out, got = mo.kv8_attention(*args, window=window, return_lse=True)
            scales[p, 1] = kept
            assert out[sees, 2:].isnan().all(), (which, j)
            assert torch.equal(out[~sees], without[~sees]) and torch.equal(out[:, :2], without[:, :2]), (which, j)
            if which == "k":
                assert got[sees, 2:].isnan().all() and torch.equal(got[~sees], lse[~sees]), j
            else:      # of rows with the NaN: two computations, each off by less than (D + 4) 2^-24 sum |q||k| scale + L 2^-24, 2^-11
                assert torch.equal(got[~sees], lse[~sees]) and (got - lse).abs().max().item() < 2.0 ** -10, j


def test_the_largest_weight_is_not_rounded(dev, kernel):
    """32 tokens in pages of one scale: the error over many rows is that of fp16 weights whose largest is a power of
    two, computed here, with a tenth to spare for the other errors (2^-20 against 2^-12).  A largest weight that is
    rounded too makes it a third larger."""
    import metalops_amd as mo
    rng, B, G, D = _rng("largest"), 32, 16, 64
    both = Both(dev, rng, B, 1, 1, D, 32)
    both.ref.bytes[1][:] = 119
    both.gpu.v_scales.fill_(119)
    q = torch.from_numpy(rng.normal(size=(B, G, D))).half()
    out = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32([32] * B, dev), scale=0.125)
    want, model = np.zeros((B, G, D)), np.zeros((B, G, D))
    for b in range(B):
        k, v = (both.ref.values(i, both.table, b, 32)[0][:, 0] for i in range(2))
        s = _np(q)[b] @ k.T * 0.125
        p = np.exp(s - s.max(1, keepdims=True))
        want[b] = p @ v / p.sum(1, keepdims=True)
        model[b] = (p * 2.0 ** 7).astype(np.float16).astype(np.float64) @ v / (p * 2.0 ** 7).sum(1, keepdims=True)
    rms = lambda x: np.sqrt(((x.astype(np.float16).astype(np.float64) - want) ** 2).mean())
    assert rms(_np(out)) <= 1.1 * rms(model)
