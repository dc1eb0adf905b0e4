"""Offsets of the new tokens that leave rows of q to no sequence, and batches of more sequences than a wave has lanes,
against the oracle, through both attention kernels, with contexts in one part and in many.  Bounds: test_gpu_kv8."""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref
from test_gpu_kv8 import DT, Both, _check, _cum, _i32, _np, _rng

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[(rows, span) for rows in ("16", "128") for span in ("1", "64")], ids=lambda p: f"rows{p[0]}-span{p[1]}")
def kernel(request, monkeypatch):
    monkeypatch.setenv("MCQ4_KV8_ROWS", request.param[0])
    monkeypatch.setenv("MCQ4_KV8_SPAN", request.param[1])
    return request.param[0]


OFFSETS = [  # T, offsets, which sequences they count for
    (70, [0, 1, 40], [0, 1]),            # a batch padded to a fixed T
    (70, [25, 26, 70], [0, 1]),
    (300, [7, 7, 20], [0, 1]),
    (70, [0, 0, 0], [0, 1]),             # no new token at all
    (70, [70, 70, 70], [0, 1]),
    (70, [0, 30, 90], [0]),              # the last one leaves q
    (70, [-4, 30, 50], [1]),
    (70, [-9, -3, 500], []),
]


@pytest.mark.parametrize("T,cu,count", OFFSETS)
def test_rows_of_no_sequence(dev, kernel, T, cu, count):
    import metalops_amd as mo
    print(f"rest {kernel} {T} {cu}", flush=True)
    rng, H, G, D, page, context = _rng("rest", T, cu), 2, 3, 80, 64, [300, 150]
    both = Both(dev, rng, 2, 5, H, D, page)
    for dt in ("f16", "bf16"):
        q = torch.from_numpy(rng.normal(size=(T, H * G, D))).to(DT[dt])
        want, lse = np.zeros((T, H * G, D)), np.full((T, H * G), -np.inf)
        terms = {"av": np.zeros((T, H * G, D)), "vmax": np.zeros((T, H * G, 1)), "sabs": np.zeros((T, H * G, 1))}
        for b in count:
            a, z = cu[b], cu[b + 1]
            if a == z:
                continue
            o, s, t = ref.attention(_np(q)[a:z], both.ref, both.table[b:b + 1], context[b:b + 1], [0, z - a], D ** -0.5)
            want[a:z], lse[a:z] = o, s
            for k in t:
                terms[k][a:z] = t[k]
        for fill in (q.new_full(q.shape, float("nan"), device=dev), torch.full((T, H * G), float("nan"), device=dev)):
            del fill                    # what the outputs' memory holds before
        out, got = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32(context, dev), _i32(cu, dev), return_lse=True)
        none = np.isinf(lse)
        assert not _np(out)[none].any() and (_np(got)[none] == -np.inf).all()
        _check(out, want, terms, 300, D, dt)
        assert np.isfinite(_np(got)[~none]).all()


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("B,H,D", [(63, 1, 16), (64, 2, 64), (65, 2, 16), (130, 1, 64), (200, 2, 16)])
def test_many_sequences(dev, kernel, B, H, D, offsets):
    """Around and above 64 sequences, contexts of 0 to 150 tokens: tokens appended, then attended to."""
    import metalops_amd as mo
    print(f"many {kernel} B={B} H={H} D={D} {offsets}", flush=True)
    rng, page, G = _rng("many", B, D), 16, 3
    new = rng.integers(0, 5, B) if offsets else np.full(B, 2)
    if offsets:
        new[[0, B // 2, B - 1]] = 0, 20, 1
    start = rng.integers(0, 130, B)
    start[rng.integers(0, B, B // 4)] = 0
    cu, T = _cum(new), int(new.sum())
    both = Both(dev, rng, B, 10, H, D, page)
    table, gcu = _i32(both.table, dev), _i32(cu, dev) if offsets else None
    x = [torch.from_numpy(rng.normal(size=(T, H, D))).half() for _ in range(2)]
    for i in range(2):
        both.ref.append(i, _np(x[i]), both.table, start, cu)
    mo.kv8_append(both.gpu, x[0].to(dev), x[1].to(dev), table, _i32(start, dev), gcu)
    both.same()
    context = start + new
    context[1::7] = 0                     # rows that see nothing
    q = torch.from_numpy(rng.normal(size=(T, H * G, D))).bfloat16()
    want, lse, terms = ref.attention(_np(q), both.ref, both.table, context.tolist(), cu, D ** -0.5)
    for window in (0, 33):
        if window:
            want, lse, terms = ref.attention(_np(q), both.ref, both.table, context.tolist(), cu, D ** -0.5, True, window)
        out, got = mo.kv8_attention(q.to(dev), both.gpu, table, _i32(context, dev), gcu, window=window, return_lse=True)
        _check(out, want, terms, 150, D, "bf16")
        none = np.isinf(lse)
        assert np.array_equal(np.isinf(_np(got)), none) and not _np(out)[none].any()
        # Scores are sums of up to 64 products of about 1, off by far less than this; a wrong sequence is off by more.
        assert np.abs(_np(got)[~none] - lse[~none]).max() < 1e-3


@pytest.mark.parametrize("B", [65, 300])
def test_many_sequences_by_the_plan(dev, B):
    """The kernels and parts that the plan takes by itself: single tokens behind contexts of 0 to 2000."""
    import metalops_amd as mo
    rng, H, G, D, page = _rng("plan", B), 1, 4, 64, 64
    context = rng.integers(0, 2000, B)
    context[::9] = 0
    both = Both(dev, rng, B, 32, H, D, page)
    q = torch.from_numpy(rng.normal(size=(B, H * G, D))).half()
    want, lse, terms = ref.attention(_np(q), both.ref, both.table, context.tolist(), list(range(B + 1)), D ** -0.5)
    args = q.to(dev), both.gpu, _i32(both.table, dev), _i32(context, dev)
    first = mo.kv8_attention(*args)
    _check(first, want, terms, 2000, D, "f16")
    assert torch.equal(mo.kv8_attention(*args, _i32(np.arange(B + 1), dev)), first)


def test_offsets_that_give_tokens_to_many_sequences(dev, monkeypatch):
    """Offsets that fall and rise again, 512 sequences of all the tokens: 2^36 pieces of context, which no count holds.
    Nothing is promised of the output; the call ends, and later ones are right."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_KV8_ROWS", "16")
    T, G, B, W, D, page = 8192, 16, 1024, 16384, 16, 64
    cache = mo.KV8Cache.empty(2, 1, D, page, dev)
    q = torch.ones(T, G, D, dtype=torch.float16, device=dev)
    table = torch.zeros(B, W, dtype=torch.int32, device=dev)
    lens = torch.full((B,), W * page, dtype=torch.int32, device=dev)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    cu[1::2] = T
    mo.kv8_attention(q, cache, table, lens, cu, causal=False)
    torch.cuda.synchronize()
    monkeypatch.delenv("MCQ4_KV8_ROWS")
    rng = _rng("after")
    both = Both(dev, rng, 1, 80, 1, 64, 64)
    x = torch.from_numpy(rng.normal(size=(1, 4, 64))).half()
    want, _, terms = ref.attention(_np(x), both.ref, both.table, [5000], [0, 1], 0.125)
    _check(mo.kv8_attention(x.to(dev), both.gpu, _i32(both.table, dev), _i32([5000], dev)), want, terms, 5000, 64, "f16")
