"""qk_norm_rope on the GPU against the formula in 64 bits.

A normalized channel is off by 2^-20 of itself (a sum of squares in 14 steps, half of whose error
counts, an inverse square root of 2 ulp, three products), a sine or cosine by 2^-22 of 1, and the
rotation's products and sum by 2^-23: 2^-19 of the pair's magnitudes together covers it.  Then comes
the result's own rounding, half a step or half the smallest subnormal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _exact(x, w, pos, inv_freq, sections, eps, interleaved):
    """The result and what it may be off by, fp64."""
    half = len(inv_freq)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    angle = pos.double()[axis].t() * inv_freq.double()               # [T, half]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    y = x.double()
    if w is not None:
        y = y * (y.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    y = y.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    ya, yb = y[..., a].clone(), y[..., b].clone()
    off = 2.0 ** -20 * y.abs() if w is not None else torch.zeros_like(y)
    off[..., a] = off[..., b] = 2.0 ** -19 * (ya.abs() + yb.abs())
    y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
    f = torch.finfo(x.dtype)
    return y, off + f.eps / 2 * (y.abs() + off) + f.smallest_normal * f.eps / 2


def _check(got, x, *args):
    want, off = _exact(x, *args)
    assert got.dtype == x.dtype and got.shape == x.shape
    wrong = ((got.double() - want).abs() > off).nonzero()
    assert len(wrong) == 0, (len(wrong), wrong[0].tolist(), got[tuple(wrong[0])].item(), want[tuple(wrong[0])].item())


def _inputs(dev, dtype, T, H, Hk, D, half, axes=1, weights=None, seed=0, far=200000):
    g = torch.Generator().manual_seed(seed + T + H + D)
    qkv = (torch.randn(T, H + 2 * Hk, D, generator=g) * (1 + 7 * (torch.rand(D, generator=g) < 0.05))).to(DT[dtype]).to(dev)
    pos = torch.randint(0, far, (axes, T), generator=g, dtype=torch.int32).to(dev)
    inv = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(dev)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(DT[weights]).to(dev) if weights else None for _ in range(2)]
    return qkv[:, :H], qkv[:, H:H + Hk], pos, inv, w


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T", [1, 3, 130, 2600])
@pytest.mark.parametrize("H,Hk,D,R,axes,weights,interleaved", [
    (32, 8, 128, 128, (64,), "f32", False), (32, 8, 128, 128, (64,), "bf16", True), (3, 1, 64, 64, (10, 22), "", False),
    (7, 7, 80, 80, (8, 16, 16), "f16", False), (5, 2, 256, 64, (1, 9, 3, 19), "bf16", False), (2, 1, 8, 8, (4,), "f32", True),
    (1, 1, 512, 504, (0, 252), "f32", False), (9, 3, 192, 96, (48,), "", True), (4, 1, 40, 16, (8,), "f16", False)])
def test_formula(dev, dtype, T, H, Hk, D, R, axes, weights, interleaved):
    import metalops_amd as mo
    print(f"rope {dtype} T={T} {H}+{Hk} x {D}, {R} turned, {axes} {weights} {interleaved}", flush=True)
    q, k, pos, inv, w = _inputs(dev, dtype, T, H, Hk, D, R // 2, len(axes), weights)
    before = q.clone(), k.clone()
    oq, ok = mo.qk_norm_rope(q, k, pos, inv, *w, eps=1e-5, sections=axes, interleaved=interleaved)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1]) and oq.is_contiguous() and ok.is_contiguous()
    _check(oq, q, w[0], pos, inv, axes, 1e-5, interleaved)
    _check(ok, k, w[1], pos, inv, axes, 1e-5, interleaved)


def test_layouts_and_outputs(dev):
    """One axis with and without a dimension for it, strides and alignments of every tensor, results in place."""
    import metalops_amd as mo
    for dtype, weights in (("bf16", "f32"), ("f32", ""), ("f16", "f16")):
        q, k, pos, inv, w = _inputs(dev, dtype, 37, 6, 2, 96, 24, weights=weights)
        q, k = q.clone(), k.clone()
        want = mo.qk_norm_rope(q, k, pos, inv, *w)
        _check(want[0], q, w[0], pos, inv, (24,), 1e-6, False)

        def same(got):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        same(mo.qk_norm_rope(q, k, pos[0], inv, *w))
        same(mo.qk_norm_rope(q, k, pos[0], inv, *w, sections=[24]))
        same(mo.qk_norm_rope(q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(1, 2).contiguous().transpose(1, 2), pos, inv, *w))
        wide = torch.zeros(37, 8, 131, dtype=q.dtype, device=dev)
        for at in (0, 1, 3, 8):
            a, b = wide.zero_()[:, :6, at:at + 96], wide[:, 6:, at:at + 96]      # what lies around them stays 0
            a.copy_(q)
            b.copy_(k)
            same(mo.qk_norm_rope(a, b, pos, inv, *w))
            got = mo.qk_norm_rope(a, b, pos, inv, *w, out=(a, b))
            assert got[0] is a and got[1] is b
            same(got)
            assert (wide[:, :, :at] == 0).all() and (wide[:, :, at + 96:] == 0).all()
        many = torch.zeros(37, 3, dtype=torch.int32, device=dev)
        many[:, 1] = pos[0]
        same(mo.qk_norm_rope(q, k, many[:, 1], inv, *w))
        freq = torch.zeros(25, device=dev)
        freq[1:] = inv
        same(mo.qk_norm_rope(q, k, pos, freq[1:], *w))
        one = mo.qk_norm_rope(q[5:6], k[5:6], pos[:, 5:6], inv, *w)
        assert torch.equal(one[0], want[0][5:6]) and torch.equal(one[1], want[1][5:6])
    empty = mo.qk_norm_rope(q[:0], k[:0], pos[:, :0], inv)
    assert empty[0].shape == (0, 6, 96) and empty[1].shape == (0, 2, 96)


def test_norm_of_one_side(dev):
    import metalops_amd as mo
    q, k, pos, inv, w = _inputs(dev, "f32", 20, 3, 2, 64, 32, weights="bf16")
    for qw, kw in ((w[0], None), (None, w[1])):
        oq, ok = mo.qk_norm_rope(q, k, pos, inv, qw, kw)
        _check(oq, q, qw, pos, inv, (32,), 1e-6, False)
        _check(ok, k, kw, pos, inv, (32,), 1e-6, False)


def test_far_and_negative_positions(dev):
    """Angles of any int32 position are those of fp64."""
    import metalops_amd as mo
    q, k, _, inv, _ = _inputs(dev, "f32", 6, 2, 1, 64, 32)
    pos = torch.tensor([0, 1, -1, 1 << 20, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32, device=dev)
    oq, ok = mo.qk_norm_rope(q, k, pos, inv)
    _check(oq, q, None, pos[None], inv, (32,), 1e-6, False)
    _check(ok, k, None, pos[None], inv, (32,), 1e-6, False)


def test_extremes_stay_in_their_head(dev):
    """Heads of zeros, of tiny and large values, with infinities and NaN: the others are as without them."""
    import metalops_amd as mo
    q, k, pos, inv, w = _inputs(dev, "f32", 9, 8, 2, 128, 64, weights="f32")
    q = q.clone()
    clean = mo.qk_norm_rope(q, k, pos, inv, *w)
    q[2, 1] = 0
    q[2, 2] *= 1e-25
    q[2, 3] *= 1e15
    q[4, 5, 7] = float("inf")
    q[4, 6, 100] = float("nan")
    got = mo.qk_norm_rope(q, k, pos, inv, *w)
    assert torch.equal(got[1], clean[1])
    keep = torch.ones(9, 8, dtype=torch.bool)
    for t, h in ((2, 1), (2, 2), (2, 3), (4, 5), (4, 6)):
        keep[t, h] = False
    assert torch.equal(got[0][keep], clean[0][keep])
    assert (got[0][2, 1] == 0).all()
    _check(got[0][2:3, 2:4], q[2:3, 2:4], w[0], pos[:, 2:3], inv, (64,), 1e-6, False)
    assert got[0][4, 6].isnan().all()


def test_graph_and_streams(dev):
    import metalops_amd as mo
    q, k, pos, inv, w = _inputs(dev, "bf16", 33, 32, 8, 128, 64, weights="bf16")
    want = mo.qk_norm_rope(q, k, pos, inv, *w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mo.qk_norm_rope(q, k, pos, inv, *w)
    side = torch.cuda.Stream()
    for _ in range(3):
        out[0].zero_()
        out[1].zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = mo.qk_norm_rope(q, k, pos, inv, *w)
        g.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(out, beside, want):
            assert torch.equal(a, c) and torch.equal(b, c)
