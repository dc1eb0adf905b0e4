"""Every kernel of the MXFP4 products and every split of K, each forced, against the 64-bit oracle.

The bounds are those of test_gpu_mxfp4: the output's rounding and K roundings of the sum of
magnitudes in fp32 (a split adds its partial sums in fp32 too).
"""
import pytest
import torch

from oracle import mx_ref as ref
from test_gpu_mxfp4 import DT, _bound, _check, _np, _rng, _values

pytestmark = pytest.mark.gpu

# K: one block, every remainder of four blocks, of eight and of sixteen; rows and columns around a tile's.
SHAPES = [(1, 32, 1), (5, 64, 40), (8, 2208, 100), (16, 1344, 70), (9, 4608, 33), (33, 96, 129), (64, 128, 256), (65, 160, 257), (130, 544, 300), (257, 288, 513),
          (300, 1024, 264), (70, 2080, 130), (256, 1184, 512), (3, 4448, 60)]


@pytest.mark.parametrize("split", ["1", "2", "5"])
@pytest.mark.parametrize("path", ["0", "1", "2", "3", "4", "5", "6", "7"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_each_kernel(dev, monkeypatch, M, K, N, path, split):
    import metalops_amd as mo
    print(f"mxfp4 path {path} split {split} {M}x{K}x{N}", flush=True)
    monkeypatch.setenv("MCQ4_MX_PATH", path)
    monkeypatch.setenv("MCQ4_MX_SPLIT", split)
    rng = _rng(M, K, N)
    p, s = ref.quantize_mxfp4(_values(rng, N, K, spread=0.7) * 0.02)
    w = ref.dequantize_mxfp4(p, s)
    x = torch.from_numpy(rng.normal(size=(M, K)))
    # Scale bytes at every alignment, rows of X wider than K with NaN behind them.
    odd = int(split)
    scales = torch.cat([torch.full((odd,), 255, dtype=torch.uint8), torch.from_numpy(s).reshape(-1)]).to(dev)[odd:].reshape(s.shape)
    packed = torch.from_numpy(p).to(dev)
    for dt in ("f16", "bf16", "f32"):
        xx = x.to(DT[dt])
        wide = torch.cat([xx, torch.full((M, 8), float("nan"), dtype=DT[dt])], 1).to(dev)[:, :K]
        Y = mo.matmul_mxfp4(wide, packed, scales)
        _check(Y, *_bound(_np(xx), w, dt))
    xp, xs = ref.quantize_mxfp4(_values(rng, M, K, spread=0.7))
    xv = ref.dequantize_mxfp4(xp, xs)
    xs = torch.cat([torch.full((3,), 255, dtype=torch.uint8), torch.from_numpy(xs).reshape(-1)]).to(dev)[3:].reshape(xs.shape)
    for dt in ("f16", "bf16", "f32"):
        Z = mo.matmul_mxfp4_mxfp4(torch.from_numpy(xp).to(dev), xs, packed, scales, DT[dt])
        _check(Z, *_bound(xv, w, dt))


@pytest.mark.parametrize("path", ["0", "1", "2", "3", "4", "5", "6", "7"])
def test_not_finite_in_each_kernel(dev, monkeypatch, path):
    """NaN scales and infinities stay in their row and column, also beside a ragged end of K."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_MX_PATH", path)
    M, K, N = 70, 416, 140
    rng = _rng(path, "nan")
    x = torch.from_numpy(rng.normal(size=(M, K)))
    p, s = (torch.from_numpy(t) for t in ref.quantize_mxfp4(rng.normal(size=(N, K))))
    s[1:, 0] = torch.where(torch.arange(N - 1) % 3 == 0, 255, s[1:, 0])        # the byte behind the row before
    x[M // 2, 40] = float("inf")
    w = torch.from_numpy(ref.dequantize_mxfp4(p.numpy(), s.numpy()))
    want = x @ w.T
    for dt in ("f16", "bf16", "f32"):
        Y = mo.matmul_mxfp4(x.to(DT[dt]).to(dev), p.to(dev), s.to(dev)).cpu()
        assert torch.equal(Y.isfinite(), want.isfinite()) and torch.equal(Y.isnan(), want.isnan()), dt
    xp, xs = mo.quantize_mxfp4(x.float().to(dev))
    Z = mo.matmul_mxfp4_mxfp4(xp, xs, p.to(dev), s.to(dev)).cpu()
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[M // 2], bad[:, 1:] = True, (torch.arange(N - 1) % 3 == 0) | bad[:, 1:]
    bad[M // 2] = True
    assert torch.equal(Z.isnan(), bad)


@pytest.mark.parametrize("path", ["0", "1", "2", "3", "4", "5", "6", "7"])
def test_output_rows_that_are_not_aligned(dev, monkeypatch, path):
    """The C call writes Y with any leading dimension at any element."""
    from metalops_amd import _lib
    monkeypatch.setenv("MCQ4_MX_PATH", path)
    monkeypatch.setenv("MCQ4_MX_SPLIT", "1")
    M, K, N = 67, 256, 200
    rng = _rng(path, "ldy")
    x = torch.from_numpy(rng.normal(size=(M, K))).half()
    p, s = ref.quantize_mxfp4(rng.normal(size=(N, K)))
    y, bound = _bound(_np(x), ref.dequantize_mxfp4(p, s), "f16")
    xg, pg, sg = x.to(dev), torch.from_numpy(p).to(dev), torch.from_numpy(s).to(dev)
    for ldy, first in ((N, 0), (N + 1, 1), (N + 8, 8), (N + 6, 3)):
        out = torch.full((M * ldy + first,), 7.0, dtype=torch.float16, device=dev)
        st = _lib.lib.mcq4_matmul_mxfp4(xg.data_ptr(), _lib.MCQ4_DTYPE_F16, K, pg.data_ptr(), sg.data_ptr(), out.data_ptr() + 2 * first,
                                        ldy, M, K, N, None, 0, torch.cuda.current_stream(dev).cuda_stream)
        assert st == 0
        got = out[first:].reshape(M, ldy)
        _check(got[:, :N], y, bound)
        assert (got[:, N:] == 7).all() and (out[:first] == 7).all()
