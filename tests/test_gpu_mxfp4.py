"""MXFP4 conversions and products on the GPU against the 64-bit oracle.

Conversions are compared bit for bit.  A product may be off by the output's own rounding (half a
step, eps / 2 of the value, or half the smallest subnormal), and by what fp32 sums in any order can
lose: K roundings of 2^-24 of the sum of magnitudes.
"""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _rng(*key):
    return np.random.default_rng(sum(map(ord, str(key))))


def _values(rng, *shape, spread=3.0):
    """Normal values whose blocks are of very different sizes."""
    x = rng.normal(size=shape)
    s = np.exp(rng.normal(size=(*shape[:-1], -(-shape[-1] // 32))) * spread)
    return x * np.repeat(s, 32, -1)[..., :shape[-1]]


def _np(t):
    return t.detach().cpu().double().numpy()


def _layouts(x, layout):
    """The matrix x [R, K] on the GPU in a layout; the values stay."""
    R, K = x.shape
    if layout == "rows":
        return x.contiguous()
    if layout == "cols":
        return x.t().contiguous().t()
    if layout == "padded":
        return torch.cat([x, x[:, :8]], 1)[:, :K]
    if layout == "shifted":                       # rows at addresses that are no multiple of 16 bytes
        return torch.cat([x[:, :1], x, x[:, :2]], 1)[:, 1:K + 1]
    if layout == "strided":
        out = torch.zeros(R, 2 * K, dtype=x.dtype, device=x.device)
        out[:, ::2] = x
        return out[:, ::2]
    return x[:1].expand(R, K)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["rows", "cols", "padded", "shifted", "strided", "same"])
@pytest.mark.parametrize("R,K", [(1, 32), (3, 64), (65, 288), (130, 4096), (1, 14336)])
def test_quantize(dev, dtype, layout, R, K):
    import metalops_amd as mo
    print(f"quantize {dtype} {layout} {R}x{K}", flush=True)
    x = torch.from_numpy(_values(_rng(R, K, dtype), R, K, spread=1.0)).to(DT[dtype]).to(dev)
    x = _layouts(x, layout)
    packed, scales = mo.quantize_mxfp4(x)
    rp, rs = ref.quantize_mxfp4(_np(x))
    np.testing.assert_array_equal(scales.cpu().numpy(), rs)
    np.testing.assert_array_equal(packed.cpu().numpy(), rp)


def test_quantize_borders(dev):
    """Ties, values beyond 6, signs of zero, the largest and smallest scales, infinities and NaN."""
    import metalops_amd as mo
    half = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = np.concatenate([half, np.nextafter(half.astype(np.float32), 0), np.nextafter(half.astype(np.float32), 9), [4.0, 7.99, 6.5, -0.0, 0.0]])
    block = np.zeros(32)
    block[:len(near)] = near
    rows = [np.ldexp(block * s, e) for e in (0, -100, 100, -123, 124, -126) for s in (1, -1)]
    rows += [np.zeros(32), -np.zeros(32), np.full(32, 1e-45), np.full(32, 3.4e38)]
    for bad in (np.nan, np.inf, -np.inf):
        rows.append(np.where(np.arange(32) == 7, bad, block))
    x = np.array(rows, dtype=np.float32)
    packed, scales = mo.quantize_mxfp4(torch.from_numpy(x).to(dev))
    rp, rs = ref.quantize_mxfp4(x)
    np.testing.assert_array_equal(scales.cpu().numpy(), rs)
    np.testing.assert_array_equal(packed.cpu().numpy(), rp)
    # The same through 3 dimensions and the strided kernel.
    p3, s3 = mo.quantize_mxfp4(torch.from_numpy(x).to(dev).reshape(1, *x.shape).transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(p3[0], packed) and torch.equal(s3[0], scales)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_dequantize_every_code_and_scale(dev, dtype):
    import metalops_amd as mo
    codes = np.arange(256, dtype=np.uint8).reshape(16, 16)            # every byte: 16 blocks
    lo, hi = {"f32": (1, 252), "bf16": (1, 252), "f16": (0, 252)}[dtype]   # fp32 and bf16: normal results
    byte = np.arange(lo, hi + 1, dtype=np.uint8)
    packed = np.broadcast_to(codes.reshape(1, 256), (len(byte), 256)).copy()
    scales = np.broadcast_to(byte[:, None], (len(byte), 16)).copy()
    y = mo.dequantize_mxfp4(torch.from_numpy(packed).to(dev), torch.from_numpy(scales).to(dev), DT[dtype])
    assert y.dtype == DT[dtype]
    want = torch.from_numpy(ref.dequantize_mxfp4(packed, scales)).to(DT[dtype])
    if dtype != "f16":
        want = torch.where(want.abs() < 2.0 ** -126, torch.zeros_like(want), want)
        y = torch.where(y.abs() < 2.0 ** -126, torch.zeros_like(y), y)
    assert torch.equal(y.cpu(), want)
    nan = mo.dequantize_mxfp4(torch.from_numpy(packed[:1]).to(dev), torch.full((1, 16), 255, dtype=torch.uint8, device=dev), DT[dtype])
    assert nan.isnan().all()


@pytest.mark.parametrize("R,K", [(1, 32), (7, 96), (33, 4128)])
def test_dequantize_sizes_and_views(dev, R, K):
    import metalops_amd as mo
    p, s = (torch.from_numpy(t).to(dev) for t in ref.quantize_mxfp4(_values(_rng(R, K), R, K)))
    want = ref.dequantize_mxfp4(p.cpu().numpy(), s.cpu().numpy())
    np.testing.assert_array_equal(_np(mo.dequantize_mxfp4(p, s, torch.float64)), want)
    shifted = torch.cat([p.new_zeros(1), p.reshape(-1)])[1:].reshape(R, K // 2)
    np.testing.assert_array_equal(_np(mo.dequantize_mxfp4(shifted, s.t().contiguous().t(), torch.float32)), want)


def _bound(x, w, dt):
    """Largest permitted error of x @ w.T in dt: the definition's value and its bound."""
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    t = DT[dt]
    own = np.abs(y) * torch.finfo(t).eps / 2 + (2.0 ** -25 if dt == "f16" else 0)
    # A sum rounded to the output's type: the sum's own error moves the value that is rounded.
    return y, own + (x.shape[1] + 4) * 2.0 ** -24 * mag * (1 + torch.finfo(t).eps)


def _check(Y, y, bound):
    assert Y.shape == y.shape
    err = np.abs(_np(Y) - y)
    assert (err <= bound).all(), f"worst {np.nanmax(err / bound)} of the bound"


SHAPES = [(1, 32, 1), (1, 4096, 4096), (3, 96, 17), (16, 14336, 272), (17, 1056, 1001), (33, 4128, 130), (64, 512, 1024),
          (77, 4128, 1001), (130, 288, 520), (200, 11008, 264), (257, 1024, 1000), (520, 640, 2056)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_matmul(dev, dtype, M, K, N):
    import metalops_amd as mo
    print(f"mxfp4 matmul {dtype} {M}x{K}x{N}", flush=True)
    rng = _rng(M, K, N, dtype)
    x = torch.from_numpy(rng.normal(size=(M, K))).to(DT[dtype])
    p, s = ref.quantize_mxfp4(_values(rng, N, K, spread=0.7) * 0.02)
    Y = mo.matmul_mxfp4(x.to(dev), torch.from_numpy(p).to(dev), torch.from_numpy(s).to(dev))
    assert Y.dtype == DT[dtype]
    _check(Y, *_bound(_np(x), ref.dequantize_mxfp4(p, s), dtype))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_matmul_of_two(dev, dtype, M, K, N):
    import metalops_amd as mo
    print(f"mxfp4 x mxfp4 {dtype} {M}x{K}x{N}", flush=True)
    rng = _rng(M, K, N)
    xp, xs = ref.quantize_mxfp4(_values(rng, M, K, spread=0.7))
    p, s = ref.quantize_mxfp4(_values(rng, N, K, spread=0.7) * 0.02)
    g = [torch.from_numpy(t).to(dev) for t in (xp, xs, p, s)]
    Y = mo.matmul_mxfp4_mxfp4(*g, dtype=DT[dtype])
    assert Y.dtype == DT[dtype]
    _check(Y, *_bound(ref.dequantize_mxfp4(xp, xs), ref.dequantize_mxfp4(p, s), dtype))


@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_views_of_the_operands(dev, M):
    """Leading dimensions, strides and addresses that the kernels do not take as they are."""
    import metalops_amd as mo
    K, N = 288, 200
    rng = _rng(M)
    x = torch.from_numpy(rng.normal(size=(M, K))).half().to(dev)
    p, s = (torch.from_numpy(t).to(dev) for t in ref.quantize_mxfp4(rng.normal(size=(N, K))))
    Y = mo.matmul_mxfp4(x, p, s)
    for layout in ("cols", "padded", "shifted", "strided"):
        assert torch.equal(mo.matmul_mxfp4(_layouts(x, layout), p, s), Y), layout
    odd = torch.cat([p.new_zeros(3), p.reshape(-1)])[3:].reshape(N, K // 2)
    assert torch.equal(mo.matmul_mxfp4(x, odd, s.t().contiguous().t()), Y)
    assert torch.equal(mo.matmul_mxfp4(x.reshape(1, M, K), p, s), Y[None])
    xp, xs = mo.quantize_mxfp4(x)
    Z = mo.matmul_mxfp4_mxfp4(xp, xs, p, s)
    assert torch.equal(mo.matmul_mxfp4_mxfp4(torch.cat([xp, xp], 1)[:, :K // 2], xs, odd, s), Z)
    assert torch.equal(mo.matmul_mxfp4_mxfp4(xp[None], xs[None], p, s), Z[None])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_values_that_are_not_finite(dev, M):
    """A NaN scale or an infinity stays in its row and column."""
    import metalops_amd as mo
    K, N = 512, 320
    rng = _rng(M, "nan")
    x = torch.from_numpy(rng.normal(size=(M, K)))
    p, s = (torch.from_numpy(t) for t in ref.quantize_mxfp4(rng.normal(size=(N, K))))
    s[7, 3] = 255
    x[M - 1, 40] = float("inf")
    col, row = np.zeros((M, N), dtype=bool), np.zeros((M, N), dtype=bool)
    col[:, 7], row[M - 1, :] = True, True
    w = torch.from_numpy(ref.dequantize_mxfp4(p.numpy(), s.numpy()))
    for dt in ("f16", "bf16", "f32"):
        Y = mo.matmul_mxfp4(x.to(DT[dt]).to(dev), p.to(dev), s.to(dev)).cpu()
        want = x @ w.T
        assert Y.isnan().numpy()[col].all()
        assert torch.equal(Y.isfinite(), want.isfinite()) and torch.equal(Y.isnan(), want.isnan()), dt
    xp, xs = mo.quantize_mxfp4(x.float().to(dev))
    Z = mo.matmul_mxfp4_mxfp4(xp, xs, p.to(dev), s.to(dev)).cpu()
    assert np.array_equal(Z.isnan().numpy(), col | row)


def test_wide_ranges(dev):
    """bf16 and fp32 keep weights whose scales fp16 could not hold."""
    import metalops_amd as mo
    K, N = 256, 64
    rng = _rng("wide")
    for M in (2, 100):
        p, s = ref.quantize_mxfp4(rng.normal(size=(N, K)) * 2.0 ** 60)
        x = torch.from_numpy(rng.normal(size=(M, K)) * 2.0 ** -70)
        for dt in ("bf16", "f32"):
            xx = x.to(DT[dt])
            Y = mo.matmul_mxfp4(xx.to(dev), torch.from_numpy(p).to(dev), torch.from_numpy(s).to(dev))
            _check(Y, *_bound(_np(xx), ref.dequantize_mxfp4(p, s), dt))


def test_empty(dev):
    import metalops_amd as mo
    u8 = dict(dtype=torch.uint8, device=dev)
    assert mo.quantize_mxfp4(torch.zeros(0, 64, device=dev))[0].shape == (0, 32)
    assert mo.quantize_mxfp4(torch.zeros(3, 0, device=dev))[1].shape == (3, 0)
    assert mo.dequantize_mxfp4(torch.zeros(0, 32, **u8), torch.zeros(0, 2, **u8)).shape == (0, 64)
    w = torch.zeros(5, 32, **u8), torch.zeros(5, 2, **u8)
    assert mo.matmul_mxfp4(torch.zeros(0, 64, device=dev), *w).shape == (0, 5)
    e = torch.zeros(5, 0, **u8), torch.zeros(5, 0, **u8)
    assert not mo.matmul_mxfp4(torch.ones(2, 0, device=dev), *e).any()
    assert not mo.matmul_mxfp4_mxfp4(torch.zeros(2, 0, **u8), torch.zeros(2, 0, **u8), *e).any()


@pytest.mark.parametrize("M", [1, 300])
def test_streams_and_graphs(dev, M):
    """Calls on another stream, and a graph that is replayed between eager calls."""
    import metalops_amd as mo
    K, N = 4096, 520
    rng = _rng(M, "graph")
    p, s = (torch.from_numpy(t).to(dev) for t in ref.quantize_mxfp4(rng.normal(size=(N, K))))
    xs = [torch.from_numpy(rng.normal(size=(M, K))).half().to(dev) for _ in range(4)]

    def step(x):
        return mo.matmul_mxfp4(x, p, s), mo.matmul_mxfp4_mxfp4(*mo.quantize_mxfp4(x), p, s)

    want = [step(x) for x in xs]
    static = xs[0].clone()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = [step(x) for x in xs]
    torch.cuda.current_stream(dev).wait_stream(side)
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in (1, 2, 3, 1):
        static.copy_(xs[i])
        graph.replay()
        eager = step(xs[(i + 1) % 4])
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want[i]))
        assert all(torch.equal(u, v) for u, v in zip(eager, want[(i + 1) % 4]))
