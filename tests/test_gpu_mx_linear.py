"""linear_mxfp4 on the GPU against the 64-bit oracle.

The product's sums may lose K roundings of 2^-24 of the sum of magnitudes; the bias adds one.  An
activation rounds its argument on the way, by 2^-22 of it at most, passes that and the error of the sums
on times 1.13 at most (its largest slope), and is off by 2^-21 of its own value (an exponential or erfc, a
quotient and a product, eight roundings of 2^-24).  The product with ``multiply`` and the sum with
``residual`` add a rounding of 2^-24 each, and the result its own: half a step, or half the smallest subnormal.
"""
import math

import numpy as np
import pytest
import torch

from oracle import mx_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def _act(x, name):
    if name is None:
        return x
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * torch.special.erfc(-x / math.sqrt(2))
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


class Case:
    def __init__(self, dev, dtype, M, K, N, bias="", mul=False, res=False, seed=0):
        g = torch.Generator().manual_seed(1000 * seed + M + K + N)
        dt = DT[dtype]
        self.X = (torch.randn(M, K, generator=g) * (1 + 7 * (torch.rand(K, generator=g) < 0.02))).to(dt).to(dev)
        w = (torch.randn(N, K, generator=g) * 0.05).numpy()
        p, s = ref.quantize_mxfp4(w)
        self.W = torch.from_numpy(p).to(dev), torch.from_numpy(s).to(dev)
        self.w = torch.from_numpy(np.asarray(ref.dequantize_mxfp4(p, s), dtype=np.float64)).to(dev)
        self.bias = torch.randn(N, generator=g).to(DT[bias]).to(dev) if bias else None
        self.mul = torch.randn(M, N, generator=g).to(dt).to(dev) if mul else None
        self.res = (3 * torch.randn(M, N, generator=g)).to(dt).to(dev) if res else None

    def check(self, Y, act):
        x = self.X.double()
        v = x @ self.w.t()
        K, dt = x.shape[1], self.X.dtype
        off = (K + 2) * 2.0 ** -24 * (x.abs() @ self.w.abs().t())
        if self.bias is not None:
            v = v + self.bias.double()
            off = off + 2.0 ** -24 * v.abs()
        a = _act(v, act)
        if act not in (None, "relu"):
            off = 1.13 * (off + 2.0 ** -22 * v.abs()) + 2.0 ** -21 * a.abs()
        if self.mul is not None:
            a = a * self.mul.double()
            off = off * self.mul.double().abs() + 2.0 ** -24 * a.abs()
        if self.res is not None:
            a = a + self.res.double()
            off = off + 2.0 ** -24 * a.abs()
        f = torch.finfo(dt)
        off = off + f.eps / 2 * (a.abs() + off) + f.smallest_normal * f.eps / 2
        assert Y.dtype == dt and tuple(Y.shape) == tuple(a.shape)
        wrong = ((Y.double() - a).abs() > off).nonzero()
        assert len(wrong) == 0, (len(wrong), wrong[0].tolist(), Y[tuple(wrong[0])].item(), a[tuple(wrong[0])].item())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,K,N", [(1, 32, 1), (1, 4096, 4096), (3, 96, 70), (17, 4128, 1001), (64, 14336, 512), (200, 1024, 776), (1100, 512, 1030)])
def test_all_operands(dev, dtype, M, K, N):
    import metalops_amd as mo
    for i, act in enumerate(ACTS):
        print(f"linear {dtype} {M}x{K}x{N} {act}", flush=True)
        c = Case(dev, dtype, M, K, N, bias=(dtype, "f32")[i % 2], mul=True, res=True, seed=i)
        c.check(mo.linear_mxfp4(c.X, *c.W, bias=c.bias, activation=act, multiply=c.mul, residual=c.res), act)


@pytest.mark.parametrize("bias,mul,res", [("", False, False), ("f16", False, False), ("", True, False), ("", False, True)])
def test_operands_left_out(dev, bias, mul, res):
    import metalops_amd as mo
    for M in (1, 40, 600):
        c = Case(dev, "f16", M, 512, 392, bias=bias, mul=mul, res=res)
        Y = mo.linear_mxfp4(c.X, *c.W, c.bias, None, c.mul, c.res)
        c.check(Y, None)
        if not (bias or mul or res):
            assert torch.equal(Y, mo.matmul_mxfp4(c.X, *c.W))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("path", range(8))
@pytest.mark.parametrize("split", [1, 3])
def test_every_kernel(dev, dtype, path, split, monkeypatch):
    """Each kernel of the product, with and without a split of K, whole tiles and parts of tiles."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_MX_PATH", str(path))
    monkeypatch.setenv("MCQ4_MX_SPLIT", str(split))
    for M, N in ((5, 40), (16, 64), (150, 333), (256, 512)):
        print(f"linear path {path} split {split} {dtype} {M}x{N}", flush=True)
        c = Case(dev, dtype, M, 1056, N, bias="f32", mul=True, res=True)
        c.check(mo.linear_mxfp4(c.X, *c.W, c.bias, "silu", c.mul, c.res), "silu")


def test_layouts(dev):
    """Leading dimensions, rows of other strides and alignments, transposed and broadcast operands."""
    import metalops_amd as mo
    c = Case(dev, "bf16", 24, 256, 104, bias="bf16", mul=True, res=True)
    want = mo.linear_mxfp4(c.X, *c.W, c.bias, "gelu", c.mul, c.res)
    c.check(want, "gelu")
    got = mo.linear_mxfp4(c.X.view(2, 3, 4, 256), *c.W, c.bias, "gelu", c.mul.view(2, 3, 4, 104), c.res.view(2, 3, 4, 104))
    assert got.shape == (2, 3, 4, 104) and torch.equal(got.view(24, 104), want)
    wide = torch.randn(24, 301, device=dev).bfloat16()
    for at in (0, 1, 5, 8):
        mul, res = wide[:, at:at + 104], wide[:, 150 + at:254 + at]
        mul.copy_(c.mul)
        res.copy_(c.res)
        assert torch.equal(mo.linear_mxfp4(c.X, *c.W, c.bias, "gelu", mul, res), want)
    assert torch.equal(mo.linear_mxfp4(c.X, *c.W, c.bias, "gelu", c.mul.t().contiguous().t(), c.res.t().contiguous().t()), want)
    bias = torch.zeros(2 * 104, dtype=torch.bfloat16, device=dev)
    bias[::2] = c.bias
    assert torch.equal(mo.linear_mxfp4(c.X, *c.W, bias[::2], "gelu", c.mul, c.res), want)
    row = c.res[:1].expand(24, 104)
    assert torch.equal(mo.linear_mxfp4(c.X, *c.W, residual=row), mo.linear_mxfp4(c.X, *c.W, residual=row.contiguous()))
    one = mo.linear_mxfp4(c.X[3], *c.W, c.bias, "gelu", c.mul[3], c.res[3])
    assert one.shape == (104,)
    for shape in ((0, 256), (2, 0, 256)):
        assert mo.linear_mxfp4(torch.zeros(shape, device=dev).half(), *c.W, residual=torch.zeros(*shape[:-1], 104, device=dev).half()).numel() == 0


def test_infinities_and_nan(dev):
    """What the formulas give of them, row by row: no other row is touched."""
    import metalops_amd as mo
    inf, nan = math.inf, math.nan
    v = torch.tensor([0.0, -0.0, 1e4, -1e4, inf, -inf, nan, 2.0], device=dev)
    for M in (1, 40):
        c = Case(dev, "f32", M, 64, 8, res=True)
        c.X.zero_()
        for act in ACTS:
            Y = mo.linear_mxfp4(c.X, *c.W, bias=v, activation=act)
            want = _act(v.double(), act).float().expand(M, 8)
            torch.testing.assert_close(Y, want, rtol=1e-6, atol=0, equal_nan=True)
        Y = mo.linear_mxfp4(c.X, *c.W, residual=torch.full_like(c.res, nan))
        assert Y.isnan().all()
        mul = torch.zeros_like(c.res)
        mul[:, 3] = inf
        Y = mo.linear_mxfp4(c.X, *c.W, bias=torch.ones(8, device=dev), multiply=mul)
        assert (Y[:, 3] == inf).all() and (Y[:, :3] == 0).all() and (Y[:, 4:] == 0).all()


def test_in_place_at_the_c_call(dev):
    """Y may be the residual (or the factor) itself."""
    import ctypes

    import metalops_amd as mo
    from metalops_amd import _lib
    for M, K, N in ((1, 512, 256), (20, 4096, 512), (700, 512, 1024), (64, 14336, 512)):
        c = Case(dev, "f16", M, K, N, bias="f16", res=True)
        want = mo.linear_mxfp4(c.X, *c.W, c.bias, "silu", None, c.res)
        Y = c.res.clone()
        e = _lib.EpilogueStruct(c.bias.data_ptr(), None, Y.data_ptr(), N, N, 1, 2)
        need = _lib.lib.mcq4_matmul_mxfp4_workspace_bytes(M, K, N, 1)
        ws = torch.zeros(max(need, 1), dtype=torch.uint8, device=dev)
        st = _lib.lib.mcq4_linear_mxfp4(c.X.data_ptr(), 1, K, c.W[0].data_ptr(), c.W[1].data_ptr(), ctypes.byref(e), Y.data_ptr(), N, M, K, N,
                                        ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream)
        assert st == 0
        assert torch.equal(Y, want)


def test_graph_and_streams(dev):
    """Captured calls (with K split, whose workspace is the graph's own) replayed among eager ones on two streams."""
    import metalops_amd as mo
    cases = [Case(dev, "bf16", M, K, N, bias="f32", mul=True, res=True) for M, K, N in ((1, 4096, 512), (16, 14336, 512), (96, 4096, 512))]

    def call(c):
        return mo.linear_mxfp4(c.X, *c.W, c.bias, "gelu_tanh", c.mul, c.res)
    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = [call(c) for c in cases]
    side = torch.cuda.Stream()
    for _ in range(4):
        for o in out:
            o.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = [call(c) for c in cases]
        g.replay()
        eager = [call(c) for c in cases]
        torch.cuda.synchronize()
        for a, b, c, d in zip(out, beside, eager, want):
            assert torch.equal(a, d) and torch.equal(b, d) and torch.equal(c, d)
