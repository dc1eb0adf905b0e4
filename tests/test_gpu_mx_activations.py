"""The activations of linear_mxfp4 in 16 bits, by their own values: the product is 0 and the fp32 bias the argument.

Relative to the result an activation may be off by 2^-15: its exponential's argument, up to 126 to base 2, carries three
roundings of 2^-24 (2^-15.7 of the exponential), everything else less than 2^-19.  The result's own rounding is half a
step, or half the smallest subnormal; the factor's is 2^-24.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
ACTS = ["relu", "silu", "gelu", "gelu_tanh"]


def _act(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * torch.special.erfc(-x / math.sqrt(2))
    return x / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))      # 1 + tanh u = 2 / (1 + e^-2u)


def _zero(dev, dtype, M, N, K=64):
    """X and a weight whose product is 0."""
    g = torch.Generator().manual_seed(N)
    packed = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8).to(dev)
    scales = torch.full((N, K // 32), 127, dtype=torch.uint8, device=dev)
    return torch.zeros(M, K, dtype=DT[dtype], device=dev), packed, scales


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 40, 300])
def test_values(dev, dtype, act, M):
    import metalops_amd as mo
    low = {"gelu": -13.0, "gelu_tanh": -9.7}.get(act, -80.0)
    v = torch.cat([torch.linspace(low, 14, 3001), torch.linspace(-5.5, -2, 1000), torch.logspace(-6, 0, 200), -torch.logspace(-6, 0, 199)]).to(dev)
    N = len(v)
    print(f"{act} {dtype} {M} x {N}", flush=True)
    X, packed, scales = _zero(dev, dtype, M, N)
    want = _act(v.double(), act)
    f = torch.finfo(DT[dtype])
    for factor in (None, 1000.0, 2.0 ** 14):         # the tail's results among a type's ordinary ones
        mul = None if factor is None else torch.full((M, N), factor, dtype=DT[dtype], device=dev)
        Y = mo.linear_mxfp4(X, packed, scales, bias=v, activation=act, multiply=mul)
        w = want * (factor or 1)
        near = w.abs() < f.max / 2
        off = 2.0 ** -15 * w.abs() + 2.0 ** -122
        off = off + f.eps / 2 * (w.abs() + off) + f.smallest_normal * f.eps / 2
        wrong = (((Y.double() - w).abs() > off) & near).nonzero()
        assert len(wrong) == 0, (factor, len(wrong), v[wrong[0][1]].item(), Y[tuple(wrong[0])].item(), w[wrong[0][1]].item())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_infinities_and_nan(dev, dtype, M):
    """What the formulas give of them, in the kernels' own forms for 16 bits; no other column is touched."""
    import metalops_amd as mo
    inf, nan = math.inf, math.nan
    v = torch.tensor([0.0, -0.0, 1e4, -1e4, inf, -inf, nan, 2.0], device=dev)
    X, packed, scales = _zero(dev, dtype, M, 8)
    for act in [None] + ACTS:
        Y = mo.linear_mxfp4(X, packed, scales, bias=v, activation=act)
        want = (v if act is None else _act(v.double(), act)).to(DT[dtype]).expand(M, 8)
        torch.testing.assert_close(Y, want, rtol=torch.finfo(DT[dtype]).eps, atol=0, equal_nan=True)
    # Finite values whose squares and cubes are not.
    far = torch.tensor([3e38, -3e38, 1e25, -1e25, 1e13, -1e13, 200.0, -200.0], device=dev)
    for act in ACTS:
        Y = mo.linear_mxfp4(X, packed, scales, bias=far, activation=act)
        want = torch.where(far > 0, far, torch.zeros_like(far)).to(DT[dtype]).expand(M, 8)
        torch.testing.assert_close(Y, want, rtol=torch.finfo(DT[dtype]).eps, atol=0)
    for operand in ("multiply", "residual"):
        t = torch.zeros(M, 8, dtype=DT[dtype], device=dev)
        t[:, 3], t[:, 5] = inf, nan
        Y = mo.linear_mxfp4(X, packed, scales, bias=torch.ones(8, device=dev), activation="silu", **{operand: t})
        assert (Y[:, 3] == inf).all() and Y[:, 5].isnan().all() and Y[:, [0, 1, 2, 4, 6, 7]].isfinite().all()
