"""The oracle of the microscaled formats against known answers, torch's own e4m3 and brute force."""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref


def test_e4m3_table_is_torchs():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ref.e4m3_decode(np.arange(256)), t)


def test_e4m3_encode_is_torchs():
    x = np.concatenate([np.random.default_rng(0).normal(size=4000) * s for s in (1e-3, 0.02, 1, 60)]).clip(-448, 448)
    half = (ref.E4M3[:126] + ref.E4M3[1:127]) / 2
    x = np.concatenate([x.astype(np.float32).astype(np.float64), half, -half, [0.0, -0.0, 448, 2.0 ** -10]])
    t = torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(ref.e4m3_encode(x), t)
    assert ref.e4m3_encode(np.array([np.nan, np.inf, -np.inf])).tolist() == [127, 127, 255]


def test_mxfp4_known_block():
    x = np.zeros(32)
    # amax 7.9: scale 1.  Ties: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4.
    x[:12] = [7.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.01, -0.2, 6.5, -0.0]
    packed, scales = ref.quantize_mxfp4(x)
    assert scales.tolist() == [127]
    assert ref.dequantize_mxfp4(packed, scales)[:12].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -6, 0, 6, 0]
    code = np.stack([packed & 15, packed >> 4], -1).reshape(-1)
    assert code[9] == 8 and code[11] == 8 and code[1] == 0
    assert packed[0] == 7 and packed[4] == 0x8F          # low nibble first


@pytest.mark.parametrize("amax,byte", [(4.0, 127), (3.999, 126), (2.0 ** -126, 0), (1e-45, 0), (0.0, 0), (3e38, 252)])
def test_mxfp4_scale(amax, byte):
    x = np.zeros(32)
    x[5] = amax
    assert ref.quantize_mxfp4(x)[1].tolist() == [byte]


def test_mxfp4_not_finite():
    x = np.ones((3, 32))
    x[0, 3], x[1, 4] = np.nan, -np.inf
    packed, scales = ref.quantize_mxfp4(x)
    assert scales[:, 0].tolist() == [255, 255, 125] and not packed[:2].any()
    assert np.isnan(ref.dequantize_mxfp4(packed, scales)[:2]).all()


def test_mxfp4_nearest_by_brute_force():
    x = np.random.default_rng(1).normal(size=(20, 32)) * np.exp(np.random.default_rng(2).normal(size=(20, 1)) * 5)
    packed, scales = ref.quantize_mxfp4(x)
    v = ref.dequantize_mxfp4(packed, scales)
    grid = np.concatenate([ref.E2M1, -ref.E2M1]) * ref.scale_value(scales)[..., None]
    best = np.abs(x[..., None] - grid).min(-1)
    np.testing.assert_allclose(np.abs(x - v), best, rtol=1e-12)


def test_kv8_scale_and_append():
    assert [ref.kv8_byte(a) for a in (448.0, 448.1, 224.0, 1.75, 1.76, 0.0)] == [127, 128, 126, 119, 120, 1]
    z = np.zeros((2, 1, 16, 16), dtype=np.uint8)
    c = ref.Cache(z, z, np.full((2, 1), 200, np.uint8), np.full((2, 1), 200, np.uint8))
    table, x = np.array([[1, 0]]), np.random.default_rng(0).normal(size=(20, 1, 16))
    c.append(0, x, table, [0], [0, 20])
    for sl, pid in ((slice(0, 16), 1), (slice(16, 20), 0)):
        assert c.bytes[0][pid, 0] == ref.kv8_byte(np.abs(x[sl]).max())
    got, here = c.values(0, table, 0, 20)
    assert here.all() and np.abs(got - x).max() <= np.abs(x).max() * 2.0 ** -4
    # A large token joins the second page: its codes are rescaled, the first page stays.
    first = c.codes[0][1].copy()
    c.append(0, np.full((1, 1, 16), 100.0), table, [20], [0, 1])
    assert c.bytes[0][0, 0] == ref.kv8_byte(100.0) and (c.codes[0][1] == first).all()
    again, _ = c.values(0, table, 0, 21)
    assert (again[20] == 104).all() or (again[20] == 96).all()
    assert np.abs(again[16:20] - x[16:20]).max() <= np.abs(x).max() * 2.0 ** -3


def test_attention_against_torch():
    g = np.random.default_rng(3)
    H, page, D, G = 2, 16, 16, 3
    c = ref.Cache(*[ref.e4m3_encode(g.normal(size=(5, H, page, D)) * 50) for _ in range(2)], *[g.integers(118, 124, (5, H)) for _ in range(2)])
    table, ctx, cu = np.array([[4, 0, 2], [1, 3, 9]]), [40, 20], [0, 3, 5]
    q = g.normal(size=(5, H * G, D))
    out, lse, _ = ref.attention(q, c, table, ctx, cu, 0.3, window=17)
    for b, n in ((0, 3), (1, 2)):
        k, v = (torch.from_numpy(c.values(w, table, b, ctx[b])[0]).repeat_interleave(G, 1).transpose(0, 1) for w in (0, 1))
        qq = torch.from_numpy(q[cu[b]:cu[b + 1]]).transpose(0, 1)
        pos, key = ctx[b] - n + torch.arange(n)[:, None], torch.arange(ctx[b])
        s = (qq @ k.transpose(1, 2) * 0.3).masked_fill((key > pos) | (key <= pos - 17), -np.inf)
        np.testing.assert_allclose(out[cu[b]:cu[b + 1]], (s.softmax(-1) @ v).transpose(0, 1).numpy(), rtol=1e-10, atol=1e-12)
        np.testing.assert_allclose(lse[cu[b]:cu[b + 1]], s.logsumexp(-1).T.numpy(), rtol=1e-10)
