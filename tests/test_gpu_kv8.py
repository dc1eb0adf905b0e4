"""The 8-bit key/value cache on the GPU against the 64-bit oracle.

Appended codes and scales are compared byte for byte, values read back bit for bit.  Attention may
be off by the output's rounding (half a step, eps / 2) and by:
  * P rounded to fp16: 2^-11 of each weight, 2^-25 where it is subnormal (weights are at most 1 and
    their sum at least 1);
  * scores in fp32: D + 4 roundings of 2^-24 of sum |q||k| scale, which move a weight by as much
    relatively, and the weights' sum too; exp2's own error of 2^-22;
  * V's codes in fp16 relative to the largest scale: 2^-25 of the largest |v|;
  * sums in fp32: one rounding of 2^-24 for each token, of the weighted sum of |v|.
"""
import numpy as np
import pytest
import torch

from oracle import mx_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _rng(*key):
    return np.random.default_rng(sum(map(ord, str(key))))


def _np(t):
    return t.detach().cpu().double().numpy()


def _cum(n):
    return [0, *np.cumsum(n).tolist()]


def _i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


class Both:
    """One cache on the GPU and in the oracle, the pages in no order, old codes in them."""

    def __init__(self, dev, rng, B, W, H, D, page, spare=2):
        import metalops_amd as mo
        P = B * W + spare
        k, v = (ref.e4m3_encode(rng.normal(size=(P, H, page, D)) * 40) for _ in range(2))
        ks, vs = (rng.integers(115, 124, (P, H)).astype(np.uint8) for _ in range(2))
        self.ref = ref.Cache(k, v, ks, vs)
        t = lambda a: torch.from_numpy(a.copy()).to(dev)
        self.gpu = mo.KV8Cache(t(k), t(v.swapaxes(2, 3)), t(ks), t(vs))
        self.table = rng.permutation(P)[:B * W].reshape(B, W).astype(np.int32)
        self.dev = dev

    def same(self):
        g = self.gpu
        torch.cuda.synchronize()
        got = (g.k_codes.cpu().numpy(), g.v_codes.cpu().numpy().swapaxes(2, 3), g.k_scales.cpu().numpy(), g.v_scales.cpu().numpy())
        for name, a, b in zip(("k", "v", "k_scales", "v_scales"), got, (*self.ref.codes, *self.ref.bytes)):
            np.testing.assert_array_equal(a, b, err_msg=name)


APPENDS = [  # new tokens, tokens before, H, D, page
    ([1], [0], 1, 16, 16),
    ([1, 1, 1], [0, 5, 31], 2, 64, 16),
    ([1] * 5, [63, 64, 65, 127, 200], 8, 128, 64),
    ([70], [3], 2, 80, 32),
    ([200, 1, 64], [0, 64, 100], 3, 128, 64),
    ([17, 300, 0, 40], [250, 0, 10, 255], 2, 256, 256),
    ([33, 33], [120, 128], 1, 96, 128),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,start,H,D,page", APPENDS)
def test_append(dev, dtype, new, start, H, D, page):
    import metalops_amd as mo
    print(f"kv8 append {dtype} {new} {start} H={H} D={D} page={page}", flush=True)
    rng = _rng(new, start, dtype)
    both = Both(dev, rng, len(new), -(-max(s + n for s, n in zip(start, new)) // page), H, D, page)
    T, cu = sum(new), _cum(new)
    table, gs = _i32(both.table, dev), _i32(start, dev)
    # Small, then larger than what is there: the second call rescales the older tokens.
    for size in (0.5, 300.0):
        x = [torch.from_numpy(rng.normal(size=(T, H, D)) * size).to(DT[dtype]) for _ in range(2)]
        for i in range(2):
            both.ref.append(i, _np(x[i]), both.table, start, cu)
        if len(set(new)) == 1 and size < 1:
            mo.kv8_append(both.gpu, x[0].to(dev), x[1].to(dev), table, gs)
        else:
            mo.kv8_append(both.gpu, x[0].to(dev), x[1].to(dev), table, gs, _i32(cu, dev))
        both.same()


def test_append_token_by_token_is_read_back(dev):
    """Forty single tokens of growing size, and the values read."""
    import metalops_amd as mo
    rng = _rng("grow")
    both = Both(dev, rng, 2, 3, 2, 64, 16)
    table = _i32(both.table, dev)
    for t in range(40):
        x = [rng.normal(size=(2, 2, 64)) * 1.2 ** t for _ in range(2)]
        x = [torch.from_numpy(a).float() for a in x]
        start = [t, max(0, t - 3)]
        for i in range(2):
            both.ref.append(i, _np(x[i]), both.table, start, [0, 1, 2])
        mo.kv8_append(both.gpu, x[0].to(dev), x[1].to(dev), table, _i32(start, dev))
    both.same()
    for dt in ("f32", "bf16", "f16"):
        got = mo.kv8_read(both.gpu, table, _i32([40, 21], dev), DT[dt])
        for i in range(2):
            want = np.zeros((2, 48, 2, 64))
            for b, L in ((0, 40), (1, 21)):
                want[b, :L] = both.ref.values(i, both.table, b, L)[0]
            w = torch.from_numpy(want).to(DT[dt])
            assert torch.equal(got[i].cpu(), w), dt


def test_append_not_finite_zero_and_views(dev):
    import metalops_amd as mo
    rng = _rng("views")
    both = Both(dev, rng, 2, 2, 3, 32, 32)
    x = torch.from_numpy(rng.normal(size=(2, 20, 3, 32))).float()
    x[0, 3, 1, 5], x[0, 4, 0, :], x[1, 7, 2, 9], x[1, 12] = float("inf"), float("nan"), -float("inf"), 0.0
    x[0, 11:] = 0.0
    cu = _i32([0, 10, 20], dev)
    for i in range(2):
        both.ref.append(i, _np(x[i]), both.table, [0, 30], [0, 10, 20])
    # Heads and tokens in another order, and rows at odd addresses.
    g = x.to(dev)
    k = g[0].transpose(0, 1).contiguous().transpose(0, 1)
    v = torch.cat([g[1].new_zeros(20, 3, 1), g[1]], 2)[:, :, 1:]
    wide = torch.cat([_i32(both.table, dev), _i32(both.table, dev)], 1)[:, :2]
    mo.kv8_append(both.gpu, k, v, wide, _i32([0, 30], dev), cu)
    got = both.gpu.k_codes[int(both.table[0, 0])].cpu().numpy()
    assert got[1, 3, 5] & 127 == 127 and (got[0, 4] & 127 == 127).all()
    # NaN's sign bit is not fixed by the definition.
    for codes in (both.gpu.k_codes, both.gpu.v_codes):
        codes[(codes & 127) == 127] = 127
    for codes in both.ref.codes:
        codes[(codes & 127) == 127] = 127
    both.same()


def test_append_skips_what_has_no_page(dev):
    """Entries that name no page, tokens past the table, offsets that make no sense."""
    import metalops_amd as mo
    rng = _rng("skip")
    both = Both(dev, rng, 3, 2, 2, 16, 16)
    both.table[1] = [-1, 10 ** 6]
    x = [torch.from_numpy(rng.normal(size=(60, 2, 16))).float() for _ in range(2)]
    for i in range(2):
        both.ref.append(i, _np(x[i]), both.table, [0, 0, 30], [0, 20, 40, 60])
    mo.kv8_append(both.gpu, x[0].to(dev), x[1].to(dev), _i32(both.table, dev), _i32([0, 0, 30], dev), _i32([0, 20, 40, 60], dev))
    both.same()
    for cu in ([0, 50, 20, 70], [-4, 0, 0, 2 ** 30]):
        mo.kv8_append(both.gpu, x[0].to(dev), x[1].to(dev), _i32(both.table, dev), _i32([100, -5, 2 ** 31 - 3], dev), _i32(cu, dev))
    both.same()


def _check(out, want, terms, L, D, dt):
    eps = torch.finfo(DT[dt]).eps
    ds = (D + 4) * 2.0 ** -24 * terms["sabs"] + 2.0 ** -21
    bound = terms["av"] * (2.0 ** -11 + 2 * ds + (L + 8) * 2.0 ** -24) + (L * 2.0 ** -25 + 2.0 ** -25) * terms["vmax"]
    bound = bound * (1 + eps) + np.abs(want) * eps / 2 + (2.0 ** -25 if dt == "f16" else 0)
    err = np.abs(_np(out) - want)
    assert (err <= bound).all(), f"worst {np.nanmax(err / np.maximum(bound, 1e-300))} of the bound"


ATTENDS = [  # new tokens, contexts, H, G, D, page, causal, window
    ([1], [1], 1, 1, 16, 16, True, 0),
    ([1], [700], 2, 4, 128, 64, True, 0),
    ([1, 1, 1, 1], [1, 63, 64, 65], 2, 8, 64, 16, True, 0),
    ([1, 1, 1], [0, 130, 5], 1, 7, 80, 32, True, 0),
    ([1, 1], [2100, 900], 1, 16, 256, 128, True, 0),
    ([3, 3], [200, 4], 2, 2, 96, 64, True, 0),
    ([5, 1, 0, 40], [5, 300, 77, 60], 2, 3, 128, 64, True, 0),
    ([20, 33], [20, 100], 2, 4, 64, 16, False, 0),
    ([1, 1], [500, 40], 2, 4, 128, 32, True, 100),
    ([30, 9], [95, 200], 1, 4, 128, 64, True, 17),
    ([12], [7], 2, 2, 64, 64, True, 0),             # more new tokens than context: the first see nothing
    ([140, 70], [300, 70], 1, 2, 128, 64, True, 0),
    ([150], [150], 1, 1, 192, 256, True, 50),
    ([130, 65], [130, 400], 1, 5, 80, 16, True, 0),
    ([100], [260], 2, 1, 256, 32, False, 0),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new,context,H,G,D,page,causal,window", ATTENDS)
def test_attention(dev, dtype, new, context, H, G, D, page, causal, window):
    import metalops_amd as mo
    print(f"kv8 attention {dtype} {new} {context} H={H} G={G} D={D} page={page} {causal} {window}", flush=True)
    rng = _rng(new, context, dtype)
    both = Both(dev, rng, len(new), -(-max(context) // page), H, D, page)
    T, cu = sum(new), _cum(new)
    q = torch.from_numpy(rng.normal(size=(T, H * G, D))).to(DT[dtype])
    want, lse, terms = ref.attention(_np(q), both.ref, both.table, context, cu, D ** -0.5, causal, window)
    gcu = None if len(set(new)) == 1 else _i32(cu, dev)
    args = q.to(dev), both.gpu, _i32(both.table, dev), _i32(context, dev)
    out, got_lse = mo.kv8_attention(*args, gcu, causal=causal, window=window, return_lse=True)
    assert out.dtype == DT[dtype] and out.shape == want.shape
    _check(out, want, terms, max(context), D, dtype)
    inf = np.isinf(lse)
    assert np.array_equal(np.isinf(_np(got_lse)), inf) and not _np(out)[inf].any()
    ds = (D + 4) * 2.0 ** -24 * terms["sabs"][..., 0] + 2.0 ** -20 + max(context) * 2.0 ** -24
    np.testing.assert_array_less(np.abs(_np(got_lse)[~inf] - lse[~inf]), (ds + np.abs(np.where(inf, 0, lse)) * 2.0 ** -22)[~inf])
    # A host bound of the contexts, tight or loose, an explicit scale, and given offsets.
    for most in (max(context), 64, 10 ** 6):
        _check(mo.kv8_attention(*args, _i32(cu, dev), D ** -0.5, causal, window, most), want, terms, max(context), D, dtype)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_views(dev, new):
    import metalops_amd as mo
    rng = _rng("view", new)
    both = Both(dev, rng, 2, 3, 2, 64, 64)
    table, ctx = _i32(both.table, dev), _i32([130, 190], dev)
    q = torch.from_numpy(rng.normal(size=(2 * new, 6, 64))).half().to(dev)
    out = mo.kv8_attention(q, both.gpu, table, ctx)
    fused = torch.cat([q, q], 1)[:, :6]                                    # as a slice of q, k and v in one
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.cat([q.new_zeros(2 * new, 6, 1), q], 2)[:, :, 1:]
    chan = q.transpose(1, 2).contiguous().transpose(1, 2)
    for name, t in (("fused", fused), ("by_head", by_head), ("odd", odd), ("chan", chan)):
        assert torch.equal(mo.kv8_attention(t, both.gpu, table, ctx), out), name
    wide = torch.cat([table, table], 1)[:, :3]
    assert torch.equal(mo.kv8_attention(q, both.gpu, wide, ctx), out)


@pytest.mark.parametrize("new,context,window", [(1, 100, 0), (1, 100, 30), (6, 100, 0), (70, 150, 0), (70, 150, 20)])
def test_masked_places_may_hold_anything(dev, new, context, window):
    """NaN codes and scales behind the context, in tokens a row does not see, and entries of the
    table that are never reached; a row that does see a NaN is NaN."""
    import metalops_amd as mo
    rng = _rng("mask", new, window)
    page, D = 64, 128
    both = Both(dev, rng, 1, 4, 1, D, page)
    q = torch.from_numpy(rng.normal(size=(new, 4, D))).half().to(dev)
    table, ctx = _i32(both.table, dev), _i32([context], dev)
    clean = mo.kv8_attention(q, both.gpu, table, ctx, window=window)
    ids = [int(i) for i in both.table[0]]
    g = both.gpu
    # Behind the context: the rest of its last page, pages after it, entries that name nothing.
    last = context // page
    g.k_codes[ids[last], :, context % page:] = 127
    g.v_codes[ids[last], :, :, context % page:] = 255
    table = table.clone()
    table[0, last + 1:] = torch.tensor([-7, 10 ** 8, 5][:table.shape[1] - last - 1], dtype=torch.int32, device=dev)
    assert torch.equal(mo.kv8_attention(q, g, table, ctx, window=window), clean)
    # Tokens only the last row sees (causal), or that the window has left behind.
    if new > 1:
        t = context - 1
        kept = g.v_codes[ids[t // page], 0, 5, t % page].clone()
        g.v_codes[ids[t // page], 0, 5, t % page] = 127
        out = mo.kv8_attention(q, g, table, ctx, window=window)
        assert torch.equal(out[:-1], clean[:-1])
        assert out[-1, :, 5].isnan().all() and torch.equal(out[-1, :, 6:], clean[-1, :, 6:])
        g.v_codes[ids[t // page], 0, 5, t % page] = kept
        kk = g.k_codes[ids[t // page], 0, t % page, 3].clone()
        g.k_codes[ids[t // page], 0, t % page, 3] = 255
        out = mo.kv8_attention(q, g, table, ctx, window=window)
        assert torch.equal(out[:-1], clean[:-1]) and out[-1].isnan().all()
        g.k_codes[ids[t // page], 0, t % page, 3] = kk
    if window:
        t = context - new - window                   # the position just before the first row's window
        g.v_codes[ids[t // page], 0, :, t % page] = 127
        g.k_codes[ids[t // page], 0, t % page] = 127
        assert torch.equal(mo.kv8_attention(q, g, table, ctx, window=window), clean)


@pytest.mark.parametrize("new", [1, 50])
def test_missing_pages_hold_nothing(dev, new):
    """An entry inside the context that names no page: its tokens are not seen."""
    import metalops_amd as mo
    rng = _rng("missing", new)
    both = Both(dev, rng, 2, 5, 2, 64, 32)
    both.table[0, 1], both.table[1, :] = -1, 10 ** 7
    context, cu = [150, 100], [0, new, 2 * new]
    q = torch.from_numpy(rng.normal(size=(2 * new, 4, 64))).half()
    want, _, terms = ref.attention(_np(q), both.ref, both.table, context, cu, 0.125)
    out = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32(context, dev))
    _check(out, want, terms, 150, 64, "f16")
    assert not out[new:].any()


def test_scales_of_very_different_pages(dev):
    """Pages whose value scales lie 2^40 apart, the large one first, last and between."""
    import metalops_amd as mo
    rng = _rng("scales")
    for new in (1, 80):
        for big in range(4):
            both = Both(dev, rng, 1, 4, 1, 64, 64)
            for i in range(4):
                b = 150 if i == big else 110
                both.ref.bytes[1][both.table[0, i]] = b
                both.gpu.v_scales[int(both.table[0, i])] = b
            q = torch.from_numpy(rng.normal(size=(new, 2, 64))).bfloat16()
            want, _, terms = ref.attention(_np(q), both.ref, both.table, [256], [0, new], 0.125)
            out = mo.kv8_attention(q.to(dev), both.gpu, _i32(both.table, dev), _i32([256], dev))
            _check(out, want, terms, 256, 64, "bf16")


def test_long_context_is_split_and_joined(dev):
    import metalops_amd as mo
    rng = _rng("long")
    B, ctx, H, G, D, page = 2, [9000, 4100], 1, 2, 64, 128
    both = Both(dev, rng, B, 71, H, D, page)
    for new in (1, 2, 33):
        q = torch.from_numpy(rng.normal(size=(B * new, H * G, D)) * 2).half()
        want, _, terms = ref.attention(_np(q), both.ref, both.table, ctx, _cum([new] * B), 0.125)
        args = q.to(dev), both.gpu, _i32(both.table, dev), _i32(ctx, dev)
        out = mo.kv8_attention(*args)
        _check(out, want, terms, 9000, D, "f16")
        assert torch.equal(out, mo.kv8_attention(*args))          # the same order of sums every time


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^32 bytes, its last pages in use."""
    import metalops_amd as mo
    H, D, page = 8, 128, 64
    P = (1 << 32) // (H * D * page) + 40
    cache = mo.KV8Cache.empty(P, H, D, page, dev)
    rng = _rng("far")
    table = np.array([[P - 1, 0, P - 17]])
    x = [torch.from_numpy(rng.normal(size=(150, H, D))).half() for _ in range(2)]
    mo.kv8_append(cache, x[0].to(dev), x[1].to(dev), _i32(table, dev), _i32([0], dev))
    k, v = mo.kv8_read(cache, _i32(table, dev), _i32([150], dev))
    small = ref.Cache(*[np.zeros((3, H, page, D), np.uint8)] * 2, *[np.zeros((3, H), np.uint8)] * 2)
    st = np.array([[0, 1, 2]])
    for i in range(2):
        small.append(i, _np(x[i]), st, [0], [0, 150])
        np.testing.assert_array_equal(_np((k, v)[i])[0, :150], small.values(i, st, 0, 150)[0])
    for new in (1, 70):
        q = torch.from_numpy(rng.normal(size=(new, H, D))).half()
        want, _, terms = ref.attention(_np(q), small, st, [150], [0, new], D ** -0.5)
        _check(mo.kv8_attention(q.to(dev), cache, _i32(table, dev), _i32([150], dev)), want, terms, 150, D, "f16")


@pytest.mark.parametrize("new", [1, 64])
def test_streams_and_graphs(dev, new):
    """A decode step on another stream and in a graph whose lengths change between replays."""
    import metalops_amd as mo
    rng = _rng("graph", new)
    H, G, D, page, B = 2, 4, 128, 64, 2
    both = [Both(dev, _rng("same"), B, 40, H, D, page) for _ in range(2)]
    table = _i32(both[0].table, dev)
    x = [torch.from_numpy(rng.normal(size=(B * new, n, D))).half().to(dev) for n in (H, H, H * G)]
    starts = [[2000, 7], [100, 1900], [2100, 300], [0, 0]]

    def step(cache, k, v, q, start):
        mo.kv8_append(cache, k, v, table, start)
        return mo.kv8_attention(q, cache, table, start + new)

    want = [step(both[0].gpu, *x, _i32(s, dev)) for s in starts]
    static = _i32(starts[0], dev)
    scratch = Both(dev, _rng("same"), B, 40, H, D, page)
    graph = torch.cuda.CUDAGraph()
    step(scratch.gpu, *x, static)
    with torch.cuda.graph(graph):
        out = step(scratch.gpu, *x, static)
    for name, t in zip(("k_codes", "v_codes", "k_scales", "v_scales"), range(4)):
        scratch.gpu._tensors[t].copy_(both[1].gpu._tensors[t])
    for i, s in enumerate(starts):
        static.copy_(_i32(s, dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = [step(both[1].gpu, *x, _i32(s, dev)) for s in starts]
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty(dev):
    import metalops_amd as mo
    cache = mo.KV8Cache.empty(4, 2, 64, 16, dev)
    table, lens = torch.zeros(0, 3, dtype=torch.int32, device=dev), torch.zeros(0, dtype=torch.int32, device=dev)
    none = torch.zeros(0, 2, 64, device=dev)
    mo.kv8_append(cache, none, none, table, lens)
    assert mo.kv8_attention(none.half(), cache, table, lens).shape == (0, 2, 64)
    assert mo.kv8_read(cache, table, lens)[0].shape == (0, 48, 2, 64)
    t2, l2 = torch.zeros(2, 0, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    out, lse = mo.kv8_attention(torch.ones(2, 4, 64, dtype=torch.float16, device=dev), cache, t2, l2, return_lse=True)
    assert not out.any() and (lse == -float("inf")).all()
