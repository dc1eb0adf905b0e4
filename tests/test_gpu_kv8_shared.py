"""kv8_shared_attention on the GPU against the formula in 64 bits over each sequence's prefix and own tokens.

The errors are those of kv8_attention: the output's rounding (half a step) and
  * P in fp16: 2^-11 of each weight, and where it is subnormal half a step of 2^-24 relative to 2^6, which a row's largest
    product of a weight and its page's scale reaches in either part, times 448, the largest code;
  * scores in fp32: D + 4 roundings of 2^-24 of sum |q||k| scale, of a weight and of the weights' sum; exp2's 2^-22;
  * sums in fp32: one rounding of 2^-24 for each token and for each of the parts that are added, of the weighted sum of |v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
I32 = torch.int32


def _cum(n):
    out = [0]
    for v in n:
        out.append(out[-1] + v)
    return out


class Batch:
    """A cache of random codes, prefixes and sequences, their pages in no order."""

    def __init__(self, dev, dtype, prefix, members, new, own, H, G, D, page, each=False, seed=0, spread=4, first=0):
        """first: sequences ahead of the groups, that have no prefix (as those behind them)."""
        import metalops_amd as mo
        g = torch.Generator().manual_seed(seed + 7 * sum(prefix) + sum(own) + D)
        self.dev, self.H, self.G, self.D, self.page = dev, H, G, D, page
        self.prefix, self.members, self.new, self.own = prefix, members, new, own
        S, B = len(prefix), len(own)
        W0, W = max(1, -(-max(prefix) // page)), max(1, -(-max(own) // page))
        P = S * W0 + B * W + 2
        k = torch.randint(0, 256, (P, H, page, D), generator=g, dtype=torch.uint8)
        v = torch.randint(0, 256, (P, H, D, page), generator=g, dtype=torch.uint8)
        for c in (k, v):                             # no NaN, and ordinary exponents
            c[(c & 127) > 110] &= 0x8F
        ks, vs = (torch.randint(118, 118 + spread, (P, H), generator=g, dtype=torch.uint8) for _ in range(2))
        ids = torch.randperm(P, generator=g)[:P - 2].to(I32)
        self.prefix_table, self.table = ids[:S * W0].view(S, W0).to(dev), ids[S * W0:].view(B, W).to(dev)
        self.cache = mo.KV8Cache(*(t.to(dev) for t in (k, v, ks, vs)))
        self.prefix_lens, self.context = self.ints(prefix), self.ints(own)
        self.groups = None if len(set(members)) == 1 and S * members[0] == B and not first else self.ints([first + c for c in _cum(members)])
        self.first = first
        self.cu = None if each else self.ints(_cum(new))
        self.q = (torch.randn(sum(new), H * G, D, generator=g) * 0.5).to(DT[dtype]).to(dev)

    def ints(self, x):
        return torch.tensor(x, dtype=I32, device=self.dev)

    def values(self, row, n, h):
        """Keys and values [n, D] of a row's first n tokens, pages that are not there cut out (their tokens: seen 0)."""
        c = self.cache
        ids = row[:-(-n // self.page)].long()
        ok = (ids >= 0) & (ids < c.num_pages)
        ids = ids.clamp(0, c.num_pages - 1)
        k = c.k_codes[ids, h].view(torch.float8_e4m3fn).double() * self.power(c.k_scales[ids, h])
        v = c.v_codes[ids, h].view(torch.float8_e4m3fn).double() * self.power(c.v_scales[ids, h])
        vs = self.power(c.v_scales[ids, h]).expand(-1, self.page, 1)
        flat = lambda t: t.reshape(-1, t.shape[-1])[:n]
        return flat(k), flat(v.transpose(1, 2)), flat(vs)[:, 0], ok[:, None].expand(-1, self.page).reshape(-1)[:n]

    @staticmethod
    def power(byte):
        p = torch.pow(2.0, byte.double() - 127)
        return torch.where(byte == 255, torch.full_like(p, math.nan), p)[:, None, None]

    def exact(self, scale):
        """out, lse and what out and lse may be off by."""
        T, HG, D = self.q.shape
        out, off = (torch.zeros(T, HG, D, dtype=torch.float64, device=self.dev) for _ in range(2))
        lse, lse_off = torch.full((T, HG), -math.inf, dtype=torch.float64, device=self.dev), torch.zeros(T, HG, dtype=torch.float64, device=self.dev)
        eps = torch.finfo(self.q.dtype).eps
        group = {}
        at = self.first
        for s, m in enumerate(self.members):
            group.update({b: s for b in range(at, at + m)})
            at += m
        cu = _cum(self.new)
        for b, (n, L) in enumerate(zip(self.new, self.own)):
            s = group.get(b)
            Lp = self.prefix[s] if s is not None else 0
            rows = slice(cu[b], cu[b + 1])
            pos = L - n + torch.arange(n, device=self.dev)
            for h in range(self.H):
                heads = slice(h * self.G, (h + 1) * self.G)
                parts = [self.values(self.table[b], L, h)]
                if s is not None:
                    parts.insert(0, self.values(self.prefix_table[s], Lp, h))
                k, v, vs, there = (torch.cat(t) for t in zip(*parts))
                q = self.q[rows, heads].double().reshape(n * self.G, D)
                sc = (q @ k.t()) * scale
                size = (q.abs() @ k.abs().t()) * abs(scale)
                seen = torch.ones(n, Lp + L, dtype=torch.bool, device=self.dev)
                seen[:, Lp:] = torch.arange(L, device=self.dev) <= pos[:, None]
                seen &= there & (pos >= 0)[:, None]
                seen = seen[:, None].expand(n, self.G, Lp + L).reshape(n * self.G, Lp + L)
                sc = sc.masked_fill(~seen, -math.inf)
                some = seen.any(1)
                w = torch.softmax(sc, 1).nan_to_num(0.0) if not bool(sc.isnan().any()) else torch.softmax(sc, 1)
                w = torch.where(some[:, None], w, torch.zeros_like(w))
                o = w @ torch.where(there[:, None], v, torch.zeros_like(v))
                av = w @ v.abs().nan_to_num(0.0)
                top = (w * 448 * vs).amax(1, keepdim=True) if Lp + L else torch.zeros(n * self.G, 1, device=self.dev)
                ds = (D + 4) * 2.0 ** -24 * torch.where(seen, size, torch.zeros_like(size)).amax(1, keepdim=True) + 2.0 ** -21 if Lp + L else 0
                bound = av * (2.0 ** -11 + 2 * ds + (Lp + L + 600) * 2.0 ** -24) + (Lp + L) * 2.0 ** -25 / 2 ** 6 * top
                bound = bound * (1 + eps) + o.abs() * eps / 2 + (2.0 ** -25 if self.q.dtype == torch.float16 else 2.0 ** -134)
                shape = (n, self.G, D)
                out[rows, heads], off[rows, heads] = o.view(shape), bound.view(shape)
                if Lp + L:
                    e = torch.logsumexp(sc, 1)
                    lse[rows, heads] = torch.where(some, e, torch.full_like(e, -math.inf)).view(shape[:2])
                    tol = ds[:, 0] + 2.0 ** -20 + (Lp + L + 600) * 2.0 ** -24 + torch.where(some, e.abs(), torch.zeros_like(e)) * 2.0 ** -22
                    lse_off[rows, heads] = tol.view(shape[:2])
        return out, lse, off, lse_off

    def call(self, **kw):
        import metalops_amd as mo
        kw = dict(dict(cu_seqlens=self.cu, groups=self.groups, max_prefix=max(self.prefix), max_context=max(self.own)), **kw)
        return mo.kv8_shared_attention(kw.pop("q", self.q), self.cache, self.prefix_table, self.prefix_lens, self.table, self.context, **kw)

    def check(self, scale=None, want=None, **kw):
        out, lse, off, lse_off = want or self.exact(self.D ** -0.5 if scale is None else scale)
        got, got_lse = self.call(scale=scale, return_lse=True, **kw)
        assert got.dtype == self.q.dtype and got.shape == out.shape
        err = (got.double() - out).abs()
        assert bool((err <= off).all()), f"worst {(err / off.clamp(min=1e-300)).max().item()} of the bound at {(err > off).nonzero()[0].tolist()}"
        inf = lse == -math.inf
        assert torch.equal(got_lse == -math.inf, inf)
        assert bool(((got_lse.double() - lse).abs() <= lse_off)[~inf].all())
        return got, got_lse


CASES = [  # prefixes, members, new tokens, own contexts, H, G, D, page
    ([1], [1], [1], [1], 1, 1, 16, 16),
    ([700], [3], [1] * 3, [1, 64, 65], 2, 4, 128, 64),
    ([64], [2], [1, 1], [10, 130], 1, 7, 80, 32),
    ([4100], [9], [1] * 9, [1 + 50 * i for i in range(9)], 2, 8, 64, 16),
    ([63, 0, 129], [2, 3, 1], [1] * 6, [5, 1, 17, 200, 64, 3], 3, 2, 96, 16),
    ([1000, 70], [20, 20], [1] * 40, [(i * 37) % 150 for i in range(40)], 1, 4, 128, 64),
    ([513], [5], [3, 1, 0, 8, 2], [3, 40, 9, 100, 65], 2, 4, 256, 128),
    ([300, 2000], [1, 3], [60, 2, 33, 1], [60, 10, 100, 1], 2, 4, 128, 32),
    ([130, 5], [2, 1], [140, 70, 9], [300, 70, 20], 1, 2, 192, 64),
    ([200], [70], [1] * 70, [1 + i % 20 for i in range(70)], 1, 1, 64, 64),
    ([90], [3], [5, 5, 5], [4, 5, 0], 2, 2, 64, 64),             # more new tokens than there are of the own context
    ([3 + i for i in range(70)], [1 + i % 2 for i in range(70)], [1] * 105, [1 + i % 5 for i in range(105)], 2, 4, 32, 16),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_formula(dev, dtype, case):
    prefix, members, new, own, H, G, D, page = CASES[case]
    print(f"shared {dtype} {prefix[:6]} {members[:6]} {new[:6]} {own[:6]} H={H} G={G} D={D} page={page}", flush=True)
    b = Batch(dev, dtype, prefix, members, new, own, H, G, D, page, each=len(set(new)) == 1 and dtype == "f16")
    b.check()
    b.check(max_prefix=None, max_context=None)


@pytest.mark.parametrize("wgs", [1, 7, 64, 2000])
@pytest.mark.parametrize("rows,tiles,cost", [(16, 16, 2), (16, 128, 2), (16, 128, 64), (256, 128, 2)])
def test_every_kernel_and_division(dev, wgs, rows, tiles, cost, monkeypatch):
    """Tiles in one stretch and in many, both kinds of tile of prefixes, both kernels of the own tokens, every number of channel tiles."""
    monkeypatch.setenv("MCQ4_KV8_PREFIX_WGS", str(wgs))
    monkeypatch.setenv("MCQ4_KV8_PREFIX_ROWS", str(tiles))
    monkeypatch.setenv("MCQ4_KV8_PREFIX_COST", str(cost))
    monkeypatch.setenv("MCQ4_KV8_ROWS", str(rows))
    for D in (16, 64, 80, 128, 160, 176, 208, 256):
        print(f"shared wgs {wgs} rows {rows} tiles {tiles} cost {cost} D {D}", flush=True)
        Batch(dev, "bf16", [900, 77, 0], [9, 4, 2], [1] * 9 + [3, 1, 2, 5] + [2, 1], [1, 30, 200] * 3 + [3, 1, 2, 90] + [70, 3], 2, 4, D, 64).check()


def test_scales(dev):
    """A scale given, negative and zero; scores of which one row's largest lies far above another's."""
    b = Batch(dev, "f16", [333], [6], [1] * 6, [1, 2, 3, 64, 65, 100], 2, 4, 128, 64)
    for scale in (0.3, -0.2, 0.0, 2.0):
        b.check(scale=scale)


@pytest.mark.parametrize("rows,tiles", [(16, 16), (16, 128), (256, 128)])
def test_pages_of_very_different_scales(dev, rows, tiles, monkeypatch):
    monkeypatch.setenv("MCQ4_KV8_ROWS", str(rows))
    monkeypatch.setenv("MCQ4_KV8_PREFIX_ROWS", str(tiles))
    b = Batch(dev, "bf16", [2000], [12], [1] * 12, [1 + 9 * i for i in range(12)], 2, 4, 128, 32)
    g = torch.Generator().manual_seed(5)
    b.cache.v_scales.copy_(torch.randint(90, 160, b.cache.v_scales.shape, generator=g, dtype=torch.uint8))
    b.check()
    b.cache.k_scales.copy_(torch.randint(100, 125, b.cache.k_scales.shape, generator=g, dtype=torch.uint8))
    b.check()


def test_sequences_of_no_group(dev):
    """Ahead of the groups and behind them: as kv8_attention of their own tokens, each off by no more than it may be."""
    import metalops_amd as mo
    for first, members in ((2, [2, 1]), (0, [1, 2]), (3, [0, 0])):
        b = Batch(dev, "f16", [100, 300], members, [1, 2, 1, 1, 3, 1, 1], [1, 5, 60, 70, 8, 100, 9], 2, 4, 64, 16, first=first)
        got, lse = b.check()
        _, _, off, lse_off = b.exact(b.D ** -0.5)
        alone, alone_lse = mo.kv8_attention(b.q, b.cache, b.table, b.context, b.cu, return_lse=True)
        rows = [t for i in range(7) if not first <= i < first + sum(members) for t in range(_cum(b.new)[i], _cum(b.new)[i + 1])]
        assert bool(((got.double() - alone.double()).abs() <= 2 * off)[rows].all()) and bool(((lse - alone_lse).abs() <= 2 * lse_off)[rows].all())


def test_rows_of_no_sequence_and_senseless_groups(dev):
    """Rows before the first offset and from the last one on are 0; groups that fall or leave the batch end without a fault,
    and rows of sequences that they do not name are right."""
    b = Batch(dev, "bf16", [200, 90], [2, 2], [2, 2, 2, 2], [5, 6, 7, 80], 2, 4, 64, 16)
    want, want_lse = b.check()
    q = torch.randn(11, 8, 64, device=dev).bfloat16()
    q[2:10] = b.q
    got, lse = b.call(q=q, cu_seqlens=b.ints([2, 4, 6, 8, 10]), groups=b.ints([0, 2, 4]), return_lse=True)
    torch.testing.assert_close(got[2:10], want, rtol=2.0 ** -7, atol=1e-3)
    assert (got[:2] == 0).all() and (got[10:] == 0).all() and (lse[:2] == -math.inf).all() and (lse[10:] == -math.inf).all()
    for groups in ([3, 1, 4], [0, 9, 4], [-1, 2, 4], [4, 4, 0], [1 << 30, 1 << 30, 1 << 30]):
        out = b.call(groups=b.ints(groups))
        torch.cuda.synchronize()
        assert out.shape == want.shape
    lens = b.prefix_lens.clone()
    b.prefix_lens.copy_(b.ints([1 << 30, -5]))       # past the table: all of it; negative: none
    b.prefix = [b.prefix_table.shape[1] * 16, 0]
    b.check()
    b.prefix_lens.copy_(lens)


@pytest.mark.parametrize("rows,tiles", [(16, 16), (16, 128), (256, 128)])
def test_missing_pages_and_nan(dev, rows, tiles, monkeypatch):
    """Pages that are not there are not seen; NaN behind a prefix's end does no harm, in it it reaches its rows only."""
    monkeypatch.setenv("MCQ4_KV8_ROWS", str(rows))
    monkeypatch.setenv("MCQ4_KV8_PREFIX_ROWS", str(tiles))
    b = Batch(dev, "f16", [150, 400], [3, 3], [1] * 6, [10, 20, 30, 64, 1, 90], 2, 4, 64, 64)
    b.prefix_table[1, 2] = -1
    b.prefix_table[0, 1] = 1 << 29
    b.check()
    want = b.call()
    c = b.cache
    p = int(b.prefix_table[1, 6])                    # tokens 384 to 447, of which 16 are seen
    c.k_codes[p, :, 16:] = 0x7F
    c.v_codes[p, :, :, 16:] = 0xFF
    spare = sorted(set(range(c.num_pages)) - set(b.prefix_table.flatten().tolist()) - set(b.table.flatten().tolist()))[0]
    c.k_scales[spare] = 255
    c.v_scales[spare] = 255
    assert torch.equal(b.call(), want)
    for what in ("k", "v", "ks", "vs"):
        keep = [t.clone() for t in c._tensors]
        q = int(b.prefix_table[1, 3])
        if what == "k":
            c.k_codes[q, 1, 5, 3] = 0x7F
        elif what == "v":
            c.v_codes[q, 1, 7, 63] = 0xFF
        elif what == "ks":
            c.k_scales[q, 1] = 255
        else:
            c.v_scales[q, 1] = 255
        got = b.call()
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[3:, 4:, 7 if what == "v" else slice(None)] = True
        assert torch.equal(got.isnan(), bad), what
        assert torch.equal(got[~bad], want[~bad])
        for t, u in zip(c._tensors, keep):
            t.copy_(u)


@pytest.mark.parametrize("rows", [16, 256])
def test_nan_in_own_tokens(dev, rows, monkeypatch):
    """NaN of the newest of several new tokens: the rows ahead of it do not see it."""
    monkeypatch.setenv("MCQ4_KV8_ROWS", str(rows))
    b = Batch(dev, "bf16", [70], [2], [5, 5], [40, 70], 2, 4, 64, 32)
    want = b.call()
    c, token = b.cache, 68                           # new tokens 65 .. 69 of sequence 1
    p, slot = int(b.table[1, token // 32]), token % 32
    for what in ("k", "v"):
        keep = [t.clone() for t in c._tensors]
        if what == "k":
            c.k_codes[p, 0, slot, 9] = 0x7F
        else:
            c.v_codes[p, 0, 11, slot] = 0xFF
        got = b.call()
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[8:, :4, 11 if what == "v" else slice(None)] = True
        assert torch.equal(got.isnan(), bad), what
        assert torch.equal(got[~bad], want[~bad])
        for t, u in zip(c._tensors, keep):
            t.copy_(u)


@pytest.mark.parametrize("rows,tiles", [(16, 16), (16, 128), (256, 128)])
def test_infinities_and_nan_in_q(dev, rows, tiles, monkeypatch):
    """They make their own row of their head NaN, lse too, and no other."""
    monkeypatch.setenv("MCQ4_KV8_ROWS", str(rows))
    monkeypatch.setenv("MCQ4_KV8_PREFIX_ROWS", str(tiles))
    b = Batch(dev, "bf16", [300, 70], [3, 2], [1, 3, 1, 2, 4], [20, 70, 130, 9, 64], 2, 4, 64, 32)
    want, want_lse = b.call(return_lse=True)
    q, bad = b.q.clone(), torch.zeros(b.q.shape[:2], dtype=torch.bool, device=dev)
    for t, h, value in ((0, 3, math.inf), (2, 5, math.nan), (5, 0, -math.inf), (10, 7, math.nan)):
        q[t, h, 11], bad[t, h] = value, True
    got, lse = b.call(q=q, return_lse=True)
    assert got[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(got[~bad], want[~bad]) and torch.equal(lse[~bad], want_lse[~bad])


def test_many_sequences(dev):
    """More sequences and prefixes than a wave counts at a time, many of them without new tokens or context."""
    n = 700
    b = Batch(dev, "f16", [(i * 29) % 90 for i in range(150)], [4 + (i % 3 == 0) for i in range(150)][:140] + [0] * 10,
              [(i * 5) % 3 for i in range(n)], [(i * 13) % 70 if i % 4 else 0 for i in range(n)], 1, 2, 32, 16)
    b.check()


def test_same_as_one_table(dev):
    """kv8_attention over tables that begin with the prefix's pages: the same tokens, within two roundings."""
    import metalops_amd as mo
    b = Batch(dev, "bf16", [256], [4], [3] * 4, [3, 70, 128, 5], 2, 4, 128, 64)
    whole = torch.cat([b.prefix_table.expand(4, -1), b.table], 1)
    one, one_lse = mo.kv8_attention(b.q, b.cache, whole, b.context + 256, return_lse=True)
    two, two_lse = b.check()
    _, _, off, lse_off = b.exact(128 ** -0.5)
    assert bool(((one.double() - two.double()).abs() <= 2 * off).all()) and bool(((one_lse - two_lse).abs() <= 2 * lse_off).all())
    # The columns of forked tables as they are.
    got = mo.kv8_shared_attention(b.q, b.cache, whole[:1, :4], b.prefix_lens, whole[:, 4:], b.context)
    _, _, off, _ = b.exact(128 ** -0.5)
    assert bool(((got.double() - two.double()).abs() <= 2 * off).all())


def test_layouts_of_q(dev):
    b = Batch(dev, "f16", [300], [5], [2] * 5, [2, 9, 70, 3, 64], 2, 4, 64, 32)
    want = b.call()
    assert torch.equal(b.call(q=b.q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    wide = torch.zeros(10, 8, 80, dtype=b.q.dtype, device=dev)
    for at in (0, 8, 1):
        wide[:, :, at:at + 64] = b.q
        assert torch.equal(b.call(q=wide[:, :, at:at + 64]), want)


def test_empty(dev):
    import metalops_amd as mo
    b = Batch(dev, "f16", [30], [2], [1, 1], [4, 5], 1, 2, 64, 16)
    alone, alone_lse = mo.kv8_attention(b.q, b.cache, b.table, b.context, return_lse=True)
    for table, lens, groups in ((b.prefix_table[:, :0], b.prefix_lens, None), (b.prefix_table[:0], b.prefix_lens[:0], None),
                                (b.prefix_table[:0], b.prefix_lens[:0], b.ints([0]))):
        out, lse = mo.kv8_shared_attention(b.q, b.cache, table, lens, b.table, b.context, groups=groups, return_lse=True)
        assert torch.equal(out, alone) and torch.equal(lse, alone_lse)
    out, lse = mo.kv8_shared_attention(b.q, b.cache, b.prefix_table, b.prefix_lens, b.table[:, :0], b.context, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert mo.kv8_shared_attention(b.q[:0], b.cache, b.prefix_table, b.prefix_lens, b.table, b.context).shape == (0, 2, 64)


def test_graph_and_streams(dev):
    """Captured calls replayed among eager ones on two streams, with longer contexts from replay to replay."""
    b = Batch(dev, "bf16", [3000, 500], [8, 4], [1] * 12, [60 + 5 * i for i in range(12)], 2, 4, 128, 64)
    b.call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = b.call(return_lse=True)
    side = torch.cuda.Stream()
    for i in range(4):
        b.own = [20 * i + 5 * j for j in range(12)]
        b.prefix = [3000 - 700 * i, 500]
        b.context.copy_(b.ints(b.own))
        b.prefix_lens.copy_(b.ints(b.prefix))
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = b.call(return_lse=True, max_prefix=3000, max_context=115)
        g.replay()
        eager = b.call(return_lse=True, max_prefix=3000, max_context=115)
        torch.cuda.synchronize()
        for x, y, z in zip((out, lse), beside, eager):
            assert torch.equal(x, y) and torch.equal(x, z)
        b.check(max_prefix=3000, max_context=115)


def test_offsets_past_32_bits(dev):
    """Pages beyond 2^32 bytes of codes."""
    import metalops_amd as mo
    H, D, page, P = 8, 128, 64, 66000
    assert P * H * D * page > 2 ** 32
    b = Batch(dev, "f16", [130], [3], [1] * 3, [1, 65, 70], H, 1, D, page)
    big = mo.KV8Cache.empty(P, H, D, page, dev)
    used = sorted(set(b.prefix_table.flatten().tolist()) | set(b.table.flatten().tolist()))
    names = torch.zeros(b.cache.num_pages, dtype=I32, device=dev)
    for i, p in enumerate(used):
        to = P - 1 - 3 * i
        names[p] = to
        for t, s in zip(big._tensors, b.cache._tensors):
            t[to] = s[p]
    want = b.call()
    b.cache, b.prefix_table, b.table = big, names[b.prefix_table.long()], names[b.table.long()]
    assert torch.equal(b.call(), want)
