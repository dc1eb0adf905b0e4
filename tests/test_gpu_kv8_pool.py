"""The pool's operators on the GPU against kv8_pool_ref: whole numbers and copied bytes, all equal."""
import random

import pytest
import torch

from kv8_pool_ref import Pool, used

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _ints(dev, values):
    return torch.tensor(values, dtype=I32, device=dev)


class Both:
    """A pool on the GPU, whose pages hold random bytes, and its reference."""

    def __init__(self, dev, layers, P, H, D, page, seed=0):
        import metalops_amd as mo
        self.mo, self.dev, self.page = mo, dev, page
        g = torch.Generator().manual_seed(seed)
        self.gpu = mo.KV8Pool.empty(layers, P, H, D, page, dev)
        for c in self.gpu.caches:
            for t in c._tensors:
                t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
        self.start = [[t.clone() for t in c._tensors] for c in self.gpu.caches]
        self.ref = Pool(P, page)

    def seed_refs(self, *tables_lens):
        self.ref.refs = [0] * self.ref.P
        for table, lens in tables_lens:
            for row, n in zip(table, lens):
                for e in row[:used(n, self.page)]:
                    if self.ref.is_page(e):
                        self.ref.refs[e] += 1
        self.gpu.refs.copy_(_ints(self.dev, self.ref.refs))

    def check(self, gpu_table=None, table=None):
        assert self.gpu.refs.tolist() == self.ref.refs
        if table is not None:
            assert gpu_table.tolist() == table
        at = torch.tensor([p for _, p in self.ref.pages], device=self.dev)
        for c, start in zip(self.gpu.caches, self.start):
            for t, s in zip(c._tensors, start):
                assert torch.equal(t, s[at])


def _dealt(rng, P, B, W, page, shared=0.3):
    """Rows of different pages, some of which begin with another row's full pages."""
    free = list(range(P))
    rng.shuffle(free)
    table, lens = [], []
    for b in range(B):
        n = rng.randint(0, W * page)
        row = [-1] * W
        k = 0
        if b and rng.random() < shared:
            a = rng.randrange(b)
            k = min(lens[a] // page, used(n, page))
            row[:k] = table[a][:k]
        for j in range(k, used(n, page)):
            if free:
                row[j] = free.pop()
            else:
                n = j * page
                break
        table.append(row)
        lens.append(n)
    return table, lens


SHAPES = [(1, 40, 1, 16, 16), (3, 130, 2, 64, 16), (2, 33, 3, 80, 32), (2, 300, 8, 128, 64), (1, 20000, 1, 16, 16), (1, 9, 1, 256, 256)]


@pytest.mark.parametrize("layers,P,H,D,page", SHAPES)
@pytest.mark.parametrize("seed", range(3))
def test_a_life_of_rows(dev, layers, P, H, D, page, seed):
    """Rows dealt out, forked, grown, cut, freed and compacted again and again."""
    print(f"pool {layers} x {P} pages of {H} x {page} x {D}, seed {seed}", flush=True)
    rng = random.Random(seed + P)
    both = Both(dev, layers, P, H, D, page, seed)
    B, W = rng.choice([1, 3, 8]), rng.choice([1, 2, 5])
    table, lens = _dealt(rng, P, B, W, page)
    both.seed_refs((table, lens))
    gpu, gpu_lens = _ints(dev, table), _ints(dev, lens)
    for _ in range(12):
        what = rng.choice(["fork", "beams", "resize", "resize", "resize", "compact"])
        if what in ("fork", "beams"):
            parents = [rng.randint(-1, len(table)) for _ in range(rng.randint(1, 12) if what == "fork" else len(table))]
            keep = gpu, gpu_lens, [r[:] for r in table], lens
            gpu, gpu_lens = both.mo.kv8_fork(both.gpu, gpu, gpu_lens, _ints(dev, parents), release=what == "beams")
            table, lens = both.ref.fork(table, lens, parents, what == "beams")
            if what == "fork":                       # the old rows end
                zero = [0] * len(keep[3])
                assert both.mo.kv8_resize(both.gpu, keep[0], keep[1], _ints(dev, zero)).item() == 0
                both.ref.resize(keep[2], keep[3], zero)
                both.check(keep[0], keep[2])
        elif what == "resize":
            to = [rng.choice([n, n + 1, rng.randint(-3, W * page + 3), 0]) for n in lens]
            got = both.mo.kv8_resize(both.gpu, gpu, gpu_lens, _ints(dev, to)).item()
            want = both.ref.resize(table, lens, to)
            assert got == want
            lens = [min(max(n, 0), W * page) if not want or n < m else m for m, n in zip(lens, to)]
            gpu_lens = _ints(dev, lens)
        else:
            assert both.mo.kv8_compact(both.gpu, gpu).item() == both.ref.compact(table)
        assert gpu_lens.tolist() == lens
        both.check(gpu, table)


@pytest.mark.parametrize("B,W,P", [(1, 1, 3), (70, 3, 400), (1500, 2, 5000), (3, 700, 2500)])
def test_many_rows_and_wide_tables(dev, B, W, P):
    rng = random.Random(B)
    both = Both(dev, 1, P, 1, 16, 16)
    table, lens = _dealt(rng, P, B, W, 16)
    both.seed_refs((table, lens))
    gpu = _ints(dev, table)
    parents = [rng.randrange(B) for _ in range(B)]
    gpu, gpu_lens = both.mo.kv8_fork(both.gpu, gpu, _ints(dev, lens), _ints(dev, parents), release=True)
    table, lens = both.ref.fork(table, lens, parents, True)
    both.check(gpu, table)
    to = [n + 1 for n in lens]
    assert both.mo.kv8_resize(both.gpu, gpu, gpu_lens, _ints(dev, to)).item() == both.ref.resize(table, lens, to)
    both.check(gpu, table)
    assert both.mo.kv8_compact(both.gpu, gpu).item() == both.ref.compact(table)
    both.check(gpu, table)


def test_too_few_pages(dev):
    """No row grows, others still shrink, and what they gave back counts."""
    both = Both(dev, 2, 6, 2, 32, 16)
    table, lens = [[0, 1, -1], [2, 3, -1], [4, -1, -1]], [20, 32, 5]
    both.seed_refs((table, lens))
    gpu = _ints(dev, table)
    for to in ([48, 48, 48], [48, 48, 5], [48, 0, 6]):
        got = both.mo.kv8_resize(both.gpu, gpu, _ints(dev, lens), _ints(dev, to)).item()
        want = both.ref.resize(table, lens, to)
        assert got == want
        both.check(gpu, table)
    assert want == 0 and both.ref.refs == [1, 1, 1, 0, 1, 0]


def test_copy_on_write(dev):
    """Two answers grow from one prompt's page: both get copies, and the prompt keeps its own while it lasts."""
    both = Both(dev, 3, 8, 2, 64, 16)
    table, lens = [[5, 2]], [20]
    both.seed_refs((table, lens))
    gpu, gpu_lens = both.mo.kv8_fork(both.gpu, _ints(dev, table), _ints(dev, lens), _ints(dev, [0, 0]))
    assert gpu.tolist() == [[5, 2], [5, 2]] and both.gpu.refs.tolist() == [0, 0, 3, 0, 0, 3, 0, 0]
    assert both.mo.kv8_resize(both.gpu, gpu, gpu_lens, _ints(dev, [21, 24])).item() == 0
    assert gpu.tolist() == [[5, 0], [5, 1]] and both.gpu.refs.tolist() == [1, 1, 1, 0, 0, 3, 0, 0]
    both.ref.refs = both.gpu.refs.tolist()
    both.ref.pages[0] = both.ref.pages[1] = ("page", 2)
    both.check()
    # A full page is shared and not copied; alone, a page is written to as it is.
    assert both.mo.kv8_resize(both.gpu, gpu, _ints(dev, [16, 24]), _ints(dev, [17, 25])).item() == 0
    assert gpu.tolist() == [[5, 3], [5, 1]]


def test_entries_that_are_no_pages(dev):
    """-1 and numbers past the cache are neither counted nor followed."""
    both = Both(dev, 1, 4, 1, 16, 16)
    table, lens = [[1, 99, -5], [-1, 2, 1 << 30]], [48, 40]
    both.seed_refs((table, lens))
    gpu, gpu_lens = _ints(dev, table), _ints(dev, lens)
    parents = [1, -7, 0, 1 << 30]
    new, new_lens = both.mo.kv8_fork(both.gpu, gpu, gpu_lens, _ints(dev, parents))
    rows, row_lens = both.ref.fork(table, lens, parents, False)
    assert new_lens.tolist() == row_lens
    both.check(new, rows)
    to = [30, 0, 48, 3]
    assert both.mo.kv8_resize(both.gpu, new, new_lens, _ints(dev, to)).item() == both.ref.resize(rows, row_lens, to)
    both.check(new, rows)
    assert both.mo.kv8_compact(both.gpu, new, gpu).item() == both.ref.compact(rows, table)
    both.check(new, rows)
    assert gpu.tolist() == table


def test_copy_pages(dev):
    for layers, P, H, D, page in SHAPES[:4]:
        both = Both(dev, layers, P, H, D, page)
        src, dst = [3, 3, -1, 5, 7, P, 1 << 30], [0, 8, 1, -1, 2, 4, 6]
        both.mo.kv8_copy_pages(both.gpu, _ints(dev, src), _ints(dev, dst))
        for s, d in ((3, 0), (3, 8), (7, 2)):
            both.ref.pages[d] = ("page", s)
        both.check()
        both.mo.kv8_copy_pages(both.gpu, _ints(dev, []), _ints(dev, []))
        both.check()


def test_layouts_and_empty(dev):
    """Tables that are parts of wider ones, several tables at once, no rows at all."""
    both = Both(dev, 2, 30, 1, 16, 16)
    table, lens = [[20, 9], [11, 29]], [32, 17]
    both.seed_refs((table, lens), ([[29], [25]], [16, 3]))
    wide = torch.full((2, 7), 8, dtype=I32, device=dev)
    part = wide[:, 2:4]
    part.copy_(_ints(dev, table))
    other = [[29], [25]]
    gpu_other = _ints(dev, other)
    assert both.mo.kv8_resize(both.gpu, part, _ints(dev, lens), _ints(dev, [32, 18])).item() == both.ref.resize(table, lens, [32, 18])
    both.check(part, table)
    assert both.mo.kv8_compact(both.gpu, part, gpu_other, gpu_other[:0]).item() == both.ref.compact(table, other)
    both.check(part, table)
    assert gpu_other.tolist() == other
    wide[:, 2:4] = 8
    assert (wide == 8).all()
    with pytest.raises(RuntimeError, match="in place"):
        both.mo.kv8_resize(both.gpu, part.t(), _ints(dev, lens), _ints(dev, lens))
    none = torch.zeros(0, 2, dtype=I32, device=dev)
    out, out_lens = both.mo.kv8_fork(both.gpu, none, _ints(dev, []), _ints(dev, [0, 1]))
    assert out.tolist() == [[-1, -1]] * 2 and out_lens.tolist() == [0, 0]
    assert both.mo.kv8_resize(both.gpu, none, _ints(dev, []), _ints(dev, [])).item() == 0
    before = sum(both.gpu.refs.tolist())
    out, out_lens = both.mo.kv8_fork(both.gpu, _ints(dev, table), _ints(dev, lens), _ints(dev, []), release=True)
    assert out.shape == (0, 2) and out_lens.shape == (0,) and sum(both.gpu.refs.tolist()) == before - 4


def test_graph_and_streams(dev):
    """A captured round of answers, replayed among eager ones of another pool on another stream."""
    import metalops_amd as mo
    pools = [Both(dev, 2, 60, 2, 64, 16) for _ in range(2)]
    table, lens = [[7, 12, 3, -1], [30, 31, -1, -1]], [40, 20]
    to = _ints(dev, [41, 60, 33, 21])
    parents, zero = _ints(dev, [0, 0, 0, 1]), _ints(dev, [0] * 4)
    gpu, gpu_lens = _ints(dev, table), _ints(dev, lens)
    for p in pools:
        p.seed_refs((table, lens))
    refs = pools[0].gpu.refs.clone()

    def round_(p):
        rows, n = mo.kv8_fork(p.gpu, gpu, gpu_lens, parents)
        missing = mo.kv8_resize(p.gpu, rows, n, to)
        grown, counts = rows.clone(), p.gpu.refs.clone()
        mo.kv8_resize(p.gpu, rows, to, zero)
        return rows, grown, counts, missing
    want = [t.clone() for t in round_(pools[0])]
    held = [[t.clone() for t in c._tensors] for c in pools[0].gpu.caches]
    assert torch.equal(pools[0].gpu.refs, refs)
    round_(pools[1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = round_(pools[0])
    side = torch.cuda.Stream()
    for _ in range(4):
        for t in out:
            t.fill_(77)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = round_(pools[1])
        g.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(out, beside, want):
            assert torch.equal(a, c) and torch.equal(b, c)
        for p in pools:
            assert torch.equal(p.gpu.refs, refs)
            for c, h in zip(p.gpu.caches, held):
                for t, u in zip(c._tensors, h):
                    assert torch.equal(t, u)


def test_appends_stay_with_their_row(dev):
    """Answers to one prompt, forked, grown and appended to, read as if each had its own cache; then compacted."""
    import metalops_amd as mo
    g = torch.Generator().manual_seed(4)
    H, D, page, W = 2, 64, 16, 6
    pool = mo.KV8Pool.empty(1, 40, H, D, page, dev)
    cache = pool.caches[0]
    prompt = torch.randn(2, 37, H, D, generator=g).to(dev)
    table = pool.table(1, W)
    zero, full = _ints(dev, [0]), _ints(dev, [37])
    assert mo.kv8_resize(pool, table, zero, full).item() == 0
    mo.kv8_append(cache, prompt[0], prompt[1], table, zero)
    rows, lens = mo.kv8_fork(pool, table, full, _ints(dev, [0] * 3))
    said = torch.randn(2, 3, 30, H, D, generator=g).to(dev)
    singles = []
    for b in range(3):
        own = mo.KV8Cache.empty(W, H, D, page, dev)
        t = torch.arange(W, dtype=I32, device=dev)[None]
        mo.kv8_append(own, prompt[0], prompt[1], t, zero)
        singles.append((own, t))
    for i in range(30):
        assert mo.kv8_resize(pool, rows, lens, lens + 1).item() == 0
        mo.kv8_append(cache, said[0, :, i], said[1, :, i], rows, lens)
        for b, (own, t) in enumerate(singles):
            mo.kv8_append(own, said[0, b:b + 1, i], said[1, b:b + 1, i], t, lens[b:b + 1])
        lens = lens + 1
        if i in (3, 20):
            mo.kv8_compact(pool, rows, table)
    for b, (own, t) in enumerate(singles):
        for x, y in zip(mo.kv8_read(cache, rows[b:b + 1], lens[b:b + 1]), mo.kv8_read(own, t, lens[b:b + 1])):
            assert torch.equal(x, y)
    for x, y in zip(mo.kv8_read(cache, table, full), mo.kv8_read(singles[0][0], singles[0][1], full)):
        assert torch.equal(x[:, :32], y[:, :32])
    assert (pool.refs > 0).sum().item() == 3 + 3 * (used(67, page) - 2)
