"""kv8_compact, kv8_copy_pages and kv8_rename's part of it in captured graphs, replayed among eager calls and beside each other."""
import random

import pytest
import torch

from kv8_pool_ref import used
from test_gpu_kv8_pool import Both, _dealt, _ints

pytestmark = pytest.mark.gpu


class _Holes:
    """A pool full of holes, two tables over it and pages to copy; `expect` is what one round leaves behind."""

    def __init__(self, dev, seed, layers=2, P=400, H=2, D=64, page=16):
        rng = random.Random(seed)
        self.both = both = Both(dev, layers, P, H, D, page, seed)
        self.rows, self.lens = _dealt(rng, P, 12, 9, page)
        both.seed_refs((self.rows, self.lens))
        n = sum(r > 0 for r in both.ref.refs)
        assert 0 < n < P - 40
        self.refs = both.gpu.refs.clone()
        self.start = [_ints(dev, self.rows[:7]), _ints(dev, self.rows[7:])]
        self.tables = [t.clone() for t in self.start]
        # Behind the pages in use after the move, which are the first n.
        to = rng.sample(range(n, P), 30)
        self.src, self.dst = [rng.randrange(n) for _ in to] + [-1, 2], to + [3, P]
        self.gpu_src, self.gpu_dst = _ints(dev, self.src), _ints(dev, self.dst)
        for t in self.rows:
            assert all(e == -1 or e < P for e in t)

    def reset(self):
        self.both.gpu.refs.copy_(self.refs)
        for t, s in zip(self.tables, self.start):
            t.copy_(s)
        for c, start in zip(self.both.gpu.caches, self.both.start):
            for t, s in zip(c._tensors, start):
                t.copy_(s)

    def round_(self):
        import metalops_amd as mo
        live = mo.kv8_compact(self.both.gpu, *self.tables)
        mo.kv8_copy_pages(self.both.gpu, self.gpu_src, self.gpu_dst)
        return live

    def check(self, live):
        ref = self.both.ref
        if not hasattr(self, "want"):
            rows = [r[:] for r in self.rows]
            self.want = ref.compact(rows)
            for s, d in zip(self.src, self.dst):
                if ref.is_page(s) and ref.is_page(d):
                    ref.pages[d] = ref.pages[s]
            self.moved = rows
        assert live.item() == self.want
        self.both.check(torch.cat(self.tables), self.moved)


def test_replayed_among_eager_calls(dev):
    one, two = _Holes(dev, 1), _Holes(dev, 2)
    for h in (one, two):
        h.check(h.round_())
    torch.cuda.synchronize()
    graphs = []
    for h in (one, two):
        h.reset()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            live = h.round_()
        graphs.append((g, live))
    side = torch.cuda.Stream()
    for i in range(5):
        one.reset()
        two.reset()
        for _, live in graphs:
            live.fill_(-7)
        side.wait_stream(torch.cuda.current_stream())
        # The two pools at once: both graphs, or a graph beside an eager call.
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            if i % 2:
                graphs[1][0].replay()
            else:
                graphs[1][1].copy_(two.round_())
        torch.cuda.synchronize()
        one.check(graphs[0][1])
        two.check(graphs[1][1])
        # And eagerly, with another count of pages in use, between the replays.
        one.reset()
        one.tables[0][0] = -1
        one.both.gpu.refs.sub_(torch.bincount(one.start[0][0][:used(one.lens[0], 16)].long(), minlength=400).int())
        one.round_()
        torch.cuda.synchronize()


def test_captured_resizes_of_two_pools(dev):
    """Graphs captured on one stream have workspaces of their own: replayed at once on two streams, again and again."""
    import metalops_amd as mo
    sides, rounds = [torch.cuda.Stream() for _ in range(2)], []
    for seed in range(2):
        rng = random.Random(seed)
        both = Both(dev, 2, 500, 2, 64, 16, seed)
        rows, lens = _dealt(rng, 300, 30, 9, 16)
        both.seed_refs((rows, lens))
        to = [min(n + rng.randint(0, 20), 9 * 16) for n in lens]
        start, refs = _ints(dev, rows), both.gpu.refs.clone()
        gpu, gpu_lens, gpu_to = start.clone(), _ints(dev, lens), _ints(dev, to)
        mo.kv8_resize(both.gpu, gpu, gpu_lens, gpu_to)
        gpu.copy_(start)
        both.gpu.refs.copy_(refs)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            missing = mo.kv8_resize(both.gpu, gpu, gpu_lens, gpu_to)
        for c, s in zip(both.gpu.caches, both.start):
            for t, u in zip(c._tensors, s):
                t.copy_(u)
        want = both.ref.resize(rows, lens, to)
        rounds.append((both, g, gpu, start, refs, missing, rows, want, (gpu_lens, gpu_to)))      # the graph reads the lengths
    for _ in range(5):
        for both, _, gpu, start, refs, missing, *_ in rounds:
            gpu.copy_(start)
            both.gpu.refs.copy_(refs)
            missing.fill_(-7)
        for side, r in zip(sides, rounds):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                r[1].replay()
        torch.cuda.synchronize()
        for both, _, gpu, _, _, missing, rows, want, _ in rounds:
            assert missing.item() == want
            both.check(gpu, rows)
