"""Lengths beyond a table's width count as the width, in every call over it, and say so in what is given back."""
import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("beyond", [1, 3, 1000, (1 << 31) - 1])
def test_a_row_that_outgrows_its_table(dev, page, beyond):
    import metalops_amd as mo
    W, H, D = 3, 2, 32
    full = W * page
    print(f"width {full}, page {page}, {beyond} beyond", flush=True)
    ints = lambda x: torch.tensor(x, dtype=I32, device=dev)
    far = min(full + beyond, (1 << 31) - 1)
    pool = mo.KV8Pool.empty(2, 20, H, D, page, dev)
    cache = pool.caches[0]
    table = pool.table(2, W)
    # From nothing and from a page: as many pages as the width has, none lacking.
    assert mo.kv8_resize(pool, table, ints([0, 0]), ints([5, page])).item() == 0
    assert mo.kv8_resize(pool, table, ints([5, page]), ints([far, far])).item() == 0
    assert sorted(table.flatten().tolist()) == list(range(2 * W)) and pool.refs.tolist() == [1] * (2 * W) + [0] * (20 - 2 * W)
    # A row that is full, or said to be more than full, gets nothing more.
    before = table.clone()
    assert mo.kv8_resize(pool, table, ints([far, full]), ints([far, far])).item() == 0
    assert torch.equal(table, before) and pool.refs.sum().item() == 2 * W
    # What is appended behind the width is dropped, and changes no page.
    g = torch.Generator().manual_seed(page)
    k, v = torch.randn(2, 2 * full, H, D, generator=g).to(dev)
    mo.kv8_append(cache, k, v, table, ints([0, 0]))
    held = [t.clone() for t in cache._tensors]
    mo.kv8_append(cache, k[:4], v[:4], table, ints([full, min(far, (1 << 31) - 8)]))
    for t, u in zip(cache._tensors, held):
        assert torch.equal(t, u)
    for x, y in zip(mo.kv8_read(cache, table, ints([far, far])), mo.kv8_read(cache, table, ints([full, full]))):
        assert torch.equal(x, y)
    # Forked rows are as long as they can be.  Of the row that is said to have 7 tokens one page is given back, the others stay counted.
    rows, lens = mo.kv8_fork(pool, table, ints([far, 7]), ints([0, 0, 1]), release=True)
    assert lens.tolist() == [full, full, 7] and rows[0].tolist() == before[0].tolist()
    mo.kv8_resize(pool, rows, ints([far, far, 7]), ints([0, 0, 0]))
    assert pool.refs.clamp(min=0).sum().item() == W - 1
    # Too few pages in the pool: those of the width are counted, not those beyond.
    small = mo.KV8Pool.empty(1, 1, H, D, page, dev)
    assert mo.kv8_resize(small, small.table(1, W), ints([0]), ints([far])).item() == W - 1
