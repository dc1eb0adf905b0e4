"""kv8_shared_attention with offsets that fall or leave their range: every result is defined, and none comes from an earlier call."""
import math

import pytest
import torch

from test_gpu_kv8_shared import I32, Batch

pytestmark = pytest.mark.gpu


def _earlier_calls(b, seed):
    """Calls whose locations of records, of prefixes' and of own tokens, stay behind in the workspace."""
    g = torch.Generator().manual_seed(seed)
    for _ in range(2):
        b.call(q=(torch.randn(b.q.shape, generator=g) * 8).to(b.q.dtype).to(b.dev), max_prefix=None, max_context=None)


@pytest.mark.parametrize("rows,tiles", [(16, 16), (16, 128), (256, 128)])
@pytest.mark.parametrize("groups", [[3, 1, 4], [0, 9, 4], [-1, 2, 4], [4, 4, 0], [1 << 30, 1 << 30, 1 << 30], [-1 << 31, 2, 4], [0, 2, 5]])
def test_groups(dev, groups, rows, tiles, monkeypatch):
    """No sequence has a prefix then: kv8_attention of the own tokens, within two roundings, after whatever calls."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_KV8_ROWS", str(rows))
    monkeypatch.setenv("MCQ4_KV8_PREFIX_ROWS", str(tiles))
    print(f"shared, groups {groups} rows {rows} tiles {tiles}", flush=True)
    b = Batch(dev, "bf16", [200, 90], [2, 2], [2, 3, 2, 2], [5, 6, 70, 80], 2, 4, 64, 16)
    none = Batch(dev, "bf16", [200, 90], [0, 0], [2, 3, 2, 2], [5, 6, 70, 80], 2, 4, 64, 16)
    _, _, off, lse_off = none.exact(b.D ** -0.5)
    alone, alone_lse = mo.kv8_attention(b.q, b.cache, b.table, b.context, b.cu, return_lse=True)
    results = []
    for seed in range(3):
        _earlier_calls(b, seed)
        out, lse = b.call(groups=b.ints(groups), max_prefix=None, max_context=None, return_lse=True)
        assert bool(((out.double() - alone.double()).abs() <= 2 * off).all())
        assert bool(((lse.double() - alone_lse.double()).abs() <= 2 * lse_off).all())
        results.append((out, lse))
    for out, lse in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(lse, results[0][1])


@pytest.mark.parametrize("tiles", [16, 128])
@pytest.mark.parametrize("cu", [[0, 5, 3, 8, 9], [0, 2, 20, 7, 9], [-3, 2, 5, 7, 9], [9, 9, 9, 9, 0], [0, 2, 5, 7, 10], [0, 2, 5, 0, 0]])
def test_offsets_of_new_tokens(dev, cu, tiles, monkeypatch):
    """No row is a sequence's then: all are 0, after whatever calls."""
    monkeypatch.setenv("MCQ4_KV8_ROWS", "16")
    monkeypatch.setenv("MCQ4_KV8_PREFIX_ROWS", str(tiles))
    print(f"shared, offsets {cu} tiles {tiles}", flush=True)
    b = Batch(dev, "f16", [200, 90], [2, 2], [2, 3, 2, 2], [5, 6, 70, 80], 2, 4, 64, 16)
    for groups in (None, b.ints([0, 2, 4]), b.ints([1, 1, 3])):
        _earlier_calls(b, 1)
        out, lse = b.call(cu_seqlens=b.ints(cu), groups=groups, max_prefix=None, max_context=None, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_offsets_of_prompts(dev, monkeypatch):
    """The prompts' kernels take the sequences whose offsets rise; those in no group's range have no prefix."""
    import metalops_amd as mo
    monkeypatch.setenv("MCQ4_KV8_ROWS", "256")
    b = Batch(dev, "f16", [200], [2], [6, 3], [30, 20], 2, 4, 64, 16)
    cu, groups = b.ints([0, 6, 4]), b.ints([0, 2])
    _, _, off, _ = Batch(dev, "f16", [200], [0], [6, 3], [30, 20], 2, 4, 64, 16).exact(b.D ** -0.5)
    alone = mo.kv8_attention(b.q, b.cache, b.table, b.context, b.ints([0, 6, 9]))
    results = []
    for seed in range(3):
        _earlier_calls(b, seed)
        results.append(b.call(cu_seqlens=cu, groups=groups, max_prefix=None, max_context=None)[:6])
        # The group ends at token 4: tokens 4 and 5 are behind it.
        assert bool(((results[-1][4:6].double() - alone[4:6].double()).abs() <= 2 * off[4:6]).all())
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


@pytest.mark.parametrize("rows,tiles", [(16, 16), (16, 128), (256, 128)])
def test_fewer_tokens_than_rows(dev, rows, tiles, monkeypatch):
    """Offsets that rise but leave rows of q ahead of the first sequence and behind the last one, with and without groups."""
    monkeypatch.setenv("MCQ4_KV8_ROWS", str(rows))
    monkeypatch.setenv("MCQ4_KV8_PREFIX_ROWS", str(tiles))
    b = Batch(dev, "bf16", [200, 90], [2, 2], [2, 3, 2, 2], [5, 6, 70, 80], 2, 4, 64, 16)
    out, _, off, _ = b.exact(b.D ** -0.5)
    q = torch.randn(14, 8, 64, device=dev).bfloat16()
    q[3:12] = b.q
    for groups in (None, b.ints([0, 2, 4])):
        _earlier_calls(b, 5)
        got, lse = b.call(q=q, cu_seqlens=b.ints([3, 5, 8, 10, 12]), groups=groups, max_prefix=None, max_context=None, return_lse=True)
        assert bool(((got[3:12].double() - out).abs() <= off).all())
        for rest in (slice(0, 3), slice(12, 14)):
            assert (got[rest] == 0).all() and (lse[rest] == -math.inf).all()
