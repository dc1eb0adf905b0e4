"""Pages of the 8-bit key/value cache that sequences share, on MI355X.

A block table says which pages a sequence has; a pool says how many table entries name each
page.  With it sequences share the pages of what they have in common: answers to one prompt,
beams of one search.  ``kv8_fork`` makes rows of others, ``kv8_resize`` gives rows the pages for
more tokens (and a copy of a page that they would write to but do not have alone) or takes
those of fewer, ``kv8_compact`` moves all pages in use to the front.

No counterpart in the reference.  As in the rest of the package the HIP kernels of
``libmcq4.so`` do all of it, on the current stream, without a fallback; counts, tables and
lengths stay on the device and nothing waits for them.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .kv8 import KV8Cache, _int32
from .quantization import _native, _require_device, _stream, _workspace

__all__ = ["KV8Pool", "kv8_copy_pages", "kv8_fork", "kv8_resize", "kv8_compact"]


class KV8Pool:
    """The caches of a model's layers, of one shape and on one device, whose pages have common numbers, and
    ``refs`` (int32 ``[P]``): how many entries of block tables name each page, 0 for a free one."""

    def __init__(self, caches: Sequence[KV8Cache], refs: Optional[torch.Tensor] = None):
        caches = tuple(caches)
        if not caches:
            raise RuntimeError("a pool must have caches")
        c = caches[0]
        for d in caches[1:]:
            if (d.num_pages, d.kv_heads, d.page_size, d.head_dim, d.device) != (c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.device):
                raise RuntimeError(f"the caches of a pool must have one shape and device, got {c} and {d}")
        if refs is None:
            refs = torch.zeros(c.num_pages, dtype=torch.int32, device=c.device)
        if refs.dtype != torch.int32 or tuple(refs.shape) != (c.num_pages,) or not refs.is_contiguous() or refs.device != c.device:
            raise RuntimeError(f"refs must be a contiguous int32 ({c.num_pages},) on {c.device}, got {refs.dtype} {tuple(refs.shape)} on {refs.device}")
        self.caches = caches
        self.num_pages, self.page_size, self.device = c.num_pages, c.page_size, c.device
        layers = torch.tensor([[t.data_ptr() for t in d._tensors] for d in caches], dtype=torch.int64).to(c.device)
        self._tensors = (refs, layers)           # what _struct points to: not to be replaced
        self._struct = _lib.Kv8PoolStruct(layers.data_ptr(), refs.data_ptr(), c.num_pages, len(caches), c.kv_heads, c.head_dim, c.page_size)
        self._address = ctypes.addressof(self._struct)

    refs = property(lambda self: self._tensors[0])

    @classmethod
    def empty(cls, layers: int, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
              device: Union[str, torch.device] = "cuda") -> "KV8Pool":
        """A pool of new caches, all of its pages free."""
        return cls([KV8Cache.empty(num_pages, kv_heads, head_dim, page_size, device) for _ in range(layers)])

    def table(self, batch: int, width: int) -> torch.Tensor:
        """A block table whose entries name no page yet, -1."""
        return torch.full((batch, width), -1, dtype=torch.int32, device=self.device)

    def __repr__(self) -> str:
        return f"KV8Pool(layers={len(self.caches)}, num_pages={self.num_pages}, page_size={self.page_size}, device={self.device})"


def _table(pool: KV8Pool, table: torch.Tensor, in_place: bool) -> torch.Tensor:
    if table.dim() != 2 or table.dtype != torch.int32:
        raise RuntimeError(f"block_table must be int32 [B, W], got {table.dtype} {tuple(table.shape)}")
    if (table.shape[1] > 1 and table.stride(1) != 1) or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        if in_place:
            raise RuntimeError("block_table is changed in place: its rows must be of neighbouring entries and not overlap")
        table = table.contiguous()
    _require_device(pool.refs, table)
    return table


def _row_stride(table: torch.Tensor) -> int:
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


def kv8_copy_pages(pool: KV8Pool, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` (int32 ``[n]``) in every layer.

    Pairs of which one is no page of the pool, as -1, are skipped.  A page may be several times a
    source, but once a destination, and not both.  Counts stay as they are.
    """
    src = _int32(src, "src", (src.numel(),))
    dst = _int32(dst, "dst", (src.numel(),))
    _require_device(pool.refs, src, dst)
    if not src.numel():
        return
    with torch.cuda.device(pool.device):
        _lib.check(_lib.lib.mcq4_kv8_copy_pages(pool._address, src.data_ptr(), dst.data_ptr(), src.numel(), _stream(pool.device)),
                   "mcq4_kv8_copy_pages")


def kv8_fork(pool: KV8Pool, block_table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, release: bool = False
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(block_table, lens)`` of new rows, row i with the pages and length of row ``parents[i]`` (int32 ``[n]``).

    The pages are shared, not copied, and counted for the new rows.  Lengths are given back as 0 to
    ``block_table.shape[1] * page_size``, what a row can hold.  A row whose parent is none of
    the table's, as -1, is empty.  Entries behind a row's pages are -1.  With ``release`` the old
    rows give up theirs, as in a beam search, where the new rows take their place; without,
    both remain.
    """
    if _native is not None:
        pair = _native.kv8_fork(pool, block_table, lens, parents, release)
        if isinstance(pair, int):                # not called again: counts may have changed
            _lib.check(pair, "mcq4_kv8_fork")
        if pair is not None:
            return pair
    table = _table(pool, block_table, False)
    B, W = table.shape
    lens = _int32(lens, "lens", (B,))
    parents = _int32(parents, "parents", (parents.numel(),))
    _require_device(pool.refs, lens, parents)
    n = parents.numel()
    out = torch.full((n, W), -1, dtype=torch.int32, device=pool.device)
    out_lens = torch.zeros(n, dtype=torch.int32, device=pool.device)
    if B and W and (n or release):
        if not n:                                # no new rows: only the old ones' release, by an empty one
            parents = torch.full((1,), -1, dtype=torch.int32, device=pool.device)
            out, out_lens = out.new_empty(1, W), out_lens.new_empty(1)
        with torch.cuda.device(pool.device):
            _lib.check(_lib.lib.mcq4_kv8_fork(pool._address, table.data_ptr(), _row_stride(table), B, W, lens.data_ptr(), parents.data_ptr(),
                                              max(n, 1), out.data_ptr(), out_lens.data_ptr(), int(bool(release)), _stream(pool.device)),
                       "mcq4_kv8_fork")
    return out[:n], out_lens[:n]


def kv8_resize(pool: KV8Pool, block_table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor) -> torch.Tensor:
    """Pages for ``new_lens[b]`` tokens instead of ``lens[b]`` (int32 ``[B]``), in place in ``block_table``.

    Rows that shrink, to 0 if a sequence ends, give back the pages that they no longer use; the
    entries become -1.  Then rows that grow get free pages, the lowest numbers first, in the
    order of rows; and where a row's last page holds tokens but is not full, and other entries name
    it too, a copy of it takes its place, so that what is appended stays the row's own.  Rows do not
    look at each other there: where all that name a page grow, each gets a copy, the last one too, and
    the page becomes free.  Returns
    an int32 ``[1]``: 0, or how many pages were lacking in the pool, in which case no row has grown.

    A row holds ``block_table.shape[1] * page_size`` tokens at most, and lengths beyond that count as that
    (as negative ones count as 0), in ``lens`` and ``new_lens``: 0 is returned for such a row as for a
    full one.  What lies behind has no pages, and ``kv8_append`` drops it.  The width is the host's
    to choose: who lets sequences grow compares their lengths with it.
    """
    if _native is not None:
        missing = _native.kv8_resize(pool, block_table, lens, new_lens)
        if isinstance(missing, int):             # not called again: counts may have changed
            _lib.check(missing, "mcq4_kv8_resize")
        if missing is not None:
            return missing
    table = _table(pool, block_table, True)
    B, W = table.shape
    lens, new_lens = _int32(lens, "lens", (B,)), _int32(new_lens, "new_lens", (B,))
    _require_device(pool.refs, lens, new_lens)
    missing = torch.zeros(1, dtype=torch.int32, device=pool.device)
    if B and W:
        stream = _stream(pool.device)
        need = int(_lib.lib.mcq4_kv8_resize_workspace_bytes(pool._address, B))
        ws = _workspace.get(pool.device, stream, need) if need else None
        with torch.cuda.device(pool.device), _workspace.guard(ws, stream):
            _lib.check(_lib.lib.mcq4_kv8_resize(pool._address, table.data_ptr(), _row_stride(table), B, W, lens.data_ptr(), new_lens.data_ptr(),
                                                missing.data_ptr(), ws.data_ptr() if need else None, ws.numel() if need else 0, stream),
                       "mcq4_kv8_resize")
    return missing


def kv8_compact(pool: KV8Pool, *block_tables: torch.Tensor) -> torch.Tensor:
    """Move the pages in use to the first numbers, codes, scales and counts, and rename them in the tables.

    ``block_tables`` are all tables that name pages of the pool, changed in place.  Pages that
    lie there already stay; the i-th of those behind them goes to the i-th free one.  Returns
    an int32 ``[1]``, the number of pages in use.
    """
    tables = [_table(pool, t, True) for t in block_tables]
    names = torch.empty(pool.num_pages, dtype=torch.int32, device=pool.device)
    live = torch.empty(1, dtype=torch.int32, device=pool.device)
    _require_device(pool.refs)
    stream = _stream(pool.device)
    need = int(_lib.lib.mcq4_kv8_compact_workspace_bytes(pool._address))
    ws = _workspace.get(pool.device, stream, need)
    with torch.cuda.device(pool.device), _workspace.guard(ws, stream):
        _lib.check(_lib.lib.mcq4_kv8_compact(pool._address, names.data_ptr(), live.data_ptr(), ws.data_ptr(), ws.numel(), stream), "mcq4_kv8_compact")
        for t in tables:
            if t.numel():
                _lib.check(_lib.lib.mcq4_kv8_rename(t.data_ptr(), _row_stride(t), *t.shape, names.data_ptr(), pool.num_pages, stream),
                           "mcq4_kv8_rename")
    return live
