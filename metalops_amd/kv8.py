"""A paged key/value cache held in 8 bits, and attention over it, on MI355X.

A page holds ``page_size`` tokens of every key/value head as e4m3 codes with one
power-of-two scale for each head (a byte ``b`` for ``2**(b - 127)``, 255 for NaN).  A block table
``[B, W]`` (int32) names the pages of B sequences: token t of sequence b is slot
``t % page_size`` of page ``block_table[b, t // page_size]``.  Keys lie token by
token, values channel by channel, so that the attention reads both in long pieces
along the axis that it sums over.

No counterpart in the reference.  As in the rest of the package the HIP kernels
of ``libmcq4.so`` do all of it, on the current stream, without a fallback; lengths
and tables stay on the device and nothing waits for them.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .quantization import _DTYPE_CODES, _native, _require_device, _stream, _workspace

__all__ = ["KV8Cache", "kv8_append", "kv8_read", "kv8_attention", "kv8_shared_attention"]


class KV8Cache:
    """The cache's tensors (uint8): ``k_codes [P, H, page, D]``, ``v_codes [P, H, D, page]``,
    ``k_scales [P, H]``, ``v_scales [P, H]``, contiguous, on one device.  ``page`` is 16, 32,
    64, 128 or 256, ``D`` a multiple of 16 up to 256."""

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        if k_codes.dim() != 4:
            raise RuntimeError(f"k_codes must be [P, H, page, D], got shape {tuple(k_codes.shape)}")
        P, H, page, D = k_codes.shape
        for name, t, shape in (("v_codes", v_codes, (P, H, D, page)), ("k_scales", k_scales, (P, H)), ("v_scales", v_scales, (P, H))):
            if tuple(t.shape) != shape:
                raise RuntimeError(f"{name} must be {shape}, got {tuple(t.shape)}")
        if page not in (16, 32, 64, 128, 256):
            raise RuntimeError(f"page size must be 16, 32, 64, 128 or 256, got {page}")
        if D % 16 or not 0 < D <= 256:
            raise RuntimeError(f"head dim must be a multiple of 16 up to 256, got {D}")
        if P == 0 or H == 0:
            raise RuntimeError("the cache must have pages and heads")
        for name, t in (("k_codes", k_codes), ("v_codes", v_codes), ("k_scales", k_scales), ("v_scales", v_scales)):
            if t.dtype != torch.uint8 or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous uint8 tensor")
            if t.device != k_codes.device:
                raise RuntimeError(f"all cache tensors must be on one device, got {k_codes.device} and {t.device}")
        for name, t in (("k_codes", k_codes), ("v_codes", v_codes)):
            if t.data_ptr() % 16:
                raise RuntimeError(f"{name} must be 16-byte aligned")
        self._tensors = (k_codes, v_codes, k_scales, v_scales)   # what _struct points to: not to be replaced
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = P, H, page, D
        self.device = k_codes.device
        self._struct = _lib.Kv8CacheStruct(k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                           P, H, D, page)
        self._address = ctypes.addressof(self._struct)

    k_codes = property(lambda self: self._tensors[0])
    v_codes = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
              device: Union[str, torch.device] = "cuda") -> "KV8Cache":
        """A cache whose pages hold nothing yet."""
        u8 = dict(dtype=torch.uint8, device=device)
        return cls(torch.zeros((num_pages, kv_heads, page_size, head_dim), **u8),
                   torch.zeros((num_pages, kv_heads, head_dim, page_size), **u8),
                   torch.full((num_pages, kv_heads), 127, **u8), torch.full((num_pages, kv_heads), 127, **u8))

    def __repr__(self) -> str:
        return (f"KV8Cache(num_pages={self.num_pages}, kv_heads={self.kv_heads}, head_dim={self.head_dim}, "
                f"page_size={self.page_size}, device={self.device})")


def _int32(t: torch.Tensor, name: str, shape: Tuple[int, ...]) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise RuntimeError(f"{name} must be int32, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise RuntimeError(f"{name} must be {shape}, got {tuple(t.shape)}")
    return t.contiguous()


def _batch(cache: KV8Cache, table: torch.Tensor, lens: torch.Tensor, cu: Optional[torch.Tensor], T: int, lens_name: str):
    """(mcq4_kv8_batch, the tensors it points to)."""
    if table.dim() != 2:
        raise RuntimeError(f"block_table must be [B, W], got shape {tuple(table.shape)}")
    B, W = table.shape
    if table.dtype != torch.int32:
        raise RuntimeError(f"block_table must be int32, got {table.dtype}")
    if W and (table.stride(1) != 1 or table.stride(0) < W):
        table = table.contiguous()
    lens = _int32(lens, lens_name, (B,))
    if cu is not None:
        cu = _int32(cu, "cu_seqlens", (B + 1,))
    elif B and T % B:
        raise RuntimeError(f"without cu_seqlens the {T} tokens must be a multiple of the {B} sequences")
    _require_device(cache.k_codes, table, lens, *([] if cu is None else [cu]))
    st = _lib.Kv8BatchStruct(table.data_ptr(), max(table.stride(0), W), B, W, lens.data_ptr(),
                             None if cu is None else cu.data_ptr(), T)
    return st, (table, lens, cu)


def _tokens(t: torch.Tensor, name: str, heads: Optional[int], D: int, rows16: bool) -> torch.Tensor:
    """``t [T, heads, D]`` with neighbouring channels (rows16: rows at 16-byte aligned addresses)."""
    if t.dim() != 3 or t.shape[2] != D or (heads is not None and t.shape[1] != heads):
        raise RuntimeError(f"{name} must be [T, {heads if heads is not None else 'heads'}, {D}], got shape {tuple(t.shape)}")
    es, (token, head) = t.element_size(), _strides(t)
    if t.stride(2) != 1 or (rows16 and (t.data_ptr() % 16 or token * es % 16 or head * es % 16)):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _strides(t: torch.Tensor) -> Tuple[int, int]:
    """Of tokens and heads; where there is one, its stride is any and not asked for."""
    return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, start_lens: torch.Tensor,
               cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Write new tokens ``k, v [T, H, D]`` (fp32, fp16 or bf16) into the pages, in place.

    Sequence b has ``start_lens[b]`` (int32 ``[B]``) tokens already; its new ones are rows
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` (int32 ``[B + 1]``), or ``T / B`` each without
    ``cu_seqlens``.  A page's scale for a head is the smallest power of two that brings the
    largest finite magnitude of its new tokens to 448, e4m3's largest, or less; a page that
    holds older tokens keeps its scale if that is larger, and has its codes rescaled if
    not.  Infinities and NaN become NaN.  Tokens beyond the table's width, or in an entry that
    names no page, are dropped.  Sequences may share full pages, but not ones that they
    append to.
    """
    if _native is not None and _native.kv8_append(cache, k, v, block_table, start_lens, cu_seqlens):
        return
    H, D = cache.kv_heads, cache.head_dim
    k, v = _tokens(k, "k", H, D, False), _tokens(v, "v", H, D, False)
    if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
        raise RuntimeError(f"k and v must have one length and type, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    if k.dtype not in _DTYPE_CODES:
        raise RuntimeError(f"k and v must be float16, bfloat16 or float32, got {k.dtype}")
    st, keep = _batch(cache, block_table, start_lens, cu_seqlens, k.shape[0], "start_lens")
    _require_device(cache.k_codes, k, v)
    if st.T == 0 or st.batch == 0 or st.width == 0:
        return
    with torch.cuda.device(cache.device):
        _lib.check(_lib.lib.mcq4_kv8_append(cache._address, ctypes.byref(st), k.data_ptr(), *_strides(k),
                                            v.data_ptr(), *_strides(v), _DTYPE_CODES[k.dtype],
                                            _stream(cache.device)),
                   "mcq4_kv8_append")
    del keep


def kv8_read(cache: KV8Cache, block_table: torch.Tensor, context_lens: torch.Tensor,
             dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of each sequence's first ``context_lens[b]`` tokens, ``(k, v)`` of
    ``[B, W * page_size, H, D]`` in ``dtype`` (default bfloat16, which holds them exactly
    down to its subnormals), zeros behind them."""
    if dtype is None:
        dtype = torch.bfloat16
    if _native is not None:
        pair = _native.kv8_read(cache, block_table, context_lens, dtype)
        if pair is not None:
            return pair
    if dtype not in _DTYPE_CODES:
        raise RuntimeError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
    st, keep = _batch(cache, block_table, context_lens, None, 0, "context_lens")
    shape = (st.batch, st.width * cache.page_size, cache.kv_heads, cache.head_dim)
    k = torch.empty(shape, dtype=dtype, device=cache.device)
    v = torch.empty(shape, dtype=dtype, device=cache.device)
    if k.numel():
        with torch.cuda.device(cache.device):
            _lib.check(_lib.lib.mcq4_kv8_read(cache._address, ctypes.byref(st), k.data_ptr(), v.data_ptr(),
                                              _DTYPE_CODES[dtype], _stream(cache.device)),
                       "mcq4_kv8_read")
    del keep
    return k, v


def kv8_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, context_lens: torch.Tensor,
                  cu_seqlens: Optional[torch.Tensor] = None, scale: Optional[float] = None, causal: bool = True,
                  window: int = 0, max_context: Optional[int] = None, return_lse: bool = False
                  ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``softmax(scale * q k^T + mask) v`` for new tokens ``q [T, heads, D]`` (fp16 or bf16).

    ``heads`` is a multiple of the cache's H; query head i reads key/value head
    ``i // (heads / H)``.  Sequence b's new tokens (``cu_seqlens`` as in ``kv8_append``) are the
    last of its ``context_lens[b]`` cached ones.  ``causal``: a token sees none after
    itself; ``window > 0``: only the last ``window`` up to its own position.  A row that
    sees nothing, or that is no sequence's by ``cu_seqlens`` (whose offsets are not to
    fall), is 0.  ``scale`` defaults to ``D ** -0.5``; scores are to stay below 2^29.
    ``max_context``, an upper bound of ``context_lens`` known to the host, sizes the division
    of the work (default: the block table's width).  ``return_lse`` also returns the fp32
    ``[T, heads]`` logarithms of the sums of exponentials, -inf for a row of either kind.
    """
    if scale is None:
        scale = cache.head_dim ** -0.5
    if _native is not None:
        out = _native.kv8_attention(q, cache, block_table, context_lens, cu_seqlens, scale, causal, window, max_context,
                                    return_lse)
        if out is not None:
            return out
    D, H = cache.head_dim, cache.kv_heads
    q = _tokens(q, "q", None, D, True)
    T, heads = q.shape[:2]
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"q must be float16 or bfloat16, got {q.dtype}")
    if heads == 0 or heads % H:
        raise RuntimeError(f"the {heads} heads of q must be a multiple of the cache's {H}")
    if not 0 <= window <= 1 << 30:              # what the C call takes; ctypes would cut a larger one to 32 bits
        raise RuntimeError(f"window must be 0 to 2**30, got {window}")
    if max_context is not None and max_context < 0:
        raise RuntimeError(f"max_context must not be negative, got {max_context}")
    st, keep = _batch(cache, block_table, context_lens, cu_seqlens, T, "context_lens")
    _require_device(cache.k_codes, q)
    out = torch.empty((T, heads, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((T, heads), dtype=torch.float32, device=q.device) if return_lse else None
    if T and (st.batch == 0 or st.width == 0):
        out.zero_()
        if lse is not None:
            lse.fill_(float("-inf"))
    elif T:
        longest = st.width * cache.page_size
        longest = longest if max_context is None else min(longest, int(max_context))
        stream = _stream(q.device)
        need = int(_lib.lib.mcq4_kv8_attention_workspace_bytes(cache._address, ctypes.byref(st), heads, int(causal), int(window),
                                                               longest))
        ws = _workspace.get(q.device, stream, need) if need else None
        with torch.cuda.device(q.device), _workspace.guard(ws, stream):
            _lib.check(_lib.lib.mcq4_kv8_attention(cache._address, ctypes.byref(st), q.data_ptr(), *_strides(q),
                                                   heads, _DTYPE_CODES[q.dtype], out.data_ptr(),
                                                   None if lse is None else lse.data_ptr(), float(scale), int(causal),
                                                   int(window), longest, ws.data_ptr() if need else None,
                                                   ws.numel() if need else 0, stream),
                       "mcq4_kv8_attention")
    del keep
    return (out, lse) if return_lse else out


def kv8_shared_attention(q: torch.Tensor, cache: KV8Cache, prefix_table: torch.Tensor, prefix_lens: torch.Tensor,
                         block_table: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                         groups: Optional[torch.Tensor] = None, scale: Optional[float] = None, max_prefix: Optional[int] = None,
                         max_context: Optional[int] = None, return_lse: bool = False
                         ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``kv8_attention`` (causal) of sequences that share prefixes, whose pages are read once for all of them.

    Prefix s is the first ``prefix_lens[s]`` (int32 ``[S]``) tokens of row s of ``prefix_table [S, W0]``.
    Sequences ``groups[s]`` to ``groups[s + 1] - 1`` (int32 ``[S + 1]``, not falling) share it, or ``B / S``
    each without ``groups``; sequences of no group have no prefix, and none has where offsets in ``groups`` fall or
    leave 0 to B.  (``cu_seqlens`` is not to fall or leave 0 to T, as in ``kv8_attention``: of few new tokens each all rows
    are 0 then.)  A sequence's context is its prefix and then
    the ``context_lens[b]`` tokens that row b of ``block_table`` has of its own, the last of them the new ones
    (``cu_seqlens`` as in ``kv8_append``); both may end inside a page.  With ``kv8_fork``'s tables, whose
    sequences share their first pages, a prefix of full pages is the first columns of one row and
    ``block_table`` the others'.

    A new token sees all of its prefix and its sequence's own tokens up to itself; one that stands
    before its sequence's own context, as where that is 0, is 0, its lse -inf.  Everything else
    is as in ``kv8_attention``.  ``max_prefix`` and ``max_context``, upper bounds of ``prefix_lens`` and
    ``context_lens`` known to the host, size the division of the work (default: the tables' widths).

    Meant for few new tokens a sequence, or a long prefix.  Whole prompts behind a short one are
    faster by ``kv8_attention`` over tables that begin with the prefix's pages (8 prompts of 100 to 499
    tokens, 32 heads over 8 of 128: behind 2048 tokens 162 us against 210, behind 16384 1092 against 845).
    """
    if scale is None:
        scale = cache.head_dim ** -0.5
    if _native is not None:
        out = _native.kv8_shared_attention(q, cache, prefix_table, prefix_lens, block_table, context_lens, cu_seqlens, groups, scale,
                                           max_prefix, max_context, return_lse)
        if out is not None:
            return out
    D, H = cache.head_dim, cache.kv_heads
    q = _tokens(q, "q", None, D, True)
    T, heads = q.shape[:2]
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"q must be float16 or bfloat16, got {q.dtype}")
    if heads == 0 or heads % H:
        raise RuntimeError(f"the {heads} heads of q must be a multiple of the cache's {H}")
    for name, most in (("max_prefix", max_prefix), ("max_context", max_context)):
        if most is not None and most < 0:
            raise RuntimeError(f"{name} must not be negative, got {most}")
    st, keep = _batch(cache, block_table, context_lens, cu_seqlens, T, "context_lens")
    if prefix_table.dim() != 2 or prefix_table.dtype != torch.int32:
        raise RuntimeError(f"prefix_table must be int32 [S, W], got {prefix_table.dtype} {tuple(prefix_table.shape)}")
    S, W = prefix_table.shape
    if W and (prefix_table.stride(1) != 1 or prefix_table.stride(0) < W):
        prefix_table = prefix_table.contiguous()
    prefix_lens = _int32(prefix_lens, "prefix_lens", (S,))
    if groups is not None:
        groups = _int32(groups, "groups", (S + 1,))
    elif S and st.batch % S:
        raise RuntimeError(f"without groups the {st.batch} sequences must be a multiple of the {S} prefixes")
    _require_device(cache.k_codes, q, prefix_table, prefix_lens, *([] if groups is None else [groups]))
    if S == 0 or W == 0 or T == 0 or st.batch == 0 or st.width == 0:
        # No prefix, or nothing of the sequences' own: none of them has a new token that sees one.
        return kv8_attention(q, cache, block_table, context_lens, cu_seqlens, scale, True, 0, max_context, return_lse)
    out = torch.empty((T, heads, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((T, heads), dtype=torch.float32, device=q.device) if return_lse else None
    px = _lib.Kv8PrefixesStruct(prefix_table.data_ptr(), max(prefix_table.stride(0), W), S, W, prefix_lens.data_ptr(),
                                None if groups is None else groups.data_ptr())
    longest = [w * cache.page_size if most is None else min(w * cache.page_size, int(most))
               for w, most in ((W, max_prefix), (st.width, max_context))]
    stream = _stream(q.device)
    need = int(_lib.lib.mcq4_kv8_shared_attention_workspace_bytes(cache._address, ctypes.byref(px), ctypes.byref(st), heads, *longest))
    ws = _workspace.get(q.device, stream, need) if need else None
    with torch.cuda.device(q.device), _workspace.guard(ws, stream):
        _lib.check(_lib.lib.mcq4_kv8_shared_attention(cache._address, ctypes.byref(px), ctypes.byref(st), q.data_ptr(), *_strides(q), heads,
                                                      _DTYPE_CODES[q.dtype], out.data_ptr(), None if lse is None else lse.data_ptr(),
                                                      float(scale), *longest, ws.data_ptr() if need else None, ws.numel() if need else 0,
                                                      stream),
                   "mcq4_kv8_shared_attention")
    del keep
    return (out, lse) if return_lse else out
