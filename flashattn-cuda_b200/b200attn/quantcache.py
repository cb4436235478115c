"""Paged KV cache held in 4 or 8 bits: write, read back, attend, select pages.

`QuantCache` is the storage (one tensor of packed blocks, and an optional
index of page bounds); `append_paged_quant`, `read_paged_quant`,
`decode_paged_quant` and `select_pages` are the operators over it, with the
block table and lengths that `append_paged` / `decode_paged` take.
`QuantPagePool` adds the host-side page allocator of `PagePool`.

A serving step over a quantised cache:

    append_paged_quant(k_new, v_new, cache, block_table, kv_lens)
    O, L = decode_paged_quant(q, cache, block_table, kv_lens)

and for long contexts, reading only the pages that matter to the query (the
cache needs an index):

    pages = select_pages(q, cache, block_table, kv_lens, top_k=128)
    O, L = decode_paged_quant(q, cache, block_table, kv_lens, pages=pages)

The formats and the arithmetic are specified in include/b200attn.h.  The
reference has no KV cache; the decode math is its online softmax
(cuda/flash_attn_fa3_db_full.cu:250-300).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import List, Optional

import torch

from . import _lib
from .attention import _DT, _decode_q, _fastcall, _ptr, _stream
from .kvcache import PagePool

GROUP = 64  # channels that share one (scale, min)


_BLOCK_BYTES = {}


def _fit(*ints):
    """Refuse what a C int does not hold (ctypes would drop its upper bits)."""
    for x in ints:
        if not -1 << 31 <= x < 1 << 31:
            raise RuntimeError(f"{x} does not fit in 32 bits")


def block_bytes(head_dim: int, page_size: int, bits: int) -> int:
    """Bytes of one (page, KV head) block."""
    n = _BLOCK_BYTES.get((head_dim, page_size, bits))
    if n is None:
        _fit(head_dim, page_size, bits)
        n = _lib.load().b2a_kvq_block_bytes(head_dim, page_size, bits)
        if n == 0:
            raise RuntimeError("head_dim must be 64 or 128, page_size 16, 32 or 64 and bits 4 or 8")
        _BLOCK_BYTES[head_dim, page_size, bits] = n
    return n


def _strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def _append_ct(k, v, data, index, index_scale, *rest):
    _fit(*rest[2:12])
    return _lib.load().b2a_kvq_append_paged(k, v, _strides(*rest[13:16]), _strides(*rest[16:]),
                                            data, index, index_scale, *rest[:13])


def _read_ct(*args):
    _fit(*args[6:16])
    return _lib.load().b2a_kvq_read_paged(*args)


def _select_ct(q, *rest):
    _fit(*rest[6:15])
    return _lib.load().b2a_kvq_select_pages(q, _strides(*rest[16:]), *rest[:16])


def _decode_ct(q, *rest):
    _fit(rest[4], *rest[8:18])
    return _lib.load().b2a_kvq_decode_paged(q, _strides(*rest[19:21]), *rest[:18], rest[21],
                                            rest[18])


_append, _read, _select, _decode = _append_ct, _read_ct, _select_ct, _decode_ct
if hasattr(_fastcall, "kvq_append"):  # the CPython binding: the same calls, cheaper to make
    _append, _read = _fastcall.kvq_append, _fastcall.kvq_read
    _select, _decode = _fastcall.kvq_select, _fastcall.kvq_decode


class QuantCache:
    """Storage of a quantised paged KV cache.

    data: uint8 [P, Hkv, block_bytes]; index: int8 [P, Hkv, 2, D] with
    index_scale fp32 [P, Hkv], or both None for a cache without an index.
    dtype is that of the keys and values written and read (float16 or bfloat16).
    """

    __slots__ = ("data", "index", "index_scale", "page_size", "head_dim", "bits", "dtype",
                 "device", "num_pages", "num_kv_heads")

    def __init__(self, data: torch.Tensor, *, page_size: int, head_dim: int, bits: int,
                 dtype: torch.dtype, index: Optional[torch.Tensor] = None,
                 index_scale: Optional[torch.Tensor] = None):
        if dtype not in _DT:
            raise RuntimeError("dtype must be torch.float16 or torch.bfloat16")
        shape = data.shape
        if (len(shape) != 3 or data.dtype is not torch.uint8 or not data.is_contiguous()
                or shape[2] != block_bytes(head_dim, page_size, bits)):
            raise RuntimeError("data must be contiguous uint8 [P, Hkv, block_bytes]")
        self.num_pages, self.num_kv_heads, _ = shape
        self.device = data.device
        if (index is None) != (index_scale is None):
            raise RuntimeError("index and index_scale must be given together")
        if index is not None:
            P, Hkv, _ = shape
            if (index.shape != (P, Hkv, 2, head_dim) or index.dtype is not torch.int8
                    or index_scale.shape != (P, Hkv) or index_scale.dtype is not torch.float32
                    or not (index.is_contiguous() and index_scale.is_contiguous())
                    or index.device != self.device or index_scale.device != self.device):
                raise RuntimeError("index must be contiguous int8 [P, Hkv, 2, D] and index_scale "
                                   "fp32 [P, Hkv] on data's device")
        self.data, self.index, self.index_scale = data, index, index_scale
        self.page_size, self.head_dim, self.bits, self.dtype = page_size, head_dim, bits, dtype

    @classmethod
    def empty(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
              bits: int = 4, dtype: torch.dtype = torch.float16, index: bool = False,
              device="cuda") -> "QuantCache":
        """A cache of `num_pages` pages that all read back as zero."""
        data = torch.zeros(num_pages, num_kv_heads, block_bytes(head_dim, page_size, bits),
                           dtype=torch.uint8, device=device)
        idx = sc = None
        if index:
            idx = torch.zeros(num_pages, num_kv_heads, 2, head_dim, dtype=torch.int8,
                              device=device)
            sc = torch.zeros(num_pages, num_kv_heads, dtype=torch.float32, device=device)
        return cls(data, page_size=page_size, head_dim=head_dim, bits=bits, dtype=dtype,
                   index=idx, index_scale=sc)

    def codes(self, side: int) -> torch.Tensor:
        """View of the K (0) or V (1) codes: uint8 [P, Hkv, page_size, D*bits/8]."""
        row = self.head_dim * self.bits // 8
        n = self.page_size * row
        return self.data[..., side * n:(side + 1) * n].unflatten(-1, (self.page_size, row))

    def params(self, side: int) -> torch.Tensor:
        """View of the K (0) or V (1) params: dtype [P, Hkv, page_size, D/64, 2] (scale, min)."""
        groups = self.head_dim // GROUP
        n = self.page_size * groups * 4
        at = 2 * self.page_size * (self.head_dim * self.bits // 8) + side * n
        return self.data[..., at:at + n].view(self.dtype).unflatten(-1, (self.page_size, groups, 2))


def _check_table(cache: QuantCache, block_table: torch.Tensor, rows: torch.Tensor, what: str,
                 extra: int = 0):
    """(B, max_pages) of block_table int32 [B, max_pages], with `rows` int32 [B + extra], both
    contiguous and on the cache's device."""
    dev = cache.device
    if dev.type != "cuda":
        raise RuntimeError("the cache must be on a CUDA device")
    shape = block_table.shape
    if (len(shape) != 2 or block_table.dtype is not torch.int32
            or not block_table.is_contiguous() or block_table.device != dev):
        raise RuntimeError("block_table must be contiguous int32 [B, max_pages] on the cache's device")
    if (rows.dim() != 1 or rows.shape[0] != shape[0] + extra or rows.dtype is not torch.int32
            or not rows.is_contiguous() or rows.device != dev):
        raise RuntimeError(f"{what} must be contiguous int32 [{shape[0] + extra}] on the cache's "
                           "device (block_table has one row per sequence)")
    return shape


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_no_guard = contextlib.nullcontext()


def _guard(device: torch.device):
    """Device guard, nothing where `device` is current (these calls are a few microseconds)."""
    return _no_guard if device.index == _current_device() else torch.cuda.device(device)


def _rows_of(t: torch.Tensor, n: int):
    """t, or a copy where its rows are not contiguous or not 16-byte aligned, and the element
    strides of its first n dims; a dim of size 1 has stride 0."""
    if not t.data_ptr() & 15:
        shape = t.shape
        if t.is_contiguous():
            d = shape[-1]
            if n == 2:
                return t, (shape[1] * d, d)
            return t, (shape[1] * shape[2] * d, shape[2] * d, d)
        st = t.stride()
        st = [0 if k == 1 else s for k, s in zip(shape, st)]
        if st[n] == 1 and not any(s & 7 for s in st[:n]):
            return t, st[:n]
    t = t.clone(memory_format=torch.contiguous_format)
    return _rows_of(t, n)


def append_paged_quant(k_new: torch.Tensor, v_new: torch.Tensor, cache: QuantCache,
                       block_table: torch.Tensor, kv_lens: torch.Tensor,
                       advance: bool = True) -> None:
    """Quantise k_new, v_new [B, Hkv, T, D] (cache.dtype, any strides) and write them at
    positions kv_lens[b] + t of the sequences in block_table (b2a_kvq_append_paged); with
    `advance`, kv_lens += T on the device (a negative length stays, its tokens are dropped).
    Updates the index of a cache that has one.
    No page may be owned by two of the sequences that write to it."""
    shape = k_new.shape
    if len(shape) != 4 or shape != v_new.shape:
        raise RuntimeError("k_new and v_new must both be [B, Hkv, T, D]")
    B, Hkv, T, D = shape
    if Hkv != cache.num_kv_heads or D != cache.head_dim:
        raise RuntimeError("k_new must match the cache's KV heads and head dim")
    if k_new.dtype is not cache.dtype or v_new.dtype is not cache.dtype:
        raise RuntimeError("k_new and v_new must have the cache's dtype")
    rows, max_pages = _check_table(cache, block_table, kv_lens, "kv_lens")
    dev = cache.device
    if k_new.device != dev or v_new.device != dev:
        raise RuntimeError("k_new and v_new must be on the cache's device")
    if rows != B:
        raise RuntimeError("block_table must have one row per sequence")
    if B == 0 or T == 0:
        return
    with _guard(dev):
        kn, ks = _rows_of(k_new, 3)
        vn, vs = _rows_of(v_new, 3)
        _lib.check(_append(
            kn.data_ptr(), vn.data_ptr(), cache.data.data_ptr(), _ptr(cache.index),
            _ptr(cache.index_scale), block_table.data_ptr(), kv_lens.data_ptr(), B, Hkv, T, D,
            cache.page_size, max_pages, cache.num_pages, cache.bits, _DT[cache.dtype],
            int(bool(advance)), _stream(dev), *ks, *vs))


def read_paged_quant(cache: QuantCache, block_table: torch.Tensor, cu_seqlens: torch.Tensor,
                     total: int, max_len: int, start: Optional[torch.Tensor] = None,
                     out=None) -> list:
    """Read tokens back: [K, V], each [total, Hkv, D] in cache.dtype, packed token-major as
    forward_varlen takes them.  Sequence b's tokens start[b] .. (None: from 0), as many as
    cu_seqlens[b+1] - cu_seqlens[b] (int32 [B+1], device), go to rows cu_seqlens[b] .. ;
    total = cu_seqlens[B] and max_len, a bound of every length, are host numbers.
    `out` = (K, V) to write into; rows that no sequence owns are left as they were."""
    B, max_pages = _check_table(cache, block_table, cu_seqlens, "cu_seqlens", 1)
    if start is not None:
        _check_table(cache, block_table, start, "start")
    dev = cache.device
    shape = (int(total), cache.num_kv_heads, cache.head_dim)
    if shape[0] < 0 or max_len < 0:
        raise RuntimeError("total and max_len must be >= 0")
    if out is not None:
        K, V = out
        for t in (K, V):
            if (t.shape != shape or t.dtype != cache.dtype or not t.is_contiguous()
                    or t.device != dev):
                raise RuntimeError("out must be two contiguous [total, Hkv, D] tensors of the "
                                   "cache's dtype on its device")
    with _guard(dev):
        if out is None:
            K = cache.data.new_empty(*shape, dtype=cache.dtype)
            V = cache.data.new_empty(*shape, dtype=cache.dtype)
        if B > 0 and total > 0 and max_len > 0:
            _lib.check(_read(
                cache.data.data_ptr(), block_table.data_ptr(), _ptr(start),
                cu_seqlens.data_ptr(), K.data_ptr(), V.data_ptr(), B, shape[1], shape[2],
                cache.page_size, max_pages, cache.num_pages, shape[0], int(min(max_len, total)),
                cache.bits, _DT[cache.dtype], _stream(dev)))
    return [K, V]


def _check_query(q: torch.Tensor, cache: QuantCache):
    """(q as [B, H, D], whether it had a length dim, B, H, D)."""
    q3, had_len = _decode_q(q)
    if not q3.is_cuda or q3.device != cache.device:
        raise RuntimeError("q must be a CUDA tensor on the cache's device")
    if q3.dtype is not cache.dtype:
        raise RuntimeError("q must have the cache's dtype")
    B, H, D = q3.shape
    if D != cache.head_dim or H == 0 or H % cache.num_kv_heads != 0:
        raise RuntimeError("q must be [B, H, D] with the cache's head dim and H a multiple of Hkv")
    return q3, had_len, B, H, D


@functools.lru_cache(maxsize=256)
def _keys_words(B: int, Hkv: int, max_pages: int) -> int:
    """Words of scratch that a selection needs."""
    return _lib.load().b2a_kvq_select_keys_words(B, Hkv, max_pages)


def select_pages(q: torch.Tensor, cache: QuantCache, block_table: torch.Tensor,
                 kv_lens: torch.Tensor, top_k: int) -> torch.Tensor:
    """The top_k pages of every (sequence, KV head) for the queries q [B, H, D] (or
    [B, H, 1, D]): int32 [B, Hkv, top_k], logical page numbers, ascending, -1 behind the
    last.  A page's score is an upper bound, from the cache's index, of its keys' products
    with the group's query heads, in 8 bits (b2a_kvq_select_pages).  Groups of up to 8 heads."""
    q3, _, B, H, D = _check_query(q, cache)
    if cache.index is None:
        raise RuntimeError("select_pages needs a cache with an index")
    if not 0 < top_k < 1 << 31:
        raise RuntimeError("top_k must be > 0 and < 2^31")
    rows, max_pages = _check_table(cache, block_table, kv_lens, "kv_lens")
    if rows != B:
        raise RuntimeError("block_table must have one row per sequence")
    dev, Hkv = cache.device, cache.num_kv_heads
    with _guard(dev):
        pages = kv_lens.new_empty(B, Hkv, int(top_k))
        if B == 0:
            return pages
        words = _keys_words(B, Hkv, max_pages)
        keys = kv_lens.new_empty(words) if words else None
        qc, qs = _rows_of(q3, 2)
        _lib.check(_select(
            qc.data_ptr(), cache.index.data_ptr(), cache.index_scale.data_ptr(),
            block_table.data_ptr(), kv_lens.data_ptr(), _ptr(keys), pages.data_ptr(), B, H,
            Hkv, D, cache.page_size, max_pages, cache.num_pages, int(top_k), _DT[cache.dtype],
            _stream(dev), *qs))
    return pages


@functools.lru_cache(maxsize=256)
def _plan(B: int, H: int, Hkv: int, D: int, bits: int, max_tokens: int, splits):
    """(warps that share a decode, floats of its workspace): functions of the sizes alone."""
    lib = _lib.load()
    if splits is not None:
        _fit(int(splits) * B * Hkv)
    workers = (lib.b2a_kvq_decode_workers(B, Hkv, D, bits, max_tokens) if splits is None
               else int(splits) * B * Hkv)
    return workers, max(lib.b2a_kvq_decode_workspace_floats(B, H, Hkv, D, workers), 1)


def decode_paged_quant(q: torch.Tensor, cache: QuantCache, block_table: torch.Tensor,
                       kv_lens: torch.Tensor, scale: Optional[float] = None,
                       pages: Optional[torch.Tensor] = None,
                       splits: Optional[int] = None) -> list:
    """Decode attention over a quantised cache: [O, L] shaped like q ([B, H, D] or
    [B, H, 1, D], H / Hkv at most 8); kv_lens may hold zeros (O = 0, L = -inf).  `pages` int32 [B, Hkv, n]
    (from select_pages) restricts each KV head to those pages; negative entries are skipped.
    `splits` overrides the number of warps that share the work, as a multiple of B * Hkv."""
    q3, had_len, B, H, D = _check_query(q, cache)
    rows, max_pages = _check_table(cache, block_table, kv_lens, "kv_lens")
    if rows != B:
        raise RuntimeError("block_table must have one row per sequence")
    dev, Hkv = cache.device, cache.num_kv_heads
    n_pages = 0
    if pages is not None:
        shape = pages.shape
        if (len(shape) != 3 or shape[0] != B or shape[1] != Hkv or shape[2] == 0
                or pages.dtype is not torch.int32 or not pages.is_contiguous()
                or pages.device != dev):
            raise RuntimeError("pages must be contiguous int32 [B, Hkv, n] on the cache's device")
        n_pages = shape[2]
    with _guard(dev):
        O = q3.new_empty(B, H, D)
        L = q3.new_empty(B, H, dtype=torch.float32)
        if B > 0:
            workers, floats = _plan(B, H, Hkv, D, cache.bits,
                                    (n_pages or max_pages) * cache.page_size, splits)
            ws = L.new_empty(floats)
            qc, qs = _rows_of(q3, 2)
            _lib.check(_decode(
                qc.data_ptr(), cache.data.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(),
                _ptr(pages), n_pages, ws.data_ptr(), O.data_ptr(), L.data_ptr(), B, H, Hkv, D,
                cache.page_size, max_pages, cache.num_pages, workers, cache.bits,
                _DT[cache.dtype], _stream(dev), *qs,
                float(D) ** -0.5 if scale is None else float(scale)))
    if had_len:
        return [O.unsqueeze(2), L.unsqueeze(2)]
    return [O, L]


class QuantPagePool(PagePool):
    """PagePool over a QuantCache: the same allocator (reserve / release / lengths), with
    `append` quantising, and `read`, `decode` over the sequences it holds.

    index=True keeps the page bounds that decode(top_k=...) selects by.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 max_seqs: int, max_pages: int, dtype=torch.float16, device="cuda",
                 bits: int = 4, index: bool = False):
        self._bits, self._index = bits, index
        super().__init__(num_pages, page_size, num_kv_heads, head_dim, max_seqs, max_pages,
                         dtype, device)

    def _make_storage(self, num_pages, page_size, num_kv_heads, head_dim, dtype, device):
        self.cache = QuantCache.empty(num_pages, page_size, num_kv_heads, head_dim, self._bits,
                                      dtype, self._index, device)

    def _write(self, k_new, v_new, block_table, kv_lens):
        append_paged_quant(k_new, v_new, self.cache, block_table, kv_lens, advance=True)

    def _rows(self, seqs: Optional[List[int]], n: int):
        """(block table rows, lengths) of `seqs` (default 0..n-1)."""
        seqs = list(range(n)) if seqs is None else list(seqs)
        if seqs == list(range(len(seqs))):
            return seqs, self.block_table[:len(seqs)], self.kv_lens[:len(seqs)]
        idx = torch.tensor(seqs, dtype=torch.long, device=self.kv_lens.device)
        return seqs, self.block_table[idx], self.kv_lens[idx]

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, seqs: Optional[List[int]] = None):
        """Quantise and append k_new, v_new [B, Hkv, T, D] to `seqs` (default 0..B-1), each
        sequence at most once."""
        if seqs is not None:
            seqs = [range(len(self._lens))[s] for s in seqs]  # -1 and its positive name are one
            if len(set(seqs)) != len(seqs):
                raise RuntimeError("a sequence may appear only once in one append")
        super().append(k_new, v_new, seqs)

    def read(self, seqs: Optional[List[int]] = None) -> list:
        """[K, V, cu_seqlens, max_len] of the whole of `seqs` (default: all), as
        forward_varlen takes them."""
        seqs, bt, _ = self._rows(seqs, len(self._lens))
        lens = [self._lens[s] for s in seqs]
        cu = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32)
        cu = cu.to(self.kv_lens.device)
        most = max(lens, default=0)
        K, V = read_paged_quant(self.cache, bt, cu, sum(lens), most)
        return [K, V, cu, most]

    def decode(self, q: torch.Tensor, seqs: Optional[List[int]] = None,
               scale: Optional[float] = None, top_k: Optional[int] = None) -> list:
        """[O, L] of the queries q [B, H, D], one per sequence of `seqs` (default 0..B-1);
        with top_k over that many pages of each KV head only.  The table is cut to the pages
        that the sequences have now: a captured step is decode_paged_quant over `block_table`
        and `kv_lens`, whose width does not change."""
        seqs, bt, lens = self._rows(seqs, q.shape[0])
        most = max((len(self._pages[s]) for s in seqs), default=0)
        bt = bt[:, :max(most, 1)].contiguous()  # the widest sequence's pages: fewer empty splits
        pages = None if top_k is None else select_pages(q, self.cache, bt, lens, top_k)
        return decode_paged_quant(q, self.cache, bt, lens, scale=scale, pages=pages)
