"""Paged KV cache: pages of keys and values shared by many sequences, and attention of a ragged batch over them.

:class:`LayerKVCache` (``cache.py``) holds one dense buffer per batch: sequences start and end together, a batch is
padded to its longest one and growing copies it.  Here the keys and values of all sequences live in one pool of pages
of ``page_size`` tokens, ``[num_pages, Hkv, page_size, D]`` per layer (head-major within a page, as the dense cache
is), and a page table names each sequence's pages.  Sequences join and leave at any time, prompts are shared by
:meth:`PagedKVCache.fork`, and one pass may mix decoding sequences with pieces of prompts.

The operators take a ragged batch of new tokens: rows ``q_offsets[b] .. q_offsets[b + 1]`` of a flat token axis
belong to sequence ``b``, which holds ``seq_lens[b]`` tokens, the new ones included; its new token ``i`` of ``n`` is at
position ``seq_lens[b] - n + i``, and token ``p`` lives in page ``page_table[b, p // page_size]``, slot
``p % page_size``.  The three tensors are int32 on the GPU, so a captured CUDA graph serves batches that change in
place.

* :func:`paged_append` writes the new tokens' keys and values into their pages;
* :func:`paged_attention`, :func:`paged_attention_with_lse`, :func:`paged_attend_into` compute their attention::

      out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i),  lse_i = ln sum_j exp(scale q_i k_j)

  over the keys at positions up to the token's own (``causal``) or over all of them.  A token that sees no key gives
  ``out = 0`` and ``lse = -inf``; rows of no sequence are left as they were; slots behind a sequence's length never
  count, whatever they hold, and neither do keys and values that a token does not see.  An infinite value that it sees
  gives that infinity (or NaN, where the kernel's arithmetic has a probability of 0);
* :func:`copy_pages` copies pages in every layer at once.

Nothing here synchronises the host.  Indices that the host cannot see are bounded on the device: a page table entry
outside the pool reads as zeros and is not written, a length that the table cannot hold is cut, and
:func:`device_status <collaborative_edge_system_b200._lib.device_status>` then returns ``DEV_BAD_PAGE`` or
``DEV_BAD_BATCH`` until it is cleared.
"""

from __future__ import annotations

import ctypes
import math
import struct
from collections import Counter
from operator import index
from typing import Dict, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib
from .attention import accumulation_dtype

Indices = Union[torch.Tensor, Sequence[int]]


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than a call needs; the cache is as it was before the call."""


# ------------------------------------------------------------------------------------------------ operators
def _check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor) -> None:
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must both be "
                         "[num_pages, Hkv, page_size, D] of one dtype")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        if k_pages.shape[3] > 1:
            raise ValueError("pages must be contiguous along the head dimension")


def _check_batch(page_table: torch.Tensor, seq_lens: torch.Tensor, q_offsets: torch.Tensor) -> None:
    i32 = torch.int32
    if page_table.dtype != i32 or seq_lens.dtype != i32 or q_offsets.dtype != i32:
        raise ValueError("page_table, seq_lens and q_offsets must be int32")
    table, lens, offsets = page_table.shape, seq_lens.shape, q_offsets.shape
    if len(table) != 2 or len(lens) != 1 or len(offsets) != 1 or table[0] != lens[0] or offsets[0] != lens[0] + 1:
        raise ValueError(f"page_table {tuple(table)}, seq_lens {tuple(lens)} and q_offsets {tuple(offsets)} must be "
                         "[B, max_pages], [B] and [B + 1]")
    if seq_lens.stride(0) != 1 or q_offsets.stride(0) != 1 or page_table.stride(1) != 1:
        if (lens[0] > 1 and seq_lens.stride(0) != 1) or (lens[0] > 0 and q_offsets.stride(0) != 1) or (
                table[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table rows, seq_lens and q_offsets must be contiguous")


def _checked(k_pages, v_pages, page_table, seq_lens, q_offsets):
    """Pages' shape and strides, ``B``, ``max_pages`` and the table's row stride, all checked (what is as usual at once,
    the rest by the functions above)."""
    i32 = torch.int32
    pages, kp, vp = k_pages.shape, k_pages.stride(), v_pages.stride()
    table, ts, (B,) = page_table.shape, page_table.stride(), seq_lens.shape[:1] or (0,)
    if not (len(pages) == 4 and pages == v_pages.shape and k_pages.dtype == v_pages.dtype and kp[3] == 1 and vp[3] == 1):
        _check_pages(k_pages, v_pages)
    if not (page_table.dtype == i32 and seq_lens.dtype == i32 and q_offsets.dtype == i32 and len(table) == 2
            and table[0] == B and ts[1] == 1 and seq_lens.stride() == (1,) and q_offsets.stride() == (1,)
            and q_offsets.shape[0] == B + 1):
        _check_batch(page_table, seq_lens, q_offsets)
    return pages, kp, vp, B, table[1], ts[0]


def _record(layout: struct.Struct, *values) -> bytes:
    try:
        return layout.pack(*values)
    except struct.error as e:  # a count, size or scale that is no number of its field
        raise ValueError(f"an argument or a size does not fit the call: {e}") from None


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, seq_lens: torch.Tensor, q_offsets: torch.Tensor) -> None:
    """Write the new tokens' ``k`` / ``v`` (``[T, Hkv, D]``, any token and head strides) into their pages, bit for bit.

    Two tokens with one place (a page that two of the batch's sequences write) leave any mix of their rows' parts there;
    :class:`PagedKVCache` makes no such batch.
    """
    dev = _lib.device_number(k, v, k_pages, v_pages, page_table, seq_lens, q_offsets)
    pages, kp, vp, B, width, table = _checked(k_pages, v_pages, page_table, seq_lens, q_offsets)
    P, H, ps, D = pages
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if len(shape) != 3 or shape != v.shape or shape[1] != H or shape[2] != D:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [T, {H}, {D}]")
    if k.dtype != k_pages.dtype or v.dtype != v_pages.dtype:
        raise ValueError("k, v and the pages must share a dtype")
    if D > 1 and (ks[2] != 1 or vs[2] != 1):
        raise ValueError("k and v must be contiguous along the head dimension")
    _lib.paged_append(_lib.PagedAppendParams.from_buffer_copy(_record(
        _lib.PAGED_APPEND_RECORD, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), q_offsets.data_ptr(),
        seq_lens.data_ptr(), page_table.data_ptr(), ks[0], ks[1], vs[0], vs[1], kp[0], kp[1], kp[2], vp[0], vp[1], vp[2],
        table, B, shape[0], H, D, ps, P, width, k.element_size())), dev)


_TAIL = bytes(ctypes.sizeof(_lib.PagedAttnParams) - _lib.PAGED_ATTN_RECORD.size)  # the workspace's fields


def _attn_params(q, k_pages, v_pages, page_table, seq_lens, q_offsets, out, lse, min_q_len, max_q_len, causal, scale):
    pages, kp, vp, B, width, table = _checked(k_pages, v_pages, page_table, seq_lens, q_offsets)
    shape, dtype, qs, os = q.shape, q.dtype, q.stride(), out.stride()
    if len(shape) != 3 or dtype != k_pages.dtype:
        raise ValueError(f"q must be [T, Hq, D] of the pages' dtype, got {tuple(shape)} of {dtype}")
    T, Hq, D = shape
    P, H, ps, Dk = pages
    if Dk != D:
        raise ValueError(f"q {tuple(shape)} and the pages {tuple(k_pages.shape)} disagree on the head dim")
    if out.shape != shape or (lse is not None and (lse.dim() != 2 or lse.shape[0] != Hq or lse.shape[1] != T)):
        raise ValueError(f"out must be {tuple(shape)} and lse [{Hq}, {T}]")
    if D > 1 and (qs[2] != 1 or os[2] != 1):
        raise ValueError("q and out must be contiguous along the head dimension")
    if lse is None:
        lp, l0, l1 = 0, 0, 0
    else:
        if lse.dtype != accumulation_dtype(dtype):
            raise ValueError(f"lse must be {accumulation_dtype(dtype)} for {dtype} inputs")
        lp, (l0, l1) = lse.data_ptr(), lse.stride()
    return _lib.PagedAttnParams.from_buffer_copy(_record(
        _lib.PAGED_ATTN_RECORD, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), lp, q_offsets.data_ptr(),
        seq_lens.data_ptr(), page_table.data_ptr(), qs[0], qs[1], kp[0], kp[1], kp[2], vp[0], vp[1], vp[2], os[0], os[1],
        l0, l1, table, B, T, Hq, H, D, ps, P, width, min_q_len,
        max(T, min_q_len) if max_q_len is None else max_q_len,
        1.0 / math.sqrt(max(D, 1)) if scale is None else scale, bool(causal), _lib.dtype_code(dtype),
        _lib.dtype_code(out.dtype)) + _TAIL)


def paged_attend_into(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                      seq_lens: torch.Tensor, q_offsets: torch.Tensor, out: torch.Tensor,
                      lse: Optional[torch.Tensor] = None, *, min_q_len: int = 0, max_q_len: Optional[int] = None,
                      causal: bool = True, scale: Optional[float] = None) -> None:
    """Attention of the new tokens ``q`` ``[T, Hq, D]`` into preallocated ``out`` (``q.dtype`` or the accumulation
    dtype) and, if given, ``lse`` ``[Hq, T]`` (accumulation dtype).

    ``min_q_len`` and ``max_q_len`` bound the number of new tokens of the sequences that have any; they choose the
    kernels and are promises (0 and ``None`` always hold): decoding sequences (up to 8 or 16 query rows per KV head)
    and chunks of prompts have a kernel each, and a batch that cannot hold one kind does not launch its kernel.

    16-bit inputs: the kernels differ in what is left of a probability when it is multiplied with the values, so a
    sequence's result differs within the following with the bounds given and with the other sequences of the call.  The
    decoding kernel keeps it to 2^-17 (bf16) or 2^-22 (f16), the chunk kernel rounds it to the input type (half a step,
    2^-8 or 2^-11), as the dense prefill kernel does; the CUDA cores, which take the shapes outside both, keep fp32.  In
    f16 no kernel loses more of a key than 2^-39 (decoding) or 2^-32 (chunks) of its row's largest probability.
    9 to 16 query rows at 128 columns go to the chunk kernel where ``min_q_len`` says that no sequence has fewer, and
    to the decoding kernel where it does not.
    """
    if lse is None:
        _lib.device_number(q, k_pages, v_pages, page_table, seq_lens, q_offsets, out)
    else:
        _lib.device_number(q, k_pages, v_pages, page_table, seq_lens, q_offsets, out, lse)
    _lib.paged_attn(_attn_params(q, k_pages, v_pages, page_table, seq_lens, q_offsets, out, lse, min_q_len, max_q_len,
                                 causal, scale), q)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, q_offsets: torch.Tensor, *, min_q_len: int = 0,
                    max_q_len: Optional[int] = None, causal: bool = True, scale: Optional[float] = None
                    ) -> torch.Tensor:
    """Attention output ``[T, Hq, D]`` in ``q.dtype`` (:func:`paged_attend_into`); rows of no sequence are zero."""
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    paged_attend_into(q, k_pages, v_pages, page_table, seq_lens, q_offsets, out, min_q_len=min_q_len,
                      max_q_len=max_q_len, causal=causal, scale=scale)
    return out


def paged_attention_with_lse(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                             seq_lens: torch.Tensor, q_offsets: torch.Tensor, *, min_q_len: int = 0,
                             max_q_len: Optional[int] = None, causal: bool = True, scale: Optional[float] = None
                             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(out [T, Hq, D], lse [Hq, T])`` in accumulation precision; rows of no sequence are 0 and ``-inf``.

    With a leading dimension of 1 they are partials for :func:`merge_attention`: ranks that hold different tokens of
    the sequences in their pages merge their results exactly.
    """
    acc = accumulation_dtype(q.dtype)
    out = torch.zeros(q.shape, dtype=acc, device=q.device)
    lse = torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=acc, device=q.device)
    paged_attend_into(q, k_pages, v_pages, page_table, seq_lens, q_offsets, out, lse, min_q_len=min_q_len,
                      max_q_len=max_q_len, causal=causal, scale=scale)
    return out, lse


def _host_indices(x: Indices) -> torch.Tensor:
    if isinstance(x, torch.Tensor):
        if x.dtype == torch.int32 and x.is_contiguous() and x.dim() == 1 and x.device.type == "cpu":
            return x
        if x.device.type != "cpu" or x.dim() != 1:
            raise ValueError("page indices are a sequence of numbers or a 1-D tensor on the CPU")
        if x.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"page indices must be whole numbers, got {x.dtype}")
    else:
        x = torch.tensor([index(i) for i in x], dtype=torch.int64)
    if x.dtype == torch.int64:
        if x.numel() and (int(x.min()) < 0 or int(x.max()) >= 1 << 31):
            raise ValueError("page index out of range")
        x = x.to(torch.int32)
    return x.contiguous()


def _page_block(pages: torch.Tensor) -> Tuple[int, int, int]:
    """``(layer stride, page stride, page elements)`` of ``[L, P, H, ps, D]`` pages, each of which must be one block
    of memory (in any order of its dimensions)."""
    if pages.is_contiguous():
        return pages.stride(0), pages.stride(1), pages.stride(1)
    n = 1
    for size, stride in sorted(zip(pages.shape[2:], pages.stride()[2:]), key=lambda x: x[1]):
        if size > 1:
            if stride != n:
                raise ValueError("each page must be one contiguous block")
            n *= size
    if pages.shape[1] > 1 and abs(pages.stride(1)) < n:
        raise ValueError("pages overlap")
    return pages.stride(0), pages.stride(1), n


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: Indices, dst: Indices) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` of both pools, ``[num_pages, Hkv, page_size, D]`` or with a leading
    layer dimension, all layers in one launch.  The indices are on the host; a destination may neither repeat nor be a
    source (``ValueError``, and nothing is copied)."""
    dev = _lib.device_number(k_pages, v_pages)
    if k_pages.dim() not in (4, 5) or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} must both be "
                         "[num_pages, Hkv, page_size, D] or [layers, num_pages, Hkv, page_size, D] of one dtype")
    if k_pages.dim() == 4:
        k_pages, v_pages = k_pages.unsqueeze(0), v_pages.unsqueeze(0)
    s, d = _host_indices(src), _host_indices(dst)
    if s.shape != d.shape:
        raise ValueError(f"{s.numel()} sources and {d.numel()} destinations")
    kl, kp, n = _page_block(k_pages)
    vl, vp, _ = _page_block(v_pages)
    size = k_pages.element_size()
    _lib.copy_pages(_lib.CopyPagesParams(
        k_pages.data_ptr(), v_pages.data_ptr(), (kl * size, kp * size), (vl * size, vp * size), n * size, s.data_ptr(),
        d.data_ptr(), s.numel(), k_pages.shape[0], k_pages.shape[1]), dev)


# ------------------------------------------------------------------------------------------------ the cache
class PageAllocator:
    """Pages of one pool with reference counts (host only).  The lowest free page is handed out first.  A call that is
    refused changes nothing."""

    def __init__(self, num_pages: int) -> None:
        if num_pages < 0:
            raise ValueError("num_pages must be >= 0")
        self.refs = [0] * num_pages
        self._free = list(range(num_pages - 1, -1, -1))  # descending: the lowest is popped

    @property
    def num_free(self) -> int:
        return len(self._free)

    def _used(self, pages: Sequence[int], times: int = 1) -> None:
        """Every page is of the pool and has at least ``times`` owners for each time that it stands in ``pages``."""
        for p, n in Counter(pages).items():
            if not 0 <= p < len(self.refs):
                raise ValueError(f"no page {p} in a pool of {len(self.refs)}")
            if self.refs[p] < max(1, times * n):
                raise ValueError(f"page {p} is free" if self.refs[p] < 1 else f"page {p} has {self.refs[p]} owners")

    def alloc(self, count: int) -> List[int]:
        if count < 0:
            raise ValueError("count must be >= 0")
        if count > len(self._free):
            raise OutOfPages(f"{count} pages needed, {len(self._free)} of {len(self.refs)} free")
        pages = [self._free.pop() for _ in range(count)]
        for p in pages:
            self.refs[p] = 1
        return pages

    def share(self, pages: Sequence[int]) -> None:
        self._used(pages, 0)
        for p in pages:
            self.refs[p] += 1

    def release(self, pages: Sequence[int]) -> None:
        self._used(pages)
        freed = []
        for p in pages:
            self.refs[p] -= 1
            if self.refs[p] == 0:
                freed.append(p)
        if freed:
            self._free = sorted(self._free + freed, reverse=True)

    def compaction(self) -> Tuple[List[int], List[int]]:
        """``(src, dst)``: the pages in use behind the first ``used`` ones, and the free pages before that they move to."""
        used = len(self.refs) - len(self._free)
        src = [p for p in range(used, len(self.refs)) if self.refs[p]]
        return src, sorted(p for p in self._free if p < used)

    def move(self, src: Sequence[int], dst: Sequence[int]) -> None:
        self._used(src)
        if len(src) != len(dst) or len(set(src)) != len(src) or len(set(dst)) != len(dst) or not set(dst) <= set(self._free):
            raise ValueError("pages in use move to as many free ones, each of them once")
        for s, d in zip(src, dst):
            self.refs[d], self.refs[s] = self.refs[s], 0
        self._free = [p for p in range(len(self.refs) - 1, -1, -1) if not self.refs[p]]


class PagedBatch:
    """A ragged batch of new tokens: the device tensors that the operators take, and what the host knows of it."""

    def __init__(self, tables: Sequence[Sequence[int]], lengths: Sequence[int], counts: Sequence[int],
                 device: torch.device) -> None:
        B, width = len(counts), max([len(t) for t in tables] + [1])
        T = int(sum(counts))
        host = np.full(2 * T + B * width + 2 * B + 1, -1, dtype=np.int32)
        at = [2 * T, 2 * T + B * width, 2 * T + B * width + B, 2 * T + B * width + 2 * B + 1]
        pos = host[: at[0]].view(np.int64)
        table, lens, offs = host[at[0] : at[1]].reshape(B, width), host[at[1] : at[2]], host[at[2] : at[3]]
        offs[0] = row = 0
        for b in range(B):
            n, total = counts[b], lengths[b]
            table[b, : len(tables[b])] = tables[b]
            lens[b] = total
            pos[row : row + n] = np.arange(total - n, total)
            row += n
            offs[b + 1] = row
        staged = torch.from_numpy(host)
        if device.type == "cuda":  # one copy from pinned memory, ordered with the current stream's work
            staged = staged.pin_memory().to(device, non_blocking=True)
        self.positions = staged[: at[0]].view(torch.int64)  # [T]
        self.page_table = staged[at[0] : at[1]].view(B, width)
        self.seq_lens = staged[at[1] : at[2]]
        self.q_offsets = staged[at[2] : at[3]]
        self.num_tokens = T
        some = [n for n in counts if n > 0]
        self.min_q_len, self.max_q_len = (min(some), max(some)) if some else (0, 0)
        self.last_rows = [int(o) - 1 for o in np.cumsum(counts)]  # row of each sequence's last new token


class PagedKVCache:
    """Keys and values of many sequences in one pool of pages per layer, ``k`` / ``v``
    ``[layers, num_pages, Hkv, page_size, D]``.

    Page tables, lengths and reference counts are kept on the host, so no call waits for the GPU.  A pass over the
    model goes: :meth:`extend` reserves the new tokens' places and describes the batch, then per layer :meth:`append`
    and :meth:`attend`.  All work is queued on the current stream: one stream (or streams ordered by the caller) uses
    a cache.
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device) -> None:
        if num_layers < 1 or page_size < 1 or num_kv_heads < 1 or head_dim < 1:
            raise ValueError("layers, page size, heads and head dim must be >= 1")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"the paged cache lives in device memory, got {device} (there is no CPU path)")
        self.page_size = page_size
        self.pool = PageAllocator(num_pages)
        self._pages: Dict[int, List[int]] = {}
        self._lengths: Dict[int, int] = {}
        self._next = 0
        self._make_buffers((num_layers, num_pages, num_kv_heads, page_size, head_dim), dtype, device)

    def _make_buffers(self, shape, dtype: torch.dtype, device: torch.device) -> None:
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.device = self.k.device

    def _copy(self, src: List[int], dst: List[int]) -> None:
        if src:
            copy_pages(self.k, self.v, src, dst)

    # ------------------------------------------------------------------ sequences
    def add(self) -> int:
        """A new empty sequence's id."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lengths[seq] = [], 0
        return seq

    def length(self, seq: int) -> int:
        return self._lengths[self._known(seq)]

    def pages(self, seq: int) -> List[int]:
        return list(self._pages[self._known(seq)])

    def _known(self, seq: int) -> int:
        if seq not in self._lengths:
            raise ValueError(f"no sequence {seq} in the cache")
        return seq

    @property
    def num_free_pages(self) -> int:
        return self.pool.num_free

    def nbytes(self) -> int:
        """Bytes of K and V of the pages in use."""
        used = len(self.pool.refs) - self.pool.num_free
        return 2 * used * self.k.element_size() * (self.k.numel() // max(1, self.k.shape[1]))

    def fork(self, seq: int, length: Optional[int] = None, count: int = 1) -> List[int]:
        """``count`` new sequences that begin with the first ``length`` tokens of ``seq`` (all of them by default).

        Full pages are shared; a partly filled last page is copied for each fork, in all layers by one launch."""
        n = self.length(seq) if length is None else index(length)
        if n < 0 or n > self.length(seq):
            raise ValueError(f"{n} tokens of a sequence that has {self.length(seq)}")
        if count < 0:
            raise ValueError("count must be >= 0")
        full, partly = divmod(n, self.page_size)
        shared = self._pages[seq][:full]
        tails = self.pool.alloc(count) if partly else []
        if tails:
            self._copy([self._pages[seq][full]] * len(tails), tails)
        new = []
        for i in range(count):
            self.pool.share(shared)
            s = self.add()
            self._pages[s], self._lengths[s] = shared + tails[i : i + 1], n
            new.append(s)
        return new

    def free(self, seq: int) -> None:
        """Forget a sequence; pages that no other one shares become free."""
        self.pool.release(self._pages[self._known(seq)])
        del self._pages[seq], self._lengths[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Keep the first ``length`` tokens (rejected proposals leave, their pages become free)."""
        length = index(length)
        if length < 0 or length > self.length(seq):
            raise ValueError(f"{length} tokens of a sequence that has {self.length(seq)}")
        keep = -(-length // self.page_size)
        self.pool.release(self._pages[seq][keep:])
        self._pages[seq] = self._pages[seq][:keep]
        self._lengths[seq] = length

    def compact(self) -> int:
        """Move pages from the end of the pool into free ones before them, so that the pages in use are the first
        ones; returns how many those are.  Page tables made before the call are out of date after it."""
        src, dst = self.pool.compaction()
        self._copy(src, dst)
        to = dict(zip(src, dst))
        for seq, pages in self._pages.items():
            self._pages[seq] = [to.get(p, p) for p in pages]
        self.pool.move(src, dst)
        return len(self.pool.refs) - self.pool.num_free

    # ------------------------------------------------------------------ passes
    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> PagedBatch:
        """Reserve places for ``counts[i]`` new tokens of ``seqs[i]`` and describe the pass.

        A partly filled last page that another sequence shares (after :meth:`truncate`) is copied first, so that no
        sequence ever writes what another one reads.  Raises :class:`OutOfPages` and changes nothing when the pool
        does not have the pages."""
        seqs, counts = list(seqs), [index(c) for c in counts]
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("extend takes each sequence once, with a count >= 0 for each")
        ps = self.page_size
        need, split = 0, []
        writers: Dict[int, int] = {}  # shared page -> sequences of this call that write it
        for s, c in zip(seqs, counts):
            n = self.length(s)
            need += -(-(n + c) // ps) - len(self._pages[s])
            if c and n % ps and self.pool.refs[self._pages[s][-1]] > 1:
                split.append(s)
                writers[self._pages[s][-1]] = writers.get(self._pages[s][-1], 0) + 1
        # where all owners of a page split from it in one call, the last of them keeps the page itself
        fresh = self.pool.alloc(need + sum(min(n, self.pool.refs[p] - 1) for p, n in writers.items()))
        src, dst = [], []
        for s in split:
            old = self._pages[s][-1]
            if self.pool.refs[old] == 1:
                continue
            self.pool.release([old])
            self._pages[s][-1] = fresh.pop()
            src.append(old)
            dst.append(self._pages[s][-1])
        self._copy(src, dst)
        for s, c in zip(seqs, counts):
            self._lengths[s] += c
            grow = -(-self._lengths[s] // ps) - len(self._pages[s])
            self._pages[s] += [fresh.pop() for _ in range(grow)]
        return PagedBatch([self._pages[s] for s in seqs], [self._lengths[s] for s in seqs], counts, self.device)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, batch: PagedBatch) -> None:
        """The new tokens' ``k`` / ``v`` ``[T, Hkv, D]`` of one layer into the pages."""
        if k.shape[:1] != (batch.num_tokens,):
            raise ValueError(f"k {tuple(k.shape)} for a batch of {batch.num_tokens} new tokens")
        paged_append(k, v, self.k[layer], self.v[layer], batch.page_table, batch.seq_lens, batch.q_offsets)

    def attend(self, layer: int, q: torch.Tensor, batch: PagedBatch, *, causal: bool = True,
               scale: Optional[float] = None) -> torch.Tensor:
        """Attention ``[T, Hq, D]`` of the new tokens over one layer's pages, theirs (appended before) included."""
        if q.shape[:1] != (batch.num_tokens,):
            raise ValueError(f"q {tuple(q.shape)} for a batch of {batch.num_tokens} new tokens")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        paged_attend_into(q, self.k[layer], self.v[layer], batch.page_table, batch.seq_lens, batch.q_offsets, out,
                          min_q_len=batch.min_q_len, max_q_len=batch.max_q_len, causal=causal, scale=scale)
        return out


__all__ = ["OutOfPages", "PageAllocator", "PagedBatch", "PagedKVCache", "copy_pages", "paged_append",
           "paged_attend_into", "paged_attention", "paged_attention_with_lse"]
