"""Sparse attention over a paged KV cache on gfx950, and eviction of its pages.

A page is cut into blocks of consecutive tokens; ``bounds`` keeps every block's channel-wise minimum and maximum key
(rounded outward to bf16 where it holds more bits, in an INT8 cache). One decode step of a layer is then::

    store_paged_kv_bounds(k, v, kv_cache, bounds, cache_location)          # the new tokens
    scores = paged_block_scores(q, bounds, indptr, indices, last, page)    # an upper bound of q . k per block
    blocks = paged_select_blocks(scores, indptr, last, page, block, n)     # the n best blocks per sequence and KV head
    out = paged_decode_blocks(q, kv_cache, indptr, indices, last, blocks, block, weights_in=w, weights=w)

after a prefill chunk ``paged_key_bounds`` computes the bounds of its blocks, and ``paged_evict_pages`` cuts a page table
down to the pages that received the most attention (``w``). Caches are those of paged_decode (bf16), paged_decode_fp8
(u8 / float8_e4m3fn with ``kv_scale``) and paged_decode_i8 (int8 with ``kv_scales``), page tables theirs too. Nothing is
read back to the host, so a step can be captured in a HIP graph. Contract violations raise ValueError.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib


# The checks build their messages only when they fail, and the stream comes straight from torch's extension module: a
# decode step makes these calls once a layer. (Looked up in the call, as a torch built without a GPU has no such function.)
_BF16, _F32, _I32, _I8, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int8, torch.uint8
_E4M3 = torch.float8_e4m3fn
_DT_BF16, _DT_E4M3 = _lib.DT_BF16, _lib.DT_FP8E4M3


def _call(name: str, tensors, *args) -> None:
    """The call on the current stream of the tensors' device, which all of them have to be on."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name}: tensors on {tensors[0].device} and {t.device}")
    if dev < 0:  # the host
        raise ValueError(f"axk operators take device tensors; got a tensor on {tensors[0].device}")
    c = torch._C
    if c._cuda_getDevice() == dev:
        _lib.call(name, *args, c._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, c._cuda_getCurrentRawStream(dev))


def _i32(t: torch.Tensor, name: str, *shape: int) -> None:
    if t.dtype is not _I32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 {list(shape)}")


def _table(indptr, last_page_len, indices=None) -> int:
    """Checks a page table and returns its sequences."""
    b = last_page_len.numel()
    if b < 1:
        raise ValueError("the page table holds no sequence")
    _i32(indptr, "indptr", b + 1)
    _i32(last_page_len, "last_page_len", b)
    if indices is not None and (indices.dtype is not _I32 or indices.dim() != 1 or not indices.is_contiguous()):
        raise ValueError("indices must be contiguous int32 [nnz]")
    return b


def _status(status) -> None:
    if status is not None and (status.dtype is not _I32 or status.numel() < 1):
        raise ValueError("status must be int32 [1]")


def _sizes(page_size: int, block_size: int) -> None:
    if page_size < 16 or page_size % 16 or page_size > 4096:
        raise ValueError(f"page_size {page_size} must be a multiple of 16, at most 4096")
    if block_size < 16 or block_size % 16 or page_size % block_size:
        raise ValueError(f"block_size {block_size} must be a multiple of 16 that divides page_size {page_size}")


def _cache(kv_cache, kv_scale, kv_scales):
    """(entry suffix, arguments naming the stored type, num_pages, page_size, HKV, D) of a bf16, FP8 or INT8 cache."""
    dtype, shape = kv_cache.dtype, kv_cache.shape
    if len(shape) != 5 or shape[1] != 2 or not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous [pages, 2, page_size, HKV, D]")
    p, _, page, hkv, d = shape
    if d != 256 and d != 128 and d != 64:
        raise ValueError(f"head_dim {d} not supported (64, 128, 256)")
    if p < 1:
        raise ValueError("kv_cache holds no page")
    if kv_scale is not None and (dtype is _BF16 or dtype is _I8):
        raise ValueError("kv_scale is for an FP8 cache")
    if kv_scales is not None and dtype is not _I8:
        raise ValueError("kv_scales are for an INT8 cache")
    if dtype is _BF16:
        return "", (_DT_BF16, 1.0), p, page, hkv, d
    if dtype is _I8:
        if (kv_scales is None or kv_scales.dtype is not _BF16 or kv_scales.shape != (p, 2, page, hkv)
                or not kv_scales.is_contiguous()):
            raise ValueError(f"an INT8 cache needs its kv_scales, contiguous bf16 [{p}, 2, {page}, {hkv}]")
        return "_i8", (kv_scales.data_ptr(),), p, page, hkv, d
    if dtype is not _U8 and dtype is not _E4M3:
        raise ValueError(f"kv_cache must be bfloat16, u8 / float8_e4m3fn or int8, got {dtype}")
    if kv_scale is None or not kv_scale > 0 or math.frexp(kv_scale)[0] != 0.5:
        raise ValueError(f"an FP8 cache needs its kv_scale, a power of two (got {kv_scale})")
    return "", (_DT_E4M3, kv_scale), p, page, hkv, d


def _bounds(bounds, p: int, hkv: int, d: int, page_size: int) -> int:
    """Checks the bounds of a pool and returns the block size they are for."""
    shape = bounds.shape
    bpp = shape[1] if len(shape) == 5 else 0
    if bpp < 1 or page_size % bpp or shape != (p, bpp, hkv, 2, d) or bounds.dtype is not _BF16 or not bounds.is_contiguous():
        raise ValueError(f"bounds must be contiguous bf16 [{p}, page_size / block_size, {hkv}, 2, {d}], "
                         f"got {tuple(shape)} {bounds.dtype}")
    block = page_size // bpp
    _sizes(page_size, block)
    return block


def _heads(hq: int, hkv: int) -> None:
    if hkv < 1 or hq < 1 or hq % hkv or hq // hkv > 16:
        raise ValueError(f"num_qo_heads {hq} must be a multiple (<= 16x) of num_kv_heads {hkv}")


def store_paged_kv_bounds(
    k: torch.Tensor,
    v: torch.Tensor,
    kv_cache: torch.Tensor,
    bounds: torch.Tensor,
    cache_location: torch.Tensor,
    kv_scale: Optional[float] = None,
    status: Optional[torch.Tensor] = None,
    kv_scales: Optional[torch.Tensor] = None,
) -> None:
    """store_paged_kv / store_paged_kv_fp8 / store_paged_kv_i8 that also folds each new key into its block's bounds, in
    one launch: k, v [rows, HKV, D] bf16 go to cache_location[r] = (page, slot). bounds [P, page / block, HKV, 2, D] bf16,
    in place: a block whose first slot is written starts afresh, any other is widened. Rows of one call may share a block
    (draft rows); where two name one slot the last is stored."""
    kind, stored, p, page, hkv, d = _cache(kv_cache, kv_scale, kv_scales)
    block = _bounds(bounds, p, hkv, d, page)
    shape = k.shape
    rows = shape[0] if shape else 0
    if (shape != (rows, hkv, d) or v.shape != shape or k.dtype is not _BF16 or v.dtype is not _BF16
            or not k.is_contiguous() or not v.is_contiguous()):
        raise ValueError(f"k and v must be contiguous bf16 [rows, {hkv}, {d}]")
    _i32(cache_location, "cache_location", rows, 2)
    _status(status)
    if rows:
        _call("axk_paged_kv_write_bounds" + kind, (k, v, kv_cache, kv_scales, bounds, cache_location, status), k.data_ptr(),
              v.data_ptr(), kv_cache.data_ptr(), *stored, bounds.data_ptr(), cache_location.data_ptr(), rows, hkv, d, page,
              block, p, _lib.ptr(status))


def paged_key_bounds(
    kv_cache: torch.Tensor,
    bounds: torch.Tensor,
    indptr: torch.Tensor,
    indices: torch.Tensor,
    last_page_len: torch.Tensor,
    start: Optional[torch.Tensor] = None,
    kv_scale: Optional[float] = None,
    status: Optional[torch.Tensor] = None,
    kv_scales: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The bounds of the page table's blocks from the cache, in place: of the blocks that hold a token at or after
    start[b] (int32 [B], the position a prefill chunk began at), or of all. Returns bounds."""
    kind, stored, p, page, hkv, d = _cache(kv_cache, kv_scale, kv_scales)
    block = _bounds(bounds, p, hkv, d, page)
    b = _table(indptr, last_page_len, indices)
    if start is not None:
        _i32(start, "start", b)
    _status(status)
    _call("axk_paged_key_bounds" + kind, (kv_cache, kv_scales, bounds, indptr, indices, last_page_len, start, status),
          kv_cache.data_ptr(), *stored, bounds.data_ptr(), indptr.data_ptr(), indices.data_ptr(),
          last_page_len.data_ptr(), _lib.ptr(start), indices.numel(), b, hkv, d, page, block, p, _lib.ptr(status))
    return bounds


def paged_block_scores(
    q: torch.Tensor,
    bounds: torch.Tensor,
    indptr: torch.Tensor,
    indices: torch.Tensor,
    last_page_len: torch.Tensor,
    page_size: int,
    output: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """f32 [HKV, nnz * page_size / block_size]: for each KV head and block of the page table, the largest
    sum_d max(q_d lo_d, q_d hi_d) over the KV head's queries of q [B, HQ, D] bf16, which no q . k in the block
    exceeds. -inf past a sequence's end. Entry e's blocks are columns e * page_size / block_size onwards."""
    b = _table(indptr, last_page_len, indices)
    shape = q.shape
    if len(shape) != 3 or shape[0] != b or q.dtype is not _BF16 or not q.is_contiguous():
        raise ValueError(f"q must be contiguous bf16 [{b}, HQ, D]")
    _, hq, d = shape
    if d not in (64, 128, 256):
        raise ValueError(f"head_dim {d} not supported (64, 128, 256)")
    if bounds.dim() != 5 or bounds.shape[0] < 1:
        raise ValueError("bounds must be bf16 [P, page_size / block_size, HKV, 2, D]")
    p, bpp, hkv = bounds.shape[:3]
    block = _bounds(bounds, p, hkv, d, page_size)
    _heads(hq, hkv)
    n = indices.numel() * bpp
    if output is None:
        output = q.new_empty((hkv, n), dtype=torch.float32)
    elif output.shape != (hkv, n) or output.dtype is not _F32 or not output.is_contiguous():
        raise ValueError(f"output must be contiguous float32 [{hkv}, {n}]")
    _status(status)
    _call("axk_paged_block_scores", (q, bounds, indptr, indices, last_page_len, output, status), q.data_ptr(),
          bounds.data_ptr(), indptr.data_ptr(), indices.data_ptr(), last_page_len.data_ptr(), output.data_ptr(),
          indices.numel(), b, hq, hkv, d, page_size, block, p, _lib.ptr(status))
    return output


def paged_select_blocks(
    scores: torch.Tensor,
    indptr: torch.Tensor,
    last_page_len: torch.Tensor,
    page_size: int,
    block_size: int,
    num_select: int,
    first: int = 1,
    keep_last: int = 1,
    output: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """int32 [B, HKV, num_select]: the blocks with the largest scores (as paged_block_scores lays them out) of each
    sequence and KV head, in ascending order, the first `first` and last `keep_last` blocks always among them; equal
    scores by the lowest block, NaN above every number; -1 behind the blocks of a shorter sequence."""
    b = _table(indptr, last_page_len)
    _sizes(page_size, block_size)
    if (scores.dim() != 2 or scores.dtype is not _F32 or not scores.is_contiguous() or scores.shape[0] < 1
            or scores.shape[1] % (page_size // block_size)):
        raise ValueError("scores must be contiguous float32 [HKV, nnz * page_size / block_size]")
    if first < 0 or keep_last < 0 or num_select < 1 or first + keep_last > num_select:
        raise ValueError(f"num_select {num_select} must be positive and at least first {first} + keep_last {keep_last}")
    hkv = scores.shape[0]
    if output is None:
        output = scores.new_empty((b, hkv, num_select), dtype=torch.int32)
    else:
        _i32(output, "output", b, hkv, num_select)
    _call("axk_paged_select_blocks", (scores, indptr, last_page_len, output), scores.data_ptr(), indptr.data_ptr(),
          last_page_len.data_ptr(), output.data_ptr(), scores.shape[1] // (page_size // block_size), b, hkv, page_size,
          block_size, num_select, first, keep_last)
    return output


def paged_decode_blocks_workspace(batch: int, num_qo_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                                  nnz: int, device, block_size: int = 16, num_select: int = 0,
                                  weights: bool = False) -> torch.Tensor:
    """A byte buffer large enough for paged_decode_blocks with this configuration (num_select 0: every block)."""
    n = _lib.load().axk_paged_decode_blocks_workspace_size(batch, num_qo_heads, num_kv_heads, head_dim, page_size, nnz,
                                                           block_size, num_select, int(weights))
    return torch.empty(n, dtype=torch.uint8, device=device)


def paged_decode_blocks(
    q: torch.Tensor,
    kv_cache: torch.Tensor,
    indptr: torch.Tensor,
    indices: torch.Tensor,
    last_page_len: torch.Tensor,
    blocks: Optional[torch.Tensor] = None,
    block_size: Optional[int] = None,
    sm_scale: Optional[float] = None,
    output: Optional[torch.Tensor] = None,
    weights_in: Optional[torch.Tensor] = None,
    weights: Optional[torch.Tensor] = None,
    decay: float = 1.0,
    kv_scale: Optional[float] = None,
    workspace: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
    kv_scales: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """paged_decode / paged_decode_fp8 / paged_decode_i8 over the listed blocks of each sequence and KV head: blocks int32
    [B, HKV, n], strictly ascending block numbers within the sequence, then -1 (as paged_select_blocks returns them), of
    block_size tokens; None: every block. q [B, HQ, D] bf16; returns bf16 [B, HQ, D], zeros where nothing is attended.

    weights f32 [HKV, nnz], if given, is set to decay * weights_in (zero without weights_in; weights_in may be weights)
    plus the attention that each page-table entry's tokens received, summed over the KV head's queries."""
    b = _table(indptr, last_page_len, indices)
    kind, stored, p, page, hkv, d = _cache(kv_cache, kv_scale, kv_scales)
    shape = q.shape
    if len(shape) != 3 or shape[0] != b or shape[2] != d or q.dtype is not _BF16 or not q.is_contiguous():
        raise ValueError(f"q must be contiguous bf16 [{b}, HQ, {d}]")
    hq, nnz, n = shape[1], indices.numel(), 0
    _heads(hq, hkv)
    if blocks is not None:
        if block_size is None:
            raise ValueError("blocks need their block_size")
        if blocks.dim() != 3 or blocks.shape[2] < 1:
            raise ValueError(f"blocks must be int32 [{b}, {hkv}, n]")
        n = blocks.shape[2]
        _i32(blocks, "blocks", b, hkv, n)
    else:
        block_size = 16
    _sizes(page, block_size)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    if output is None:
        output = torch.empty_like(q)
    elif output.shape != shape or output.dtype is not _BF16 or not output.is_contiguous():
        raise ValueError(f"output must be contiguous bf16 [{b}, {hq}, {d}]")
    if weights is None and weights_in is not None:
        raise ValueError("weights_in without weights")
    for t in (weights_in, weights):
        if t is not None and (t.dtype is not _F32 or t.shape != (hkv, nnz) or not t.is_contiguous()):
            raise ValueError(f"weights_in and weights must be contiguous float32 [{hkv}, {nnz}]")
    _status(status)
    if workspace is None:
        workspace = paged_decode_blocks_workspace(b, hq, hkv, d, page, nnz, q.device, block_size, n, weights is not None)
    elif workspace.dtype is not _U8 or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous uint8")
    _call("axk_paged_decode_blocks" + kind,
          (q, kv_cache, kv_scales, indptr, indices, last_page_len, blocks, output, weights_in, weights, status, workspace),
          q.data_ptr(), kv_cache.data_ptr(), *stored, indptr.data_ptr(), indices.data_ptr(), last_page_len.data_ptr(),
          _lib.ptr(blocks), block_size, n, output.data_ptr(), _lib.ptr(weights_in), _lib.ptr(weights), decay, nnz, b, hq,
          hkv, d, page, p, sm_scale, _lib.ptr(status), workspace.data_ptr(), workspace.numel())
    return output


def paged_evict_pages(
    weights: torch.Tensor,
    indptr: torch.Tensor,
    indices: torch.Tensor,
    budget: int,
    first: int = 1,
    keep_last: int = 1,
):
    """Cuts every sequence of more than `budget` pages down to the `budget` pages of largest weight (weights f32 [HKV, nnz]
    of paged_decode_blocks, summed over the KV heads; equal sums by the lowest place), the first `first` and last
    `keep_last` (>= 1) pages always among them. Returns (indptr [B + 1], indices [nnz], weights [HKV, nnz], freed [nnz]):
    the kept pages in their order with their weights, then -1 and 0, and the other pages' ids, then -1. last_page_len,
    the cache and the bounds stay as they are. A page that several sequences hold is freed for each that drops it."""
    b = indptr.numel() - 1
    if b < 1:
        raise ValueError("the page table holds no sequence")
    _i32(indptr, "indptr", b + 1)
    if indices.dtype is not _I32 or indices.dim() != 1 or not indices.is_contiguous():
        raise ValueError("indices must be contiguous int32 [nnz]")
    nnz = indices.numel()
    if (weights.dim() != 2 or weights.shape[0] < 1 or weights.shape[1] != nnz or weights.dtype is not _F32
            or not weights.is_contiguous()):
        raise ValueError(f"weights must be contiguous float32 [HKV, {nnz}]")
    if first < 0 or keep_last < 1 or first + keep_last > budget:
        raise ValueError(f"budget {budget} must hold first {first} (>= 0) + keep_last {keep_last} (>= 1) pages")
    out = (torch.empty_like(indptr), torch.empty_like(indices), torch.empty_like(weights), torch.empty_like(indices))
    _call("axk_paged_evict_pages", (weights, indptr, indices, *out), weights.data_ptr(), indptr.data_ptr(),
          indices.data_ptr(), *(t.data_ptr() for t in out), nnz, b, weights.shape[0], budget, first, keep_last)
    return out
