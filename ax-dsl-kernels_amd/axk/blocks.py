"""Sparse attention over a paged KV cache on gfx950, and eviction of its pages.

A page is cut into blocks of consecutive tokens; ``bounds`` keeps every block's channel-wise minimum and maximum key. One
decode step of a layer is then::

    store_paged_kv_bounds(k, v, kv_cache, bounds, cache_location)          # the new tokens
    scores = paged_block_scores(q, bounds, indptr, indices, last, page)    # an upper bound of q . k per block
    blocks = paged_select_blocks(scores, indptr, last, page, block, n)     # the n best blocks per sequence and KV head
    out = paged_decode_blocks(q, kv_cache, indptr, indices, last, blocks, block, weights_in=w, weights=w)

after a prefill chunk ``paged_key_bounds`` computes the bounds of its blocks, and ``paged_evict_pages`` cuts a page table
down to the pages that received the most attention (``w``). Caches are those of paged_decode (bf16) and paged_decode_fp8
(u8 / float8_e4m3fn with ``kv_scale``), page tables theirs too. Nothing is read back to the host, so a step can be
captured in a HIP graph. Contract violations raise ValueError.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _call(name: str, tensors, *args) -> None:
    """The call on the current stream of the tensors' device, which all of them have to be on."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: tensors on {dev} and {t.device}")
    if dev.type != "cuda":
        raise ValueError(f"axk operators take device tensors; got a tensor on {dev}")
    if torch.cuda.current_device() == dev.index:
        _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)


def _i32(t: torch.Tensor, name: str, *shape: int) -> None:
    _check(t.dtype == torch.int32 and tuple(t.shape) == shape and t.is_contiguous(),
           f"{name} must be contiguous int32 {list(shape)}")


def _table(indptr, last_page_len, indices=None) -> int:
    """Checks a page table and returns its sequences."""
    b = last_page_len.numel()
    _check(b > 0, "the page table holds no sequence")
    _i32(indptr, "indptr", b + 1)
    _i32(last_page_len, "last_page_len", b)
    if indices is not None:
        _check(indices.dtype == torch.int32 and indices.dim() == 1 and indices.is_contiguous(),
               "indices must be contiguous int32 [nnz]")
    return b


def _status(status) -> None:
    _check(status is None or (status.dtype == torch.int32 and status.numel() >= 1), "status must be int32 [1]")


def _sizes(page_size: int, block_size: int) -> None:
    _check(page_size >= 16 and page_size % 16 == 0 and page_size <= 4096,
           f"page_size {page_size} must be a multiple of 16, at most 4096")
    _check(block_size >= 16 and block_size % 16 == 0 and page_size % block_size == 0,
           f"block_size {block_size} must be a multiple of 16 that divides page_size {page_size}")


def _cache(kv_cache, kv_scale):
    """(dtype code, scale, num_pages, page_size, HKV, D) of a bf16 or FP8 cache."""
    if kv_cache.dtype == torch.bfloat16:
        _check(kv_scale is None, "kv_scale is for an FP8 cache")
        code, scale = _lib.DT_BF16, 1.0
    else:
        _check(kv_cache.dtype in (torch.uint8, torch.float8_e4m3fn),
               f"kv_cache must be bfloat16 or u8 / float8_e4m3fn, got {kv_cache.dtype}")
        _check(kv_scale is not None and kv_scale > 0 and math.frexp(kv_scale)[0] == 0.5,
               f"an FP8 cache needs its kv_scale, a power of two (got {kv_scale})")
        code, scale = _lib.DT_FP8E4M3, float(kv_scale)
    _check(kv_cache.dim() == 5 and kv_cache.shape[1] == 2 and kv_cache.is_contiguous(),
           "kv_cache must be contiguous [pages, 2, page_size, HKV, D]")
    p, _, page, hkv, d = kv_cache.shape
    _check(d in (64, 128, 256), f"head_dim {d} not supported (64, 128, 256)")
    _check(p > 0, "kv_cache holds no page")
    return code, scale, p, page, hkv, d


def _bounds(bounds, p: int, hkv: int, d: int, page_size: int) -> int:
    """Checks the bounds of a pool and returns the block size they are for."""
    _check(bounds.dim() == 5 and bounds.dtype == torch.bfloat16 and bounds.is_contiguous() and bounds.shape[1] > 0
           and page_size % bounds.shape[1] == 0 and bounds.shape[0] == p and tuple(bounds.shape[2:]) == (hkv, 2, d),
           f"bounds must be contiguous bf16 [{p}, page_size / block_size, {hkv}, 2, {d}], got {tuple(bounds.shape)}")
    block = page_size // bounds.shape[1]
    _sizes(page_size, block)
    return block


def _heads(hq: int, hkv: int) -> None:
    _check(hkv > 0 and hq % hkv == 0 and hq // hkv <= 16,
           f"num_qo_heads {hq} must be a multiple (<= 16x) of num_kv_heads {hkv}")


def store_paged_kv_bounds(
    k: torch.Tensor,
    v: torch.Tensor,
    kv_cache: torch.Tensor,
    bounds: torch.Tensor,
    cache_location: torch.Tensor,
    kv_scale: Optional[float] = None,
    status: Optional[torch.Tensor] = None,
) -> None:
    """store_paged_kv / store_paged_kv_fp8 that also folds each new key into its block's bounds, in one launch: k, v
    [rows, HKV, D] bf16 go to cache_location[r] = (page, slot). bounds [P, page / block, HKV, 2, D] bf16, in place: a
    block whose first slot is written starts afresh, any other is widened. Rows of one call may share a block (draft
    rows); where two name one slot the last is stored."""
    code, scale, p, page, hkv, d = _cache(kv_cache, kv_scale)
    block = _bounds(bounds, p, hkv, d, page)
    _check(k.dim() == 3 and k.shape == v.shape and tuple(k.shape[1:]) == (hkv, d) and k.dtype == torch.bfloat16
           and v.dtype == torch.bfloat16 and k.is_contiguous() and v.is_contiguous(),
           f"k and v must be contiguous bf16 [rows, {hkv}, {d}]")
    rows = k.shape[0]
    _i32(cache_location, "cache_location", rows, 2)
    _status(status)
    if rows:
        _call("axk_paged_kv_write_bounds", (k, v, kv_cache, bounds, cache_location, status), k.data_ptr(), v.data_ptr(),
              kv_cache.data_ptr(), code, scale, bounds.data_ptr(), cache_location.data_ptr(), rows, hkv, d, page, block, p,
              _lib.ptr(status))


def paged_key_bounds(
    kv_cache: torch.Tensor,
    bounds: torch.Tensor,
    indptr: torch.Tensor,
    indices: torch.Tensor,
    last_page_len: torch.Tensor,
    start: Optional[torch.Tensor] = None,
    kv_scale: Optional[float] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The bounds of the page table's blocks from the cache, in place: of the blocks that hold a token at or after
    start[b] (int32 [B], the position a prefill chunk began at), or of all. Returns bounds."""
    code, scale, p, page, hkv, d = _cache(kv_cache, kv_scale)
    block = _bounds(bounds, p, hkv, d, page)
    b = _table(indptr, last_page_len, indices)
    if start is not None:
        _i32(start, "start", b)
    _status(status)
    _call("axk_paged_key_bounds", (kv_cache, bounds, indptr, indices, last_page_len, start, status), kv_cache.data_ptr(),
          code, scale, bounds.data_ptr(), indptr.data_ptr(), indices.data_ptr(), last_page_len.data_ptr(),
          _lib.ptr(start), indices.numel(), b, hkv, d, page, block, p, _lib.ptr(status))
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
    sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d over the KV head's queries of q [B, HQ, D] bf16, which no q . k in the block
    exceeds. -inf past a sequence's end. Entry e's blocks are columns e * page_size / block_size onwards."""
    b = _table(indptr, last_page_len, indices)
    _check(q.dim() == 3 and q.shape[0] == b and q.dtype == torch.bfloat16 and q.is_contiguous(),
           f"q must be contiguous bf16 [{b}, HQ, D]")
    hq, d = q.shape[1:]
    _check(d in (64, 128, 256), f"head_dim {d} not supported (64, 128, 256)")
    _check(bounds.dim() == 5 and bounds.shape[0] > 0, "bounds must be bf16 [P, page_size / block_size, HKV, 2, D]")
    p, bpp, hkv = bounds.shape[:3]
    block = _bounds(bounds, p, hkv, d, page_size)
    _heads(hq, hkv)
    n = indices.numel() * bpp
    if output is None:
        output = torch.empty((hkv, n), dtype=torch.float32, device=q.device)
    _check(tuple(output.shape) == (hkv, n) and output.dtype == torch.float32 and output.is_contiguous(),
           f"output must be contiguous float32 [{hkv}, {n}]")
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
    _check(scores.dim() == 2 and scores.dtype == torch.float32 and scores.is_contiguous() and scores.shape[0] > 0
           and scores.shape[1] % (page_size // block_size) == 0,
           "scores must be contiguous float32 [HKV, nnz * page_size / block_size]")
    _check(first >= 0 and keep_last >= 0 and num_select > 0 and first + keep_last <= num_select,
           f"num_select {num_select} must be positive and at least first {first} + keep_last {keep_last}")
    hkv = scores.shape[0]
    if output is None:
        output = torch.empty((b, hkv, num_select), dtype=torch.int32, device=scores.device)
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
) -> torch.Tensor:
    """paged_decode / paged_decode_fp8 over the listed blocks of each sequence and KV head: blocks int32 [B, HKV, n],
    strictly ascending block numbers within the sequence, then -1 (as paged_select_blocks returns them), of block_size
    tokens; None: every block. q [B, HQ, D] bf16; returns bf16 [B, HQ, D], zeros where nothing is attended.

    weights f32 [HKV, nnz], if given, is set to decay * weights_in (zero without weights_in; weights_in may be weights)
    plus the attention that each page-table entry's tokens received, summed over the KV head's queries."""
    b = _table(indptr, last_page_len, indices)
    code, scale, p, page, hkv, d = _cache(kv_cache, kv_scale)
    _check(q.dim() == 3 and q.shape[0] == b and q.shape[2] == d and q.dtype == torch.bfloat16 and q.is_contiguous(),
           f"q must be contiguous bf16 [{b}, HQ, {d}]")
    hq, nnz, n = q.shape[1], indices.numel(), 0
    _heads(hq, hkv)
    if blocks is not None:
        _check(block_size is not None, "blocks need their block_size")
        _check(blocks.dim() == 3 and blocks.shape[2] > 0, f"blocks must be int32 [{b}, {hkv}, n]")
        n = blocks.shape[2]
        _i32(blocks, "blocks", b, hkv, n)
    else:
        block_size = 16
    _sizes(page, block_size)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    if output is None:
        output = torch.empty_like(q)
    _check(output.shape == q.shape and output.dtype == q.dtype and output.is_contiguous(), "bad output tensor")
    _check(weights is not None or weights_in is None, "weights_in without weights")
    for name, t in (("weights_in", weights_in), ("weights", weights)):
        _check(t is None or (t.dtype == torch.float32 and tuple(t.shape) == (hkv, nnz) and t.is_contiguous()),
               f"{name} must be contiguous float32 [{hkv}, {nnz}]")
    _status(status)
    if workspace is None:
        workspace = paged_decode_blocks_workspace(b, hq, hkv, d, page, nnz, q.device, block_size, n, weights is not None)
    _check(workspace.dtype == torch.uint8 and workspace.is_contiguous(), "workspace must be contiguous uint8")
    _call("axk_paged_decode_blocks",
          (q, kv_cache, indptr, indices, last_page_len, blocks, output, weights_in, weights, status, workspace),
          q.data_ptr(), kv_cache.data_ptr(), code, scale, indptr.data_ptr(), indices.data_ptr(), last_page_len.data_ptr(),
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
    _check(b > 0, "the page table holds no sequence")
    _i32(indptr, "indptr", b + 1)
    _check(indices.dtype == torch.int32 and indices.dim() == 1 and indices.is_contiguous(),
           "indices must be contiguous int32 [nnz]")
    nnz = indices.numel()
    _check(weights.dim() == 2 and weights.shape[0] > 0 and weights.shape[1] == nnz and weights.dtype == torch.float32
           and weights.is_contiguous(), f"weights must be contiguous float32 [HKV, {nnz}]")
    _check(first >= 0 and keep_last >= 1 and first + keep_last <= budget,
           f"budget {budget} must hold first {first} (>= 0) + keep_last {keep_last} (>= 1) pages")
    out = (torch.empty_like(indptr), torch.empty_like(indices), torch.empty_like(weights), torch.empty_like(indices))
    _call("axk_paged_evict_pages", (weights, indptr, indices, *out), weights.data_ptr(), indptr.data_ptr(),
          indices.data_ptr(), *(t.data_ptr() for t in out), nnz, b, weights.shape[0], budget, first, keep_last)
    return out
