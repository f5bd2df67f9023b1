"""Oracle: sparse attention over a paged KV cache and the eviction of its pages (CPU, 64 bits, test infrastructure only).

Blocks, bounds, page tables and argument meaning as include/axk.h describes them. Everything is computed one sequence and
one KV head at a time from gathered rows. Pinned by tests/test_oracle_blocks.py: the bounds contain every key, the scores
bound every product, decode over every block equals the paged decode oracle, the weights of a row sum to its queries, and
the selection and eviction agree with a sort in plain Python.
"""
from __future__ import annotations

import math

import torch

from .paged_attn import quant_kv_i8, seq_lens


def attended(x: torch.Tensor, kv_scale=None) -> torch.Tensor:
    """Stored cache values as attention reads them, in 64 bits. kv_scale: None for bf16, the static scale of FP8 bytes, or
    the scales of int8 codes, one per row of the last dimension."""
    if isinstance(kv_scale, torch.Tensor):
        return x.double() * kv_scale.double()[..., None]
    return x.double() if kv_scale is None else x.view(torch.float8_e4m3fn).double() / kv_scale


def seq_rows(cache, indptr, indices, last, b: int, kv_scale=None):
    """(K, V) [len, HKV, D] in 64 bits, and which tokens lie on pages inside the pool."""
    p, _, page, hkv, d = cache.shape
    n = seq_lens(indptr, last, page)[b]
    ids = indices[int(indptr[b]):int(indptr[b + 1])].long()
    good = (ids >= 0) & (ids < p)
    at = torch.where(good, ids, 0)
    kv = attended(cache[at], kv_scale[at] if isinstance(kv_scale, torch.Tensor) else kv_scale)
    kv = kv.transpose(0, 1).reshape(2, -1, hkv, d)[:, :n]
    return kv[0], kv[1], good.repeat_interleave(page)[:n]


def outward(lo: torch.Tensor, hi: torch.Tensor):
    """(lo rounded down, hi rounded up) to bf16, so that they still contain what they bounded; NaN stays."""
    a, b = lo.to(torch.bfloat16), hi.to(torch.bfloat16)
    a = torch.where(a.double() > lo, torch.nextafter(a, torch.full_like(a, -math.inf)), a)
    return a, torch.where(b.double() < hi, torch.nextafter(b, torch.full_like(b, math.inf)), b)


def key_bounds(cache, bounds, indptr, indices, last, start=None, kv_scale=None) -> torch.Tensor:
    out = bounds.clone()
    page = cache.shape[2]
    bpp = bounds.shape[1]
    block = page // bpp
    for b, n in enumerate(seq_lens(indptr, last, page)):
        k, _, good = seq_rows(cache, indptr, indices, last, b, kv_scale)
        for j in range(-(-n // block)):
            if (start is not None and (j + 1) * block <= int(start[b])) or not good[j * block]:
                continue
            rows = k[j * block:min(n, (j + 1) * block)]
            at = int(indices[int(indptr[b]) + j // bpp])
            out[at, j % bpp] = torch.stack(outward(rows.amin(0), rows.amax(0)), 1)
    return out


def store(k, v, cache, bounds, loc, kv_scale=None):
    """(cache, bounds) after the rows are written in order; an int8 cache's scales, kv_scale, are written in place."""
    cache, out = cache.clone(), bounds.double()
    p, _, page = cache.shape[:3]
    block = page // bounds.shape[1]
    good = [(r, int(a), int(o)) for r, (a, o) in enumerate(loc.tolist()) if 0 <= a < p and 0 <= o < page]
    fresh = {(a, o // block) for _, a, o in good if o % block == 0}
    begun = set()
    for r, a, o in good:
        for i, x in enumerate((k, v)):
            row, s = x[r], kv_scale
            if isinstance(kv_scale, torch.Tensor):
                row, s = quant_kv_i8(row)
                kv_scale[a, i, o] = s
            elif kv_scale is not None:
                row = (row.float() * kv_scale).to(torch.bfloat16).to(torch.float8_e4m3fn).view(torch.uint8)
            cache[a, i, o] = row
            if i == 0:
                key = attended(row, s)
        at = (a, o // block)
        if at in fresh and at not in begun:
            out[at] = torch.stack([key, key], 1)
        else:
            out[at] = torch.stack([torch.minimum(out[at][:, 0], key), torch.maximum(out[at][:, 1], key)], 1)
        begun.add(at)
    return cache, torch.stack(outward(out[:, :, :, 0], out[:, :, :, 1]), 3)


def block_scores(q, bounds, indptr, indices, last, page: int):
    """(scores, sums of the products' magnitudes) f64 [HKV, nnz * bpp]; NaN where nothing is to be written."""
    p, bpp, hkv, _, d = bounds.shape
    block, group = page // bpp, q.shape[1] // hkv
    out = torch.full((hkv, indices.numel() * bpp), math.nan, dtype=torch.float64)
    mag = out.clone()
    for b, n in enumerate(seq_lens(indptr, last, page)):
        for e in range(int(indptr[b]), int(indptr[b + 1])):
            for s in range(bpp):
                j = (e - int(indptr[b])) * bpp + s
                at = int(indices[e])
                if j * block >= n or not 0 <= at < p:
                    out[:, e * bpp + s] = -math.inf
                    mag[:, e * bpp + s] = 0
                    continue
                lo, hi = bounds[at, s, :, 0].double(), bounds[at, s, :, 1].double()
                x = q[b].double().view(hkv, group, d)
                t = torch.maximum(x * lo[:, None], x * hi[:, None])
                out[:, e * bpp + s] = t.sum(2).amax(1)
                mag[:, e * bpp + s] = t.abs().sum(2).amax(1)
    return out, mag


def order(row):
    """Places by descending value, NaN first, equal ones in order."""
    return sorted(range(len(row)), key=lambda i: (not math.isnan(row[i]), 0.0 if math.isnan(row[i]) else -row[i], i))


def pick(row, n: int, first: int, keep_last: int):
    """The places that a selection of n keeps, ascending."""
    if len(row) <= n:
        return list(range(len(row)))
    always = list(range(first)) + list(range(len(row) - keep_last, len(row)))
    rest = [i for i in order(row) if i not in set(always)]
    return sorted(always + rest[:n - len(always)])


def select_blocks(scores, indptr, last, page: int, block: int, n: int, first: int = 1, keep_last: int = 1):
    hkv, bpp = scores.shape[0], page // block
    lens = seq_lens(indptr, last, page)
    out = torch.full((len(lens), hkv, n), -1, dtype=torch.int32)
    for b, x in enumerate(lens):
        at = int(indptr[b]) * bpp
        for h in range(hkv):
            got = pick(scores[h, at:at - (-x // block)].tolist(), n, first, keep_last)
            out[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out


def decode_blocks(q, cache, indptr, indices, last, blocks=None, block: int = 16, sm_scale=None, weights_in=None,
                  decay: float = 1.0, kv_scale=None):
    """(out f64 [B, HQ, D], weights f64 [HKV, nnz], a bound of the rounding errors of each). The bounds follow the
    arithmetic that is allowed to round: fp32 sums of D exact products and of the tokens, an fp32 exponential, and
    probabilities in bf16 (half a step: 2^-8) where they meet V."""
    p, _, page, hkv, d = cache.shape
    bsz, hq, _ = q.shape
    group = hq // hkv
    sm_scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    out = torch.zeros(bsz, hq, d, dtype=torch.float64)
    slack = torch.zeros_like(out)
    w = torch.zeros(hkv, indices.numel(), dtype=torch.float64) if weights_in is None else weights_in.double() * decay
    wslack = w.abs() * 2 ** -22
    for b, n in enumerate(seq_lens(indptr, last, page)):
        k, v, good = seq_rows(cache, indptr, indices, last, b, kv_scale)
        t = torch.arange(n)
        for h in range(hkv):
            rows = t[good]
            if blocks is not None:
                ids, prev = [], -1
                for slot, i in enumerate(blocks[b, h].tolist()):
                    if 0 <= i < -(-n // block) and (slot == 0 or (i > prev and prev != -1)):
                        ids.append(i)
                    prev = i
                rows = torch.cat([rows[rows // block == i] for i in ids] or [rows[:0]])
            if not len(rows):
                continue
            x = q[b, h * group:(h + 1) * group].double()
            kk, vv = k[rows, h], v[rows, h]
            s = x @ kk.t() * sm_scale
            pr = torch.softmax(s, 1)
            # a score is off by its sum's roundings and by the exponential's argument's
            off = 2.0 ** -24 * (d + 8) * abs(sm_scale) * (x.abs() @ kk.abs().t()) + 2.0 ** -22 * (s.abs() + s.abs().amax(1, keepdim=True))
            rel = 2 * off.amax(1, keepdim=True) + 2.0 ** -24 * (len(rows) + 64)
            out[b, h * group:(h + 1) * group] = pr @ vv
            slack[b, h * group:(h + 1) * group] = (2.0 ** -8 + rel) * (pr @ vv.abs())
            w[h].index_add_(0, int(indptr[b]) + rows // page, pr.sum(0))
            wslack[h].index_add_(0, int(indptr[b]) + rows // page, (pr * rel).sum(0))
    return out, w, slack, wslack + w.abs() * 2.0 ** -22


def evict_pages(weights, indptr, indices, budget: int, first: int = 1, keep_last: int = 1):
    nnz = indices.numel()
    total = weights.double().sum(0).tolist()
    keep, gone, ptr = [], [], [0]
    for b in range(len(indptr) - 1):
        lo, hi = int(indptr[b]), int(indptr[b + 1])
        got = [lo + i for i in pick(total[lo:hi], budget, first, keep_last)]
        keep += got
        gone += sorted(set(range(lo, hi)) - set(got))
        ptr.append(len(keep))
    out_i, freed = torch.full((nnz,), -1, dtype=torch.int32), torch.full((nnz,), -1, dtype=torch.int32)
    out_i[:len(keep)] = indices[keep]
    freed[:len(gone)] = indices[gone]
    out_w = torch.zeros_like(weights)
    out_w[:, :len(keep)] = weights[:, keep]
    return torch.tensor(ptr, dtype=torch.int32), out_i, out_w, freed
