"""The measured work of sparse attention over a long paged KV cache, and of keeping such a cache within a budget.

A cache page is cut into blocks of consecutive tokens; every block and KV head keeps the channel-wise bounds of its keys.
A decode step bounds the attention scores of each block from them, attends the best blocks only, adds up how much
attention every page received, and drops the pages that received least. A case is a dict of plain values whose "kind"
names the operator:
  token   the new tokens' K / V written into the cache and folded into the bounds of their blocks (a decode step, or the
          draft rows of a speculative step)
  bounds  the bounds computed from the cache, for the blocks a prefill chunk touched or for whole sequences
  scores  one upper bound of the attention scores per block and KV head
  select  the best blocks of every sequence and KV head, the first and last ones always among them
  decode  one query token per sequence over its selected blocks (n > 0) or all of them (n = 0), and, with "weights",
          each page's share of the attention added to what it had
  evict   the page table cut down to the pages with the most attention
"own" chooses between the plain forms (elementary torch operations) and the framework's operators.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
INF = float("inf")
KV_SCALE = 8.0  # an FP8 cache holds e4m3(x * KV_SCALE)
DECAY = 0.97  # what a page keeps of its attention weight from one step to the next


def _axk():
    if "axk" in sys.modules:
        return sys.modules["axk"]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "ax-dsl-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import axk

    return axk


# ---- cases ----
def listed():
    return [
        # One decode step's K / V of 16 sequences: a latency-bound call made once per layer and token.
        {"name": "token_b16", "kind": "token", "kv": "bf16", "batch": 16, "rows": 1, "lo": 512, "hi": 4096, "hkv": 2,
         "d": 256, "page": 64, "block": 64},
        # The bounds of the blocks that one 512-token prefill chunk of a prompt wrote, after 3485 earlier tokens.
        {"name": "bounds_chunk512", "kind": "bounds", "kv": "bf16", "batch": 1, "lo": 3997, "hi": 3997, "new": 512,
         "hkv": 2, "d": 256, "page": 256, "block": 64},
        # The bounds of a whole FP8 cache of 16 sequences, as when a cache arrives without them.
        {"name": "bounds_fp8_b16", "kind": "bounds", "kv": "fp8", "batch": 16, "lo": 1024, "hi": 16384, "new": 0,
         "hkv": 2, "d": 256, "page": 64, "block": 32},
        # The block scores of one sequence of ordinary length.
        {"name": "scores_b1", "kind": "scores", "batch": 1, "lo": 5003, "hi": 5003, "hq": 16, "hkv": 2, "d": 256,
         "page": 64, "block": 64},
        # The block scores of the hybrid decode group: 8 sequences of 131072 tokens on 256-token pages.
        {"name": "scores_b8_long", "kind": "scores", "batch": 8, "lo": 131072, "hi": 131072, "hq": 32, "hkv": 4,
         "d": 256, "page": 256, "block": 64},
        # 64 of the 313 blocks of one sequence.
        {"name": "select_b1", "kind": "select", "batch": 1, "lo": 5003, "hi": 5003, "hkv": 2, "page": 64, "block": 16,
         "n": 64},
        # 256 of 8192 blocks for each of 8 sequences and 4 KV heads: the finest blocks of the longest sequences.
        {"name": "select_b8_long", "kind": "select", "batch": 8, "lo": 131072, "hi": 131072, "hkv": 4, "page": 256,
         "block": 16, "n": 256},
        # One sequence of 32003 tokens attending 64 blocks of 64: a single user's decode step.
        {"name": "decode_b1", "kind": "decode", "kv": "bf16", "batch": 1, "lo": 32003, "hi": 32003, "hq": 16, "hkv": 2,
         "d": 256, "page": 64, "block": 64, "n": 64, "weights": False},
        # The hybrid decode group over 4096 selected tokens of 131072 each, with the pages' weights: a 4.3 GB cache.
        {"name": "decode_b8_long", "kind": "decode", "kv": "bf16", "batch": 8, "lo": 131072, "hi": 131072, "hq": 32,
         "hkv": 4, "d": 256, "page": 256, "block": 64, "n": 64, "weights": True},
        # A serving step over the whole FP8 cache of 16 uneven sequences, with the pages' weights.
        {"name": "decode_all_fp8_b16", "kind": "decode", "kv": "fp8", "batch": 16, "lo": 1024, "hi": 16384, "hq": 16,
         "hkv": 2, "d": 256, "page": 64, "block": 64, "n": 0, "weights": True},
        # Four short sequences brought down to 24 pages each.
        {"name": "evict_b4", "kind": "evict", "batch": 4, "lo": 10, "hi": 100, "hkv": 2, "budget": 24},
        # 64 sequences of up to 2048 pages brought down to 512.
        {"name": "evict_b64", "kind": "evict", "batch": 64, "lo": 256, "hi": 2048, "hkv": 4, "budget": 512},
    ]


def _log(rng, lo, hi):
    """An integer spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["token", "bounds", "scores", "select", "decode", "decode", "decode", "evict"])
    kv = rng.choice(["bf16", "fp8"])
    hq, hkv, d = rng.choice([(16, 2, 256), (32, 4, 256), (16, 4, 256), (8, 2, 128), (32, 8, 128), (6, 2, 128),
                             (16, 1, 64), (7, 7, 64)])
    if d == 64:
        kv = "bf16"
    page, block = rng.choice([(16, 16), (64, 16), (64, 32), (64, 64), (256, 64), (256, 128), (256, 256), (96, 48)])
    batch = _log(rng, 1, 64)
    if kind == "evict":
        hi = _log(rng, 2, min(4096, 131072 // batch))
        return {"kind": kind, "batch": batch, "lo": max(1, hi // 8), "hi": hi, "hkv": hkv,
                "budget": _log(rng, 2, max(2, hi))}
    hi = _log(rng, 1, max(1, min(131072, 262144 * 512 // (batch * hkv * d))))
    case = {"kind": kind, "batch": batch, "lo": max(1, hi // 8), "hi": hi, "hkv": hkv, "page": page, "block": block}
    if kind == "token":
        return {**case, "kv": kv, "rows": rng.choice([1, 1, 2, 4, 5]), "d": d, "lo": min(hi + 4, case["lo"] + 4),
                "hi": hi + 4}
    if kind == "bounds":
        return {**case, "kv": kv, "d": d, "new": rng.choice([0, _log(rng, 1, 4096)])}
    if kind == "scores":
        return {**case, "hq": hq, "d": d}
    n = _log(rng, 2, 256)
    if kind == "select":
        return {**case, "n": n}
    return {**case, "kv": kv, "hq": hq, "d": d, "n": rng.choice([0, n, n]), "weights": rng.random() < 0.5}


def _lens(case):
    """The length of each sequence (tokens; pages for evict), spread over [lo, hi] by the case's own sizes."""
    rng = random.Random(case["batch"] * 1000003 + case["lo"] * 1009 + case["hi"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def _cdiv(a, b):
    return -(-a // b)


def work(case):
    kind, lens, hkv = case["kind"], _lens(case), case["hkv"]
    if kind == "evict":
        kept, nnz = sum(min(x, case["budget"]) for x in lens), sum(lens)
        return {"bytes": 4 * hkv * nnz + 4 * nnz + 4 * hkv * kept + 4 * nnz + 8 * len(lens), "flops": hkv * nnz}
    block = case["block"]
    blocks = [_cdiv(x, block) for x in lens]
    if kind == "select":
        out = len(lens) * hkv * case["n"]
        return {"bytes": 4 * hkv * sum(blocks) + 4 * out, "flops": hkv * sum(blocks)}
    d = case["d"]
    size = 1 if case.get("kv") == "fp8" else 2
    bound = 4 * hkv * d  # a block's two bf16 bounds over the heads
    if kind == "token":
        rows = case["batch"] * case["rows"]
        touched = sum(len({(x - 1 - r) // block for r in range(case["rows"])}) for x in lens)
        return {"bytes": 2 * rows * hkv * d * (2 + size) + 2 * touched * bound, "flops": 2 * rows * hkv * d}
    if kind == "bounds":
        first = [0 if not case["new"] else max(0, x - case["new"]) // block for x in lens]
        rows = sum(x - f * block for x, f in zip(lens, first))
        touched = sum(b - f for b, f in zip(blocks, first))
        return {"bytes": rows * hkv * d * size + touched * bound, "flops": 2 * rows * hkv * d}
    hq = case["hq"]
    if kind == "scores":
        return {"bytes": sum(blocks) * bound + 2 * len(lens) * hq * d + 4 * hkv * sum(blocks),
                "flops": 4.0 * sum(blocks) * hq * d}
    n = case["n"] or max(blocks)
    toks = sum(x if b <= n else x - (b - n) * block for x, b in zip(lens, blocks))
    pages = sum(_cdiv(x, case["page"]) for x in lens)
    return {"bytes": 2 * toks * hkv * d * size + 4 * len(lens) * hq * d + (8 * hkv * pages if case["weights"] else 0),
            "flops": 4.0 * toks * hq * d}


# ---- inputs ----
def _table(pages, gen, extra=3):
    """indptr, indices of sequences of so many pages each, and the pool they lie in, in random order."""
    nnz = sum(pages)
    pool = nnz + extra
    indptr = torch.tensor([0] + list(np.cumsum(pages)), dtype=torch.int32, device=DEV)
    indices = torch.randperm(pool, generator=gen, device=DEV)[:nnz].to(torch.int32)
    return indptr, indices, pool


def _cache(pool, page, hkv, d, kv, gen):
    """A KV pool: keys with channels of uneven size, as projections give them, and values of one size."""
    x = torch.randn(pool, 2, page, hkv, d, generator=gen, device=DEV, dtype=torch.bfloat16)
    x[:, 0] *= torch.exp(0.5 * torch.randn(hkv, d, generator=gen, device=DEV)).to(torch.bfloat16)
    return x if kv == "bf16" else (x * KV_SCALE).to(torch.float8_e4m3fn).view(torch.uint8)


def _attended(x, kv):
    """What attention reads for stored values x, in 32 bits."""
    return x.float() if kv == "bf16" else x.view(torch.float8_e4m3fn).float() / KV_SCALE


def _page_bounds(cache, kv, block):
    """bf16 [P, page / block, HKV, 2, D]: the bounds of every full block of a pool, chunk by chunk."""
    p, _, page, hkv, d = cache.shape
    out = torch.empty(p, page // block, hkv, 2, d, dtype=torch.bfloat16, device=DEV)
    for at in range(0, p, 1024):
        k = _attended(cache[at:at + 1024, 0], kv).reshape(-1, page // block, block, hkv, d)
        out[at:at + 1024, :, :, 0] = k.amin(2).to(torch.bfloat16)
        out[at:at + 1024, :, :, 1] = k.amax(2).to(torch.bfloat16)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 7919 + 17)
    kind, hkv = case["kind"], case["hkv"]
    lens = _lens(case)
    st = {"case": case, "kind": kind}
    if kind == "evict":
        st["indptr"], st["indices"], _ = _table(lens, gen)
        # attention weights are spread over decades; equal ones occur (pages never attended)
        w = torch.exp(2.0 * torch.randn(hkv, sum(lens), generator=gen, device=DEV))
        st["weights"] = torch.where(w < 0.1, torch.zeros_like(w), w)
        st["most"] = max(lens)
        return st
    page, block = case["page"], case["block"]
    pages = [_cdiv(x, page) for x in lens]
    st["indptr"], st["indices"], pool = _table(pages, gen)
    st["last"] = torch.tensor([x - (p - 1) * page for x, p in zip(lens, pages)], dtype=torch.int32, device=DEV)
    st["most"] = max(_cdiv(x, block) for x in lens)
    if kind == "select":
        s = torch.randn(hkv, sum(pages) * (page // block), generator=gen, device=DEV) * 6 + 20
        st["scores"] = torch.where(s < 12, torch.round(s), s)  # some equal scores
        return st
    d = case["d"]
    if kind in ("token", "bounds", "decode"):
        kv = case["kv"]
        st["kv_scale"] = KV_SCALE if kv == "fp8" else None
        st["cache"] = _cache(pool, page, hkv, d, kv, gen)
    if kind == "token":
        # the last `rows` tokens of every sequence are new: their slots, and the bounds of the blocks before them
        rows = case["rows"]
        st["k"] = torch.randn(case["batch"] * rows, hkv, d, generator=gen, device=DEV, dtype=torch.bfloat16)
        st["v"] = torch.randn(case["batch"] * rows, hkv, d, generator=gen, device=DEV, dtype=torch.bfloat16)
        first = np.cumsum([0] + pages)
        at = [(first[b] + t // page, t % page) for b, x in enumerate(lens) for t in range(max(0, x - rows), x)]
        at = torch.tensor(np.array(at), device=DEV)
        st["loc"] = torch.stack([st["indices"][at[:, 0]].long(), at[:, 1]], 1).to(torch.int32).contiguous()
        st["bounds"] = _page_bounds(st["cache"], kv, block)
        return st
    if kind == "bounds":
        st["bounds"] = torch.zeros(pool, page // block, hkv, 2, d, dtype=torch.bfloat16, device=DEV)
        st["start"] = None
        if case["new"]:
            st["start"] = torch.tensor([max(0, x - case["new"]) for x in lens], dtype=torch.int32, device=DEV)
        return st
    q = torch.randn(case["batch"], case["hq"], d, generator=gen, device=DEV, dtype=torch.bfloat16) * 2
    st["q"] = q.contiguous()
    if kind == "scores":
        mid = torch.randn(pool, page // block, hkv, 1, d, generator=gen, device=DEV)
        half = 2.0 + torch.rand(pool, page // block, hkv, 1, d, generator=gen, device=DEV)
        st["bounds"] = torch.cat([mid - half, mid + half], 3).to(torch.bfloat16)
        return st
    st["scale"] = 1.0 / math.sqrt(d)
    st["blocks"] = None
    if case["n"]:  # a selection as the select operator gives it: the first and last block and random ones between
        nb = torch.tensor([_cdiv(x, block) for x in lens], device=DEV)[:, None, None]
        j = torch.arange(st["most"], device=DEV)[None, None]
        s = torch.rand(case["batch"], hkv, st["most"], generator=gen, device=DEV)
        s = torch.where((j == 0) | (j == nb - 1), 2.0, torch.where(j < nb, s, -1.0))
        got = torch.topk(s, min(case["n"], st["most"]), dim=2)
        got = torch.where(got.values >= 0, got.indices, 1 << 30).sort(2).values
        got = torch.where(got < (1 << 30), got, -1).to(torch.int32)
        st["blocks"] = torch.full((case["batch"], hkv, case["n"]), -1, dtype=torch.int32, device=DEV)
        st["blocks"][:, :, :got.shape[2]] = got
    st["weights"] = None
    if case["weights"]:
        st["weights"] = torch.rand(hkv, sum(pages), generator=gen, device=DEV)
    return st


# ---- one pass ----
def run(st):
    if own:
        return _run_own(st)
    return {"token": _token, "bounds": _bounds, "scores": _scores, "select": _select, "decode": _decode,
            "evict": _evict}[st["kind"]](st)


def _run_own(st):
    axk, case, kind = _axk(), st["case"], st["kind"]
    if kind == "token":
        axk.store_paged_kv_bounds(st["k"], st["v"], st["cache"], st["bounds"], st["loc"], kv_scale=st["kv_scale"])
        return {"bounds": st["bounds"], "cache": _stored(st)}
    if kind == "bounds":
        return axk.paged_key_bounds(st["cache"], st["bounds"], st["indptr"], st["indices"], st["last"],
                                    start=st["start"], kv_scale=st["kv_scale"])
    if kind == "scores":
        return axk.paged_block_scores(st["q"], st["bounds"], st["indptr"], st["indices"], st["last"], case["page"])
    if kind == "select":
        return axk.paged_select_blocks(st["scores"], st["indptr"], st["last"], case["page"], case["block"], case["n"])
    if kind == "evict":
        return axk.paged_evict_pages(st["weights"], st["indptr"], st["indices"], case["budget"])
    w = None if st["weights"] is None else torch.empty_like(st["weights"])
    out = axk.paged_decode_blocks(st["q"], st["cache"], st["indptr"], st["indices"], st["last"], blocks=st["blocks"],
                                  block_size=case["block"], sm_scale=st["scale"], weights_in=st["weights"], weights=w,
                                  decay=DECAY, kv_scale=st["kv_scale"])
    return {"out": out} if w is None else {"out": out, "weights": w}


def _stored(st):
    """The cache as the values its bytes stand for."""
    return st["cache"] if st["case"]["kv"] == "bf16" else st["cache"].view(torch.float8_e4m3fn)


# ---- the plain forms ----
def _lengths(st):
    """[B] tokens of each sequence, from the page table."""
    pages = (st["indptr"][1:] - st["indptr"][:-1]).long()
    return torch.where(pages > 0, (pages - 1) * st["case"]["page"] + st["last"].long(), 0)


def _owners(st):
    """[nnz] the sequence of each page-table entry."""
    entry = torch.arange(st["indices"].numel() if "indices" in st else st["scores"].shape[1], device=DEV,
                         dtype=torch.int32)
    return torch.searchsorted(st["indptr"], entry, right=True) - 1


def _token(st):
    case, loc = st["case"], st["loc"].long()
    k, v, cache = st["k"], st["v"], st["cache"]
    if case["kv"] == "fp8":
        k, v = (x.float() * KV_SCALE for x in (k, v))
        k, v = (x.to(torch.bfloat16).to(torch.float8_e4m3fn).view(torch.uint8) for x in (k, v))
    cache[loc[:, 0], 0, loc[:, 1]] = k
    cache[loc[:, 0], 1, loc[:, 1]] = v
    block, bounds = case["block"], st["bounds"]
    at = loc[:, 0] * (case["page"] // block) + loc[:, 1] // block
    flat = bounds.view(-1, *bounds.shape[2:])
    lo, hi = flat[:, :, 0].float(), flat[:, :, 1].float()
    fresh = torch.zeros(flat.shape[0], device=DEV).index_add(0, at, (loc[:, 1] % block == 0).float()) > 0
    lo = torch.where(fresh[:, None, None], INF, lo)
    hi = torch.where(fresh[:, None, None], -INF, hi)
    key = _attended(k, case["kv"])
    lo = lo.index_reduce(0, at, key, "amin")
    hi = hi.index_reduce(0, at, key, "amax")
    flat[:, :, 0] = lo.to(torch.bfloat16)
    flat[:, :, 1] = hi.to(torch.bfloat16)
    return {"bounds": bounds, "cache": _stored(st)}


def _bounds(st):
    case, bounds = st["case"], st["bounds"]
    page, block = case["page"], case["block"]
    b = _owners(st)
    entry = torch.arange(b.numel(), device=DEV) - st["indptr"][b].long()  # a page's place in its sequence
    k = _attended(st["cache"][st["indices"].long(), 0], case["kv"])
    t = entry[:, None] * page + torch.arange(page, device=DEV)
    there = (t < _lengths(st)[b][:, None])[:, :, None, None]
    blocks = (-1, page // block, block, case["hkv"], case["d"])
    lo = torch.where(there, k, INF).view(blocks).amin(2)
    hi = torch.where(there, k, -INF).view(blocks).amax(2)
    first = torch.zeros_like(b) if st["start"] is None else st["start"].long()[b]
    start = t[:, ::block]  # each block's first token
    todo = ((start < _lengths(st)[b][:, None]) & (start + block > first[:, None]))[:, :, None, None, None]
    new = torch.stack([lo, hi], 3).to(torch.bfloat16)
    at = st["indices"].long()
    bounds[at] = torch.where(todo, new, bounds[at])
    return bounds


def _entries(st):
    """[B, most] the page-table entry of each sequence's block, and whether it exists."""
    case = st["case"]
    j = torch.arange(st["most"], device=DEV)
    there = j < (_lengths(st)[:, None] + case["block"] - 1) // case["block"]
    entry = st["indptr"][:-1].long()[:, None] + j // (case["page"] // case["block"])
    return torch.where(there, entry, 0), j % (case["page"] // case["block"]), there


def _scores(st):
    case = st["case"]
    entry, sub, there = _entries(st)
    bounds = st["bounds"][st["indices"].long()[entry], sub].permute(3, 0, 2, 1, 4).float()  # [2, B, HKV, most, D]
    b, hq, d = st["q"].shape
    q = st["q"].float().view(b, case["hkv"], hq // case["hkv"], d).transpose(2, 3)
    s = torch.matmul(bounds[0], q.clamp(max=0)) + torch.matmul(bounds[1], q.clamp(min=0))
    s = torch.where(there[:, None], s.amax(3), -INF)
    bpp = case["page"] // case["block"]
    owner = _owners(st)
    place = (torch.arange(owner.numel(), device=DEV) - st["indptr"][owner].long())[:, None] * bpp \
        + torch.arange(bpp, device=DEV)
    got = s[owner[:, None], :, place.clamp(max=st["most"] - 1)]  # [nnz, bpp, HKV]
    return torch.where((place < st["most"])[:, :, None], got, -INF).permute(2, 0, 1).reshape(case["hkv"], -1)


def _kept(key, there, n):
    """Where the n largest of each row's `key` are, equal ones by the lowest place."""
    order = torch.sort(torch.where(there, key, -INF), dim=-1, descending=True, stable=True).indices
    return torch.zeros_like(there).scatter(-1, order[..., :n], True) & there


def _select(st):
    case = st["case"]
    entry, sub, there = _entries(st)
    at = torch.where(there, entry * (case["page"] // case["block"]) + sub, 0)
    s = st["scores"][:, at].transpose(0, 1)  # [B, HKV, most]
    j = torch.arange(st["most"], device=DEV)
    nb = there.sum(1, keepdim=True)
    always = (j < 1) | (j >= nb - 1)
    keep = _kept(torch.where(always[:, None], INF, s), there[:, None].expand_as(s), case["n"])
    place = torch.where(keep, j, 1 << 30).sort(-1).values[..., :case["n"]]
    out = torch.full((*s.shape[:2], case["n"]), -1, dtype=torch.int32, device=DEV)
    out[..., :place.shape[-1]] = torch.where(place < (1 << 30), place, -1).to(torch.int32)
    return out


def _decode(st):
    case = st["case"]
    page, block, hkv = case["page"], case["block"], case["hkv"]
    b, hq, d = st["q"].shape
    blocks = st["blocks"]
    if blocks is None:
        blocks = torch.arange(st["most"], device=DEV, dtype=torch.int32).expand(b, hkv, -1)
    t = blocks.long()[..., None] * block + torch.arange(block, device=DEV)
    there = (blocks[..., None] >= 0) & (t < _lengths(st)[:, None, None, None])
    t = torch.where(there, t, 0).flatten(2)  # [B, HKV, n * block]
    there = there.flatten(2)
    at = st["indices"].long()[st["indptr"][:-1].long()[:, None, None] + t // page]
    head = torch.arange(hkv, device=DEV)[None, :, None]
    q = st["q"].float().view(b, hkv, hq // hkv, d)
    k = _attended(st["cache"][at, 0, t % page, head], case["kv"])
    s = torch.matmul(q, k.transpose(2, 3)) * st["scale"]
    del k
    s = torch.where(there[:, :, None], s, -INF)
    p = torch.exp(s - s.amax(3, keepdim=True).clamp(min=-3e38))
    total = p.sum(3, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = _attended(st["cache"][at, 1, t % page, head], case["kv"])
    v = torch.where(there[..., None], v, 0.0)
    out = {"out": torch.matmul(p, v).reshape(b, hq, d).to(torch.bfloat16)}
    if st["weights"] is not None:
        share = p.sum(2).view(b, hkv, -1, block).sum(3)  # [B, HKV, n]: over the group's heads and the block's tokens
        bpp = page // block
        most = _cdiv(st["most"], bpp) * bpp
        each = torch.zeros(b, hkv, most + 1, device=DEV).scatter(2, torch.where(blocks < 0, most, blocks).long(), share)
        each = each[..., :most].reshape(b, hkv, most // bpp, bpp).sum(3)
        owner = _owners(st)
        place = torch.arange(owner.numel(), device=DEV) - st["indptr"][owner].long()
        out["weights"] = st["weights"] * DECAY + each[owner, :, place].t()
    return out


def _evict(st):
    w, indptr, indices, budget = st["weights"], st["indptr"], st["indices"], st["case"]["budget"]
    nnz = indices.numel()
    pages = (indptr[1:] - indptr[:-1]).long()[:, None]
    j = torch.arange(st["most"], device=DEV)
    there = j < pages
    total = w.double().sum(0)[torch.where(there, indptr[:-1].long()[:, None] + j, 0)]
    total = torch.where((j < 1) | (j >= pages - 1), INF, total)
    owner = _owners(st)
    keep = _kept(total, there, budget)[owner, torch.arange(nnz, device=DEV) - indptr[owner].long()]
    at = torch.where(keep, torch.cumsum(keep, 0) - 1, nnz)
    out_indices = torch.full((nnz + 1,), -1, dtype=torch.int32, device=DEV).scatter(0, at, indices)[:nnz]
    out_w = torch.zeros(w.shape[0], nnz + 1, device=DEV).scatter(1, at.expand_as(w), w)[:, :nnz]
    off = torch.where(keep, nnz, torch.cumsum(~keep, 0) - 1)
    freed = torch.full((nnz + 1,), -1, dtype=torch.int32, device=DEV).scatter(0, off, indices)[:nnz]
    out_indptr = torch.zeros_like(indptr)
    out_indptr[1:] = torch.cumsum(pages[:, 0].clamp(max=budget), 0).to(torch.int32)
    return out_indptr, out_indices, out_w, freed


# ---- the definitions, in 64 bits, one sequence at a time ----
def _values(x, kv):
    """Stored values in 64 bits; an E4M3 byte by its fields."""
    if kv == "bf16":
        return x.double()
    x = x.long()
    sign, e, m = 1.0 - 2.0 * (x >> 7).double(), (x >> 3) & 15, (x & 7).double()
    return sign * torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m / 512) / KV_SCALE


def exact(case, seed):
    st = prepare(case, seed)
    kind, hkv = case["kind"], case["hkv"]
    lens = _lens(case)
    ptr = st["indptr"].tolist()
    if kind == "evict":
        w, idx = st["weights"].cpu().numpy(), st["indices"].cpu().numpy()
        total, keep = w.astype(np.float64).sum(0), []
        for b, n in enumerate(lens):
            t = total[ptr[b]:ptr[b + 1]].copy()
            t[0] = t[-1] = np.inf
            keep += sorted(np.lexsort((np.arange(n), -t))[:case["budget"]] + ptr[b])
        gone = sorted(set(range(ptr[-1])) - set(keep))
        out_w = np.zeros(w.shape, dtype=np.float64)
        out_w[:, :len(keep)] = w[:, keep]
        fill = lambda x: np.concatenate([idx[x], np.full(len(idx) - len(x), -1, np.int32)]).astype(np.int32)  # noqa: E731
        counts = [min(n, case["budget"]) for n in lens]
        return np.cumsum([0] + counts).astype(np.int32), fill(keep), out_w, fill(gone)
    page, block = case["page"], case["block"]
    bpp = page // block
    if kind == "select":
        out = np.full((len(lens), hkv, case["n"]), -1, dtype=np.int32)
        s = st["scores"].cpu().numpy()
        for b, x in enumerate(lens):
            nb = _cdiv(x, block)
            for h in range(hkv):
                row = s[h, ptr[b] * bpp:ptr[b] * bpp + nb].astype(np.float64)
                row[0] = row[-1] = np.inf
                best = np.sort(np.lexsort((np.arange(nb), -row))[:case["n"]])
                out[b, h, :len(best)] = best
        return out
    d = case["d"]
    if kind == "token":
        k = st["k"].double()
        if case["kv"] == "fp8":
            k = (k * KV_SCALE).to(torch.bfloat16).to(torch.float8_e4m3fn).double() / KV_SCALE
        bounds = st["bounds"].double()
        mine = {}
        for r, (p, s) in enumerate(st["loc"].tolist()):
            mine.setdefault((p, s // block), []).append((s % block, r))
        for (p, s), rows in mine.items():
            keys = [k[r] for _, r in rows]
            if all(o for o, _ in rows):
                keys += [bounds[p, s, :, 0], bounds[p, s, :, 1]]
            keys = torch.stack(keys)
            bounds[p, s] = torch.stack([keys.amin(0), keys.amax(0)], 1)
        return {"bounds": bounds, "cache": None}
    if kind == "bounds":
        bounds = st["bounds"].double()
        for b, x in enumerate(lens):
            ids = st["indices"][ptr[b]:ptr[b + 1]].long()
            k = _values(st["cache"][ids, 0], case["kv"]).reshape(-1, hkv, d)[:x]
            first = 0 if not case["new"] else max(0, x - case["new"]) // block
            rest = x // block * block
            both = []
            if rest > first * block:
                full = k[first * block:rest].reshape(-1, block, hkv, d)
                both.append(torch.stack([full.amin(1), full.amax(1)], 2))
            if x > rest:
                both.append(torch.stack([k[rest:].amin(0), k[rest:].amax(0)], 1)[None])
            at = torch.arange(first, _cdiv(x, block), device=DEV)
            bounds[ids[at // bpp], at % bpp] = torch.cat(both)
        return bounds
    q = st["q"].double()
    group = case["hq"] // hkv
    if kind == "scores":
        out = torch.full((hkv, ptr[-1] * bpp), -INF, dtype=torch.float64, device=DEV)
        for b, x in enumerate(lens):
            ids = st["indices"][ptr[b]:ptr[b + 1]].long()
            both = st["bounds"][ids].double().reshape(-1, hkv, 2, d)[:_cdiv(x, block)]
            for h in range(hkv):
                best = [torch.maximum(both[:, h, 0] * q[b, i], both[:, h, 1] * q[b, i]).sum(1)
                        for i in range(h * group, (h + 1) * group)]
                out[h, ptr[b] * bpp:ptr[b] * bpp + both.shape[0]] = torch.stack(best).amax(0)
        return out
    out = torch.zeros(len(lens), case["hq"], d, dtype=torch.float64, device=DEV)
    weights = None if st["weights"] is None else st["weights"].double() * DECAY
    for b, x in enumerate(lens):
        ids = st["indices"][ptr[b]:ptr[b + 1]].long()
        for h in range(hkv):
            rows = torch.arange(x, device=DEV)
            if st["blocks"] is not None:
                mine = st["blocks"][b, h].long()
                rows = rows[torch.isin(rows // block, mine[mine >= 0])]
            k, v = (_values(st["cache"][ids[rows // page], i, rows % page, h], case["kv"]) for i in (0, 1))
            s = (q[b, h * group:(h + 1) * group] @ k.t()) * st["scale"]
            p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
            out[b, h * group:(h + 1) * group] = p @ v
            if weights is not None:
                weights[h].index_add_(0, ptr[b] + rows // page, p.sum(0))
    return {"out": out} if weights is None else {"out": out, "weights": weights}
