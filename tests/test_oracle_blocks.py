"""The oracle of the block operators against independent statements (CPU)."""
import math
import random

import pytest
import torch

from axk import configs
from oracle import paged_attn
from oracle import paged_blocks as ob


def case(lens, hq, hkv, d, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    return configs.paged_case(lens, hq, hkv, d, page, g, extra_pages=2)


@pytest.mark.parametrize("page,block", [(32, 16), (48, 48)])
def test_bounds_contain_every_key_and_scores_bound_every_product(page, block):
    lens = [1, 16, 70]
    c = case(lens, 6, 2, 64, page)
    cache, ptr, idx, last = c["cache"], c["indptr"], c["indices"], c["last_page_len"]
    bounds = ob.key_bounds(cache, torch.zeros(cache.shape[0], page // block, 2, 2, 64, dtype=torch.bfloat16), ptr, idx, last)
    scores, mag = ob.block_scores(c["q"], bounds, ptr, idx, last, page)
    bpp = page // block
    for b, n in enumerate(lens):
        k, _, _ = ob.seq_rows(cache, ptr, idx, last, b)
        prod = torch.einsum("hgd,thd->thg", c["q"][b].double().view(2, 3, 64), k).amax(2)  # [t, HKV]
        for t in range(n):
            e, s = int(ptr[b]) + t // page, t % page // block
            bb = bounds[idx[e].long(), s].double()
            assert (bb[:, 0] <= k[t]).all() and (k[t] <= bb[:, 1]).all()
            assert (prod[t] <= scores[:, e * bpp + s] + 1e-12 * mag[:, e * bpp + s]).all()
        j = torch.arange((int(ptr[b + 1]) - int(ptr[b])) * bpp)
        tail = scores[:, int(ptr[b]) * bpp + j[j * block >= n]]
        assert (tail == -math.inf).all()


def test_decode_over_every_block_is_the_paged_decode_oracle_and_weights_sum_to_the_queries():
    lens = [0, 5, 64, 100]
    c = case(lens, 6, 2, 64, 32, seed=1)
    args = [c[n] for n in ("q", "cache", "indptr", "indices", "last_page_len")]
    out, w, slack, _ = ob.decode_blocks(*args, sm_scale=0.125)
    ref = paged_attn.paged_decode(*args, 0.125)
    torch.testing.assert_close(out, ref.double(), rtol=1e-5, atol=1e-5)
    for b, n in enumerate(lens):
        lo, hi = int(c["indptr"][b]), int(c["indptr"][b + 1])
        torch.testing.assert_close(w[:, lo:hi].sum(1), torch.full((2,), 3.0 if n else 0.0, dtype=torch.float64))
    every = torch.full((4, 2, 8), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        nb = -(-n // 16)
        every[b, :, :nb] = torch.arange(nb, dtype=torch.int32)
    out2, w2, _, _ = ob.decode_blocks(*args, blocks=every, block=16, sm_scale=0.125)
    torch.testing.assert_close(out2, out, rtol=0, atol=0)
    torch.testing.assert_close(w2, w, rtol=0, atol=0)


def test_pick_against_a_sort_of_pairs():
    rng = random.Random(3)
    for _ in range(300):
        n = rng.randint(1, 40)
        row = [rng.choice([rng.gauss(0, 1), 0.0, -0.0, 1.0, math.inf, -math.inf, math.nan]) for _ in range(n)]
        first, keep_last = rng.randint(0, 3), rng.randint(0, 3)
        want = rng.randint(max(1, first + keep_last), 12)
        got = ob.pick(row, want, first, keep_last)
        assert got == sorted(set(got)) and len(got) == min(n, want)
        if n > want:
            assert set(range(first)) <= set(got) and set(range(n - keep_last, n)) <= set(got)
            value = lambda i: math.inf if math.isnan(row[i]) else row[i]  # noqa: E731
            for i in set(range(first, n - keep_last)) - set(got):  # what is left out is no better than what is kept
                for j in set(got) & set(range(first, n - keep_last)):
                    assert math.isnan(row[j]) or (not math.isnan(row[i]) and
                                                  (value(i) < value(j) or (value(i) == value(j) and i > j)))


def test_store_then_bounds_from_the_cache_agree():
    g = torch.Generator().manual_seed(4)
    page, block, hkv, d = 32, 16, 2, 64
    cache = torch.zeros(4, 2, page, hkv, d, dtype=torch.bfloat16)
    bounds = torch.full((4, 2, hkv, 2, d), 9.0, dtype=torch.bfloat16)
    ptr, idx = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([3, 1], dtype=torch.int32)
    for at in range(0, 50, 5):
        k = torch.randn(5, hkv, d, generator=g).to(torch.bfloat16)
        loc = torch.tensor([[int(idx[t // page]), t % page] for t in range(at, at + 5)], dtype=torch.int32)
        cache, bounds = ob.store(k, k + 1, cache, bounds, loc)
        last = torch.tensor([(at + 5 - 1) % page + 1], dtype=torch.int32)
        n = torch.tensor([0, 1 + (at + 4) // page], dtype=torch.int32)
        assert torch.equal(ob.key_bounds(cache, bounds, n, idx[:int(n[1])], last), bounds)
    assert ptr[-1] == 2


def test_evict_keeps_budget_pages_and_frees_the_rest():
    w = torch.tensor([[5.0, 1, 2, 3, 9, 0, 7]]).repeat(2, 1)
    ptr = torch.tensor([0, 5, 5, 7], dtype=torch.int32)
    idx = torch.tensor([10, 11, 12, 13, 14, 15, 16], dtype=torch.int32)
    p, i, ww, f = ob.evict_pages(w, ptr, idx, 3)
    assert p.tolist() == [0, 3, 3, 5] and i.tolist() == [10, 13, 14, 15, 16, -1, -1]
    assert f.tolist() == [11, 12, -1, -1, -1, -1, -1] and ww[0].tolist() == [5, 3, 9, 0, 7, 0, 0]


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("page,block", [(32, 16), (48, 48), (16, 16)])
def test_bounds_contain_and_scores_bound_in_every_cache(kv, page, block):
    """lo <= key <= hi and q . k <= score for the keys as attention reads them (int8: code * scale, unrounded), where the
    bounds come from the cache and where they are folded at the write, one-token blocks among them."""
    lens, hq, hkv, d = [1, 16, 70, 33], 6, 2, 64
    c = case(lens, hq, hkv, d, page, seed=7)
    cache, ptr, idx, last, scale = c["cache"], c["indptr"], c["indices"], c["last_page_len"], None
    if kv == "fp8":
        scale = 8.0
        cache = (cache * scale).to(torch.float8_e4m3fn).view(torch.uint8)
    elif kv == "i8":
        cache, scale = paged_attn.quant_kv_i8(cache)
    empty = torch.zeros(cache.shape[0], page // block, hkv, 2, d, dtype=torch.bfloat16)
    read = ob.key_bounds(cache, empty, ptr, idx, last, kv_scale=scale)
    loc = torch.tensor([[int(idx[int(ptr[b]) + t // page]), t % page] for b, n in enumerate(lens) for t in range(n)],
                       dtype=torch.int32)
    written, folded = ob.store(*c["cache"][loc[:, 0].long(), :, loc[:, 1].long()].unbind(1), cache, empty, loc, scale)
    assert torch.equal(written.view(torch.uint8), cache.view(torch.uint8)) and torch.equal(folded, read)
    scores, mag = ob.block_scores(c["q"], read, ptr, idx, last, page)
    bpp = page // block
    for b, n in enumerate(lens):
        k, _, _ = ob.seq_rows(cache, ptr, idx, last, b, scale)
        prod = (c["q"][b].double().view(1, hkv, hq // hkv, d) * k[:, :, None]).sum(3).amax(2)  # [t, HKV]
        for t in range(n):
            e, s = int(ptr[b]) + t // page, t % page // block
            bb = read[idx[e].long(), s].double()
            assert (bb[:, 0] <= k[t]).all() and (k[t] <= bb[:, 1]).all()
            # sums of D terms in 64 bits on both sides
            assert (prod[t] <= scores[:, e * bpp + s] + 2 * d * 2.0 ** -53 * mag[:, e * bpp + s]).all()


def test_bounds_of_an_int8_cache_are_the_tightest_in_bf16():
    """The minimum rounded down and the maximum rounded up by less than a step; a NaN key makes both NaN."""
    x = torch.tensor([-3.0, -1.00390625, -1.0, -0.0, 0.0, 1.0, 1.00390625, 3.0], dtype=torch.float64)
    lo, hi = ob.outward(x, x)
    assert lo.dtype == hi.dtype == torch.bfloat16
    assert lo.tolist() == [-3.0, -1.0078125, -1.0, 0.0, 0.0, 1.0, 1.0, 3.0]
    assert hi.tolist() == [-3.0, -1.0, -1.0, 0.0, 0.0, 1.0, 1.0078125, 3.0]
    top = torch.finfo(torch.bfloat16).max  # past it: the largest finite value inside, infinity outside
    assert [float(t) for t in ob.outward(*2 * [torch.tensor(1.001 * top, dtype=torch.float64)])] == [top, math.inf]
    y = torch.randn(4096, generator=torch.Generator().manual_seed(0)).double()
    lo, hi = ob.outward(y, y)
    step = torch.where(lo.double() == y, 0.0, y.abs() * 2.0 ** -7)
    assert (lo.double() <= y).all() and (y <= hi.double()).all() and (hi.double() - lo.double() <= step).all()
    assert all(t.isnan().all() for t in ob.outward(torch.tensor([math.nan]).double(), torch.tensor([math.nan]).double()))


def test_a_block_named_again_behind_a_fall_counts_again():
    """[0, 2, 1, 2]: 1 is skipped, and 2, above its predecessor, is attended a second time."""
    c = case([64], 4, 2, 64, 32, seed=5)
    args = [c[n] for n in ("q", "cache", "indptr", "indices", "last_page_len")]
    blocks = torch.tensor([[[0, 2, 1, 2], [0, 2, -1, -1]]], dtype=torch.int32)
    out, w, _, _ = ob.decode_blocks(*args, blocks=blocks, block=16)
    k, v, _ = ob.seq_rows(c["cache"], c["indptr"], c["indices"], c["last_page_len"], 0)
    for h, rows in enumerate(([*range(16), *range(32, 48), *range(32, 48)], [*range(16), *range(32, 48)])):
        p = torch.softmax(c["q"][0, 2 * h:2 * h + 2].double() @ k[rows, h].t() / 8, 1)
        torch.testing.assert_close(out[0, 2 * h:2 * h + 2], p @ v[rows, h])
        torch.testing.assert_close(w[h], torch.stack([p[:, :16].sum(), p[:, 16:].sum()]))
