"""Block bounds, scores, selection, decode over blocks and page eviction on the GPU against the 64-bit oracle."""
import math
import random

import pytest
import torch

import axk
from oracle import paged_attn
from oracle import paged_blocks as ob

pytestmark = pytest.mark.gpu
NAN = math.nan


def make(lens, hq, hkv, d, page, kv="bf16", seed=0, extra=3):
    """A pool with the given sequences on shuffled pages; every slot that no token has holds NaN. CPU tensors."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    pool = sum(pages) + extra
    idx = torch.randperm(pool, generator=g)[:sum(pages)].to(torch.int32)
    ptr = torch.tensor([sum(pages[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    last = torch.tensor([n - (p - 1) * page if p else 0 for n, p in zip(lens, pages)], dtype=torch.int32)
    x = torch.randn(pool, 2, page, hkv, d, generator=g).to(torch.bfloat16)
    x[:, 0] *= torch.exp(0.5 * torch.randn(hkv, d, generator=g)).to(torch.bfloat16)
    used = torch.zeros(pool, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[int(idx[int(ptr[b]) + t // page]), t % page] = True
    scale = None
    if kv == "fp8":
        scale = 8.0
        x = (x * scale).to(torch.float8_e4m3fn).view(torch.uint8)
        x.masked_fill_(~used[:, None, :, None, None], 0x7F)
    elif kv == "bf16":
        x.masked_fill_(~used[:, None, :, None, None], NAN)
    if kv == "i8":
        codes, scale = paged_attn.quant_kv_i8(x)
        x = codes.masked_fill(~used[:, None, :, None, None], 127)
        scale.masked_fill_(~used[:, None, :, None], NAN)
    q = (1.5 * torch.randn(len(lens), hq, d, generator=g)).to(torch.bfloat16)
    return dict(lens=lens, q=q, cache=x, ptr=ptr, idx=idx, last=last, scale=scale, page=page, hkv=hkv, d=d)


def table(c, dev):
    return c["ptr"].to(dev), c["idx"].to(dev), c["last"].to(dev)


def kv_of(c, dev=None):
    """The scale arguments of the operators for this cache (an int8 cache's scales on the device)."""
    s = c["scale"]
    if isinstance(s, torch.Tensor):
        return {"kv_scales": s.to(dev)}
    return {"kv_scale": s}


def empty_bounds(c, block, fill=0.0):
    return torch.full((c["cache"].shape[0], c["page"] // block, c["hkv"], 2, c["d"]), fill, dtype=torch.bfloat16)


def random_blocks(c, block, n, seed=0):
    rng = random.Random(seed)
    out = torch.full((len(c["lens"]), c["hkv"], n), -1, dtype=torch.int32)
    for b, x in enumerate(c["lens"]):
        nb = -(-x // block)
        for h in range(c["hkv"]):
            got = sorted(rng.sample(range(nb), min(nb, rng.randint(1, n)))) if nb else []
            out[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out


def within(got, ref, slack):
    """Every value within its bound; a bf16 result adds half a step of its own."""
    got, ref = got.double().cpu(), ref.double()
    assert not got.isnan().any()
    tol = slack + (ref.abs() * 2.0 ** -8 if got.dtype == torch.bfloat16 else 0)
    bad = (got - ref).abs() > tol * 1.01 + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float(((got - ref).abs() / (tol + 1e-30)).max())}"


def check_decode(c, dev, blocks=None, block=16, weights=True, decay=0.75, sm_scale=None, win=True):
    g = torch.Generator().manual_seed(5)
    w0 = torch.rand(c["hkv"], c["idx"].numel(), generator=g) if win else None
    ref, rw, slack, wslack = ob.decode_blocks(c["q"], c["cache"], c["ptr"], c["idx"], c["last"], blocks, block, sm_scale,
                                              w0, decay, c["scale"])
    w = torch.full((c["hkv"], c["idx"].numel()), NAN, device=dev) if weights else None
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = axk.paged_decode_blocks_workspace(len(c["lens"]), c["q"].shape[1], c["hkv"], c["d"], c["page"], c["idx"].numel(), dev,
                                           block, 0 if blocks is None else blocks.shape[2], weights)
    ws.fill_(255)  # NaNs: nothing may be read that the call has not written
    out = axk.paged_decode_blocks(c["q"].to(dev), c["cache"].to(dev), *table(c, dev), workspace=ws,
                                  blocks=None if blocks is None else blocks.to(dev), block_size=block, sm_scale=sm_scale,
                                  weights_in=w0.to(dev) if weights and win else None, weights=w, decay=decay,
                                  status=status, **kv_of(c, dev))
    within(out, ref, slack + ref.abs() * 2.0 ** -8)
    if weights:
        within(w, rw, wslack)
    return out, w, int(status)


# ---- key bounds ----
@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("hkv,d,page,block", [(2, 256, 64, 64), (1, 64, 16, 16), (3, 64, 96, 48), (8, 128, 256, 128),
                                              (16, 256, 32, 16), (5, 128, 64, 32)])
def test_bounds_from_the_cache(dev, kv, hkv, d, page, block):
    c = make([0, 1, block, page + 3, 2 * page, 5 * block - 1], hkv, hkv, d, page, kv, seed=hkv)
    fill = empty_bounds(c, block, 7.0)
    for start in (None, torch.tensor([0, 0, block, page, 2 * page - block - 1, block + 1], dtype=torch.int32)):
        ref = ob.key_bounds(c["cache"], fill, c["ptr"], c["idx"], c["last"], start, c["scale"])
        got = axk.paged_key_bounds(c["cache"].to(dev), fill.to(dev), *table(c, dev), **kv_of(c, dev),
                                   start=None if start is None else start.to(dev)).cpu()
        assert torch.equal(got, ref)


def test_bounds_skip_pages_outside_the_pool_and_padding(dev):
    c = make([40, 64], 2, 2, 64, 32)
    c["idx"][1] = c["cache"].shape[0]
    c["idx"][2] = -1
    fill = empty_bounds(c, 16, 7.0)
    idx = torch.cat([c["idx"], torch.full((3,), 1 << 30, dtype=torch.int32)])  # a table with room to spare
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = axk.paged_key_bounds(c["cache"].to(dev), fill.to(dev), c["ptr"].to(dev), idx.to(dev), c["last"].to(dev),
                               status=status).cpu()
    assert torch.equal(got, ob.key_bounds(c["cache"], fill, c["ptr"], c["idx"], c["last"])) and int(status) == 1


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("hkv,d,page,block,rows", [(2, 256, 64, 64, 1), (1, 64, 16, 16, 5), (3, 64, 96, 48, 3),
                                                   (16, 256, 32, 16, 2)])
def test_store_folds_rows_in_order(dev, kv, hkv, d, page, block, rows):
    """Sequences grown from nothing, `rows` tokens of each a call; afterwards the bounds are those of the cache."""
    n, bsz = 2 * page + 5, 3
    c = make([n] * bsz, hkv, hkv, d, page, kv)
    cache = torch.zeros_like(c["cache"]).to(dev)
    bounds = empty_bounds(c, block, 9.0).to(dev)
    kvs = kv_of(c, dev)
    g = torch.Generator().manual_seed(1)
    for at in range(0, n, rows):
        t = list(range(at, min(n, at + rows)))
        k, v = (torch.randn(bsz * len(t), hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
        loc = torch.tensor([[int(c["idx"][int(c["ptr"][b]) + i // page]), i % page] for b in range(bsz) for i in t],
                           dtype=torch.int32)
        rc, rb = ob.store(k, v, cache.cpu(), bounds.cpu(), loc, c["scale"])
        axk.store_paged_kv_bounds(k.to(dev), v.to(dev), cache, bounds, loc.to(dev), **kvs)
        assert torch.equal(cache.cpu().view(torch.uint8), rc.view(torch.uint8)) and torch.equal(bounds.cpu(), rb)
    if kv == "i8":
        assert torch.equal(kvs["kv_scales"].cpu().view(torch.int16), c["scale"].view(torch.int16))
    used = axk.paged_key_bounds(cache, bounds.clone(), *table(c, dev), **kvs)
    assert torch.equal(used, bounds)


def test_store_matches_the_plain_writes_and_handles_shared_slots(dev):
    """600 rows in one call: some share blocks, some a slot (the last is stored), some lie outside the pool."""
    hkv, d, page, block, pool = 2, 128, 64, 16, 12
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(600, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    loc = torch.stack([torch.randint(0, pool, (600,), generator=g), torch.randint(0, page, (600,), generator=g)], 1).int()
    loc[5], loc[300], loc[17] = torch.tensor([-1, 3]), torch.tensor([2, page]), torch.tensor([pool, 0])
    cache = torch.zeros(pool, 2, page, hkv, d, dtype=torch.bfloat16)
    bounds = torch.randn(pool, page // block, hkv, 2, d, generator=g).to(torch.bfloat16)
    rc, rb = ob.store(k, v, cache, bounds, loc)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    gc, gb = cache.to(dev), bounds.to(dev)
    axk.store_paged_kv_bounds(k.to(dev), v.to(dev), gc, gb, loc.to(dev), status=status)
    assert torch.equal(gc.cpu(), rc) and torch.equal(gb.cpu(), rb) and int(status) == 1
    # distinct slots: the bytes are those of store_paged_kv and store_paged_kv_fp8
    loc = torch.tensor([[3, 1], [4, 0], [4, 63], [9, 16]], dtype=torch.int32).to(dev)
    for dtype, scale in ((torch.bfloat16, None), (torch.uint8, 4.0)):
        a = torch.zeros(pool, 2, page, hkv, d, dtype=dtype, device=dev)
        b = a.clone()
        axk.store_paged_kv_bounds(k[:4].to(dev), v[:4].to(dev), a, gb, loc, kv_scale=scale)
        if scale is None:
            axk.store_paged_kv(k[:4].to(dev), v[:4].to(dev), b, loc)
        else:
            axk.store_paged_kv_fp8(k[:4].to(dev), v[:4].to(dev), b, loc, scale)
        assert torch.equal(a, b)
    a, b = (torch.zeros(pool, 2, page, hkv, d, dtype=torch.int8, device=dev) for _ in range(2))
    sa, sb = (torch.zeros(pool, 2, page, hkv, dtype=torch.bfloat16, device=dev) for _ in range(2))
    axk.store_paged_kv_bounds(k[:4].to(dev), v[:4].to(dev), a, gb, loc, kv_scales=sa)
    axk.store_paged_kv_i8(k[:4].to(dev), v[:4].to(dev), b, sb, loc)
    assert torch.equal(a, b) and torch.equal(sa, sb)
    axk.store_paged_kv_bounds(k[:0].to(dev), v[:0].to(dev), gc, gb, loc[:0])  # no rows: nothing happens


# ---- scores ----
@pytest.mark.parametrize("hq,hkv,d,page,block", [(16, 2, 256, 64, 64), (16, 1, 64, 16, 16), (7, 7, 64, 64, 32),
                                                 (6, 2, 128, 96, 48), (32, 8, 128, 256, 256)])
def test_scores(dev, hq, hkv, d, page, block):
    lens = [0, 1, 16, 700, page, 0, 0, 3 * page + 1, 5] + [3] * 20
    c = make(lens, hq, hkv, d, page, seed=d)
    bounds = ob.key_bounds(c["cache"], empty_bounds(c, block, NAN), c["ptr"], c["idx"], c["last"])
    ref, mag = ob.block_scores(c["q"], bounds, c["ptr"], c["idx"], c["last"], page)
    got = axk.paged_block_scores(c["q"].to(dev), bounds.to(dev), *table(c, dev), page).cpu().double()
    assert torch.equal(got == -math.inf, ref == -math.inf)
    there = ref > -math.inf
    # fp32 sums of 2 D exact products, half of them zero: each addition is off by half a step of the sum of magnitudes
    assert ((got - ref).abs()[there] <= (2 * d * 2.0 ** -24 * mag)[there]).all()


def test_scores_leave_padding_alone_and_flag_bad_pages(dev):
    c = make([100, 33], 4, 2, 64, 32)
    bounds = ob.key_bounds(c["cache"], empty_bounds(c, 16, NAN), c["ptr"], c["idx"], c["last"])
    c["idx"][1] = 1 << 20
    idx = torch.cat([c["idx"], torch.zeros(5, dtype=torch.int32)])
    ref, _ = ob.block_scores(c["q"], bounds, c["ptr"], c["idx"], c["last"], 32)
    out = torch.full((2, idx.numel() * 2), 3.0, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    axk.paged_block_scores(c["q"].to(dev), bounds.to(dev), c["ptr"].to(dev), idx.to(dev), c["last"].to(dev), 32,
                           output=out, status=status)
    assert (out[:, -10:] == 3.0).all() and int(status) == 1 and (out[:, 2:4] == -math.inf).all()
    assert torch.equal(out[:, :-10].cpu() == -math.inf, ref == -math.inf)


def test_scores_keep_a_nan(dev):
    """A block with a NaN bound scores NaN, and its neighbours do not."""
    c = make([64], 4, 1, 64, 64)
    bounds = ob.key_bounds(c["cache"], empty_bounds(c, 16), c["ptr"], c["idx"], c["last"])
    bounds[c["idx"][0].long(), 2, 0, 1, 5] = NAN
    got = axk.paged_block_scores(c["q"].to(dev), bounds.to(dev), *table(c, dev), 64).cpu()
    assert got.isnan().tolist() == [[False, False, True, False]]


# ---- selection ----
@pytest.mark.parametrize("kind", ["normal", "equal", "few values", "special", "wide"])
@pytest.mark.parametrize("blocks,n,first,keep_last", [(1, 1, 0, 0), (40, 8, 1, 1), (300, 64, 2, 3), (300, 5, 5, 0),
                                                      (4500, 256, 1, 1), (20000, 1000, 0, 1), (40, 40, 1, 1)])
def test_select(dev, kind, blocks, n, first, keep_last):
    g = torch.Generator().manual_seed(blocks)
    page, block = 32, 16
    lens = [blocks * block - 3, max(1, blocks * block // 2), 0, 5]
    c = dict(ptr=[0], last=[])
    for x in lens:
        p = -(-x // page)
        c["ptr"].append(c["ptr"][-1] + p)
        c["last"].append(x - (p - 1) * page if p else 0)
    ptr, last = (torch.tensor(c[k], dtype=torch.int32) for k in ("ptr", "last"))
    s = torch.randn(3, int(ptr[-1]) * 2, generator=g)
    if kind == "equal":
        s = torch.zeros_like(s)
    elif kind == "few values":
        s = torch.round(s)  # -0.0 among them
    elif kind == "special":
        pick = torch.randint(0, 6, s.shape, generator=g)
        for i, x in enumerate((NAN, math.inf, -math.inf, -NAN)):
            s[pick == i] = x
    elif kind == "wide":
        s = s * torch.exp(20 * torch.randn(s.shape, generator=g))
    ref = ob.select_blocks(s, ptr, last, page, block, n, first, keep_last)
    got = axk.paged_select_blocks(s.to(dev), ptr.to(dev), last.to(dev), page, block, n, first, keep_last).cpu()
    assert torch.equal(got, ref)


# ---- decode ----
@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("hq,hkv,d,page,block,n", [(16, 2, 256, 64, 64, 9), (16, 1, 64, 16, 16, 40), (7, 7, 64, 64, 32, 3),
                                                   (6, 2, 128, 96, 48, 12), (32, 8, 128, 256, 128, 4),
                                                   (16, 2, 256, 64, 16, 200), (3, 1, 256, 4096, 16, 7), (16, 1, 256, 64, 32, 33)])
def test_decode_over_listed_blocks(dev, kv, hq, hkv, d, page, block, n):
    c = make([0, 1, 17, page + 2, 1500, 3200], hq, hkv, d, page, kv, seed=n)
    blocks = random_blocks(c, block, n)
    a, wa, status = check_decode(c, dev, blocks, block)
    assert status == 0
    b, wb, _ = check_decode(c, dev, blocks, block)
    assert torch.equal(a, b) and torch.equal(wa, wb)  # the same bits again
    x, _, _ = check_decode(c, dev, blocks, block, weights=False)
    if n * block > 128 * 16:  # the same cut either way
        assert torch.equal(a, x)


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 2, 256, 64), (16, 1, 64, 16), (7, 7, 64, 64), (6, 2, 128, 96),
                                           (16, 4, 256, 256)])
def test_decode_over_every_block(dev, kv, hq, hkv, d, page):
    c = make([0, 1, 16, page, 2 * page + 15, 0, 2500, 3], hq, hkv, d, page, kv, seed=page)
    out, _, status = check_decode(c, dev)
    assert status == 0 and not out[0].any() and not out[5].any()
    check_decode(c, dev, weights=False, sm_scale=0.01)
    check_decode(c, dev, win=False)


def test_decode_over_every_block_agrees_with_paged_decode(dev):
    c = make([700, 64, 3000], 16, 2, 256, 64)
    args = (c["q"].to(dev), c["cache"].to(dev), *table(c, dev))
    a, b = axk.paged_decode_blocks(*args), axk.paged_decode(*args)
    ref, _, slack, _ = ob.decode_blocks(c["q"], c["cache"], c["ptr"], c["idx"], c["last"])
    within(a, ref, slack + ref.abs() * 2.0 ** -8)
    torch.testing.assert_close(a.float(), b.float(), rtol=2e-2, atol=1e-2)
    torch.testing.assert_close(a.float().cpu(), paged_attn.paged_decode(c["q"], c["cache"], c["ptr"], c["idx"], c["last"],
                                                                        1 / 16).float(), rtol=2e-2, atol=1e-2)


@pytest.mark.parametrize("lens", [[0], [0, 0, 700], [700, 0]])
def test_decode_of_empty_sequences_beside_others(dev, lens):
    """Empty sequences yield zeros whatever the workspace or another sequence's values hold."""
    c = make(lens, 4, 2, 128, 32)
    check_decode(c, dev)
    check_decode(c, dev, random_blocks(c, 16, 40), 16)
    if max(lens):
        c["cache"][:, 1] = math.inf
        out = axk.paged_decode_blocks(c["q"].to(dev), c["cache"].to(dev), *table(c, dev)).cpu()
        for b, n in enumerate(lens):
            assert (out[b] == (math.inf if n else 0.0)).all()


@pytest.mark.parametrize("batch", [1, 63, 64, 300, 700])
def test_decode_many_short_sequences(dev, batch):
    rng = random.Random(batch)
    c = make([rng.choice([0, 1, 5, 16, 40, 130]) for _ in range(batch)], 4, 2, 64, 16, seed=batch)
    check_decode(c, dev)
    check_decode(c, dev, random_blocks(c, 16, 3), 16)


@pytest.mark.parametrize("page,block", [(64, 16), (4096, 16), (48, 48)])
def test_decode_over_a_long_list(dev, page, block):
    """Lists longer than the merge keeps in LDS (2048 blocks), whose pages straddle its rounds."""
    c = make([50000, 33, 40000], 2, 1, 64, page, seed=page)
    blocks = torch.full((3, 1, 50000 // block + 3), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(0)
    for b, n in enumerate(c["lens"]):
        nb = -(-n // block)
        got = torch.arange(nb)[torch.rand(nb, generator=g) < 0.9]
        blocks[b, 0, :len(got)] = got.int()
    check_decode(c, dev, blocks, block)


def test_decode_of_more_rows_than_run_at_once(dev):
    """520 (sequence, KV head) rows: pieces of 2048 tokens, in the listed form and over every block."""
    lens = [20] * 130
    lens[3], lens[70], lens[129] = 2100, 4500, 2048
    c = make(lens, 8, 4, 64, 64)
    check_decode(c, dev, random_blocks(c, 32, 150), 32)
    check_decode(c, dev)


def test_decode_skips_bad_pages_and_bad_lists(dev):
    c = make([300, 200], 4, 2, 64, 32)
    c["idx"][2], c["idx"][11] = -5, c["cache"].shape[0]
    blocks = random_blocks(c, 16, 8)
    _, _, status = check_decode(c, dev, weights=True)
    assert status == 1
    blocks[0, 0] = torch.tensor([0, 4, 4, 3, 6, 1 << 30, -7, 18])  # twice, falling, past the end, negative
    blocks[1, 1] = torch.tensor([1, 2, 3, 10, 12, 13, 5, -1])
    _, _, status = check_decode(c, dev, blocks, 16)
    assert status == 1
    blocks[:, :] = torch.tensor([2, 5, -1, 2, 5, -1, -1, 7])  # blocks behind padding, some of them twice
    _, _, status = check_decode(c, dev, blocks, 16, weights=True)
    assert status == 1
    c["idx"][:] = -1  # nothing left to attend
    out, w, status = check_decode(c, dev, blocks, 16)
    assert status == 1 and not out.any()


def test_offsets_that_fall_back_or_leave_the_table(dev):
    """Sequences overlap, run backwards or end past the table: nothing leaves an array, and what does not meet is right."""
    c = make([150, 150, 150, 150, 150, 150], 4, 2, 64, 32)
    nnz = c["idx"].numel()
    c["cache"].nan_to_num_(0.5)
    c["ptr"] = torch.tensor([0, 5, -4, 3, 2**31 - 1, 1, nnz], dtype=torch.int32)
    c["last"][:] = torch.tensor([32, 9, 40, -3, 5, 2**31 - 1], dtype=torch.int32)
    spans = [(0, 5), (5, 5), (0, 3), (3, nnz), (nnz, nnz), (1, nnz)]
    blocks = torch.tensor([0, 1, 3, 5, -1], dtype=torch.int32).expand(6, 2, 5).contiguous()
    t = table(c, dev)
    cache, q = c["cache"].to(dev), c["q"].to(dev)
    got = axk.paged_decode_blocks(q, cache, *t, blocks=blocks.to(dev), block_size=16)
    for b, (lo, hi) in enumerate(spans):
        last = min(max(int(c["last"][b]), 0), 32) if hi > lo else 0
        ref, _, slack, _ = ob.decode_blocks(c["q"][b:b + 1], c["cache"], torch.tensor([0, hi - lo]), c["idx"][lo:hi],
                                            torch.tensor([last]), blocks[b:b + 1], 16)
        within(got[b:b + 1], ref, slack + ref.abs() * 2.0 ** -8)
    w = torch.ones(2, nnz, device=dev)
    axk.paged_decode_blocks(q, cache, *t, weights_in=w, weights=w)
    bounds = axk.paged_key_bounds(cache, empty_bounds(c, 16).to(dev), *t)
    scores = axk.paged_block_scores(q, bounds, *t, 32)
    picked = axk.paged_select_blocks(scores, t[0], t[2], 32, 16, 4).cpu()
    for b, (lo, hi) in enumerate(spans):
        assert (picked[b] < 2 * (hi - lo)).all() and (picked[b] >= -1).all()
    p, i, ww, f = axk.paged_evict_pages(torch.rand(2, nnz, device=dev), t[0], t[1], 3)
    assert p.tolist() == [0, 3, 3, 6, 9, 9, 12]
    assert set(i.tolist()) <= set(c["idx"].tolist()) | {-1}


def test_evict_offsets_whose_sums_pass_32_bits(dev):
    n = 1 << 18
    ptr = torch.zeros(20001, dtype=torch.int32)
    ptr[1::2] = n  # 10000 sequences of the whole table, and as many that fall back
    idx = torch.arange(n, dtype=torch.int32, device=dev)
    for budget in (n, 300):
        p, i, w, f = axk.paged_evict_pages(torch.ones(1, n, device=dev), ptr.to(dev), idx, budget)
        assert p[:3].tolist() == [0, budget, budget]
        assert int(i.min()) >= -1 and int(i.max()) < n and int(f.min()) >= -1 and int(f.max()) < n


def test_decode_extreme_scores(dev):
    """Scores of thousands, all equal ones, and a sign-flipped scale."""
    c = make([500, 33], 16, 2, 128, 64)
    c["q"] *= 64
    check_decode(c, dev)
    check_decode(c, dev, sm_scale=-0.3)
    check_decode(c, dev, sm_scale=0.0)
    c["q"][:] = 0
    check_decode(c, dev, random_blocks(c, 32, 6), 32)


def test_a_last_page_without_a_token(dev):
    """last_page_len 0: the page counts for nothing, keeps its weight, and its blocks score -inf."""
    for lens in ([1024, 33, 64], [64, 2048]):
        c = make(lens, 6, 2, 64, 64)
        extra = c["cache"].shape[0] - c["idx"].numel()
        ptr, idx, free = [0], [], sorted(set(range(c["cache"].shape[0])) - set(c["idx"].tolist()))[:extra]
        for b, n in enumerate(lens):  # the first and last sequences get a page with nothing in it
            idx += c["idx"][int(c["ptr"][b]):int(c["ptr"][b + 1])].tolist()
            if b != 1 or len(lens) == 2:
                idx.append(free.pop())
                c["last"][b] = 0
            ptr.append(len(idx))
        idx.append(free.pop())  # and a sequence of one empty page
        c["ptr"] = torch.tensor(ptr + [len(idx)], dtype=torch.int32)
        c["idx"], c["last"] = torch.tensor(idx, dtype=torch.int32), torch.cat([c["last"], torch.zeros(1, dtype=torch.int32)])
        c["q"], c["lens"] = torch.cat([c["q"], c["q"][:1]]), lens + [0]
        out, _, status = check_decode(c, dev)
        assert status == 0 and not out[-1].any()
        check_decode(c, dev, random_blocks(c, 16, 9), 16)
        bounds = ob.key_bounds(c["cache"], empty_bounds(c, 32, 1.0), c["ptr"], c["idx"], c["last"])
        assert torch.equal(axk.paged_key_bounds(c["cache"].to(dev), empty_bounds(c, 32, 1.0).to(dev), *table(c, dev)).cpu(),
                           bounds)
        got = axk.paged_block_scores(c["q"].to(dev), bounds.to(dev), *table(c, dev), 64).cpu()
        ref, _ = ob.block_scores(c["q"], bounds, c["ptr"], c["idx"], c["last"], 64)
        assert torch.equal(got == -math.inf, ref == -math.inf)


def test_infinite_and_nan_rows_stay_where_they_are(dev):
    """Blocks that the list leaves out may hold anything; a NaN value that is attended reaches its own heads only."""
    c = make([640, 640], 4, 2, 64, 64)
    blocks = torch.tensor([[[0, 3, 9]] * 2] * 2, dtype=torch.int32)
    for b in range(2):
        for j in range(10):
            if j not in (0, 3, 9):
                c["cache"][c["idx"][int(c["ptr"][b]) + j].long()] = NAN if b else math.inf
    check_decode(c, dev, blocks, 64)
    c["cache"][c["idx"][3].long(), 1, 7, 1] = NAN  # sequence 0, KV head 1
    out = axk.paged_decode_blocks(c["q"].to(dev), c["cache"].to(dev), *table(c, dev), blocks=blocks.to(dev), block_size=64)
    assert out[0, 2:].isnan().all() and not out[0, :2].isnan().any() and not out[1].isnan().any()


def test_weights_in_place_and_padding_untouched(dev):
    c = make([100, 260], 6, 2, 128, 32)
    g = torch.Generator().manual_seed(0)
    nnz = c["idx"].numel()
    idx = torch.cat([c["idx"], torch.zeros(4, dtype=torch.int32)]).to(dev)
    blocks = random_blocks(c, 16, 5).to(dev)
    w0 = torch.rand(2, nnz + 4, generator=g).to(dev)
    for bl in (None, blocks):
        args = (c["q"].to(dev), c["cache"].to(dev), c["ptr"].to(dev), idx, c["last"].to(dev), bl, 16)
        w1 = torch.full_like(w0, 5.0)
        axk.paged_decode_blocks(*args, weights_in=w0, weights=w1, decay=0.5)
        assert (w1[:, nnz:] == 5.0).all() and not w1.isnan().any()
        w2 = w0.clone()
        axk.paged_decode_blocks(*args, weights_in=w2, weights=w2, decay=0.5)
        assert torch.equal(w2[:, :nnz], w1[:, :nnz]) and torch.equal(w2[:, nnz:], w0[:, nnz:])
        w3 = torch.empty_like(w0)
        axk.paged_decode_blocks(*args, weights=w3, decay=0.5)
        torch.testing.assert_close(w3[:, :nnz] + 0.5 * w0[:, :nnz], w1[:, :nnz], rtol=1e-6, atol=1e-7)


def test_offsets_past_32_bits(dev):
    """A 5.2 GB cache whose used pages lie at its end."""
    page, hkv, d = 64, 2, 256
    c = make([1000, 130], 16, hkv, d, page)
    pool, own = 40000, c["cache"].shape[0]
    cache = torch.empty(pool, 2, page, hkv, d, dtype=torch.bfloat16, device=dev)
    cache[pool - own:] = c["cache"].to(dev)
    bounds = torch.empty(pool, 4, hkv, 2, d, dtype=torch.bfloat16, device=dev)
    ptr, idx, last = table(c, dev)
    idx = idx + (pool - own)
    axk.paged_key_bounds(cache, bounds, ptr, idx, last)
    small = ob.key_bounds(c["cache"], empty_bounds(c, 16), c["ptr"], c["idx"], c["last"])
    used = c["idx"].long()
    full = torch.ones(used.numel(), 4, dtype=torch.bool)
    full[15], full[18, 1:] = torch.tensor([True, True, True, False]), False  # 1000 tokens end in block 62, 130 in 8
    assert torch.equal(bounds[pool - own:].cpu()[used][full], small[used][full])
    blocks = random_blocks(c, 16, 20)
    a = axk.paged_decode_blocks(c["q"].to(dev), cache, ptr, idx, last, blocks.to(dev), 16)
    b = axk.paged_decode_blocks(c["q"].to(dev), c["cache"].to(dev), *table(c, dev), blocks.to(dev), 16)
    assert torch.equal(a, b)
    loc = torch.tensor([[pool - 1, 63]], dtype=torch.int32, device=dev)
    k = torch.ones(1, hkv, d, dtype=torch.bfloat16, device=dev)
    axk.store_paged_kv_bounds(k, 2 * k, cache, bounds, loc)
    assert (cache[-1, 0, 63] == 1).all() and (cache[-1, 1, 63] == 2).all()


# ---- eviction ----
@pytest.mark.parametrize("hkv,pages,budget,first,keep_last", [
    (2, [0, 1, 5, 30, 100], 8, 1, 1), (1, [7], 7, 0, 1), (4, [3, 0, 0, 9000, 12], 512, 4, 2), (8, [50] * 70, 3, 1, 2),
    (2, [20, 21], 2, 1, 1), (3, [6000, 1], 5000, 0, 1), (2, [0, 0], 4, 1, 1)])
@pytest.mark.parametrize("kind", ["normal", "equal", "special"])
def test_evict(dev, kind, hkv, pages, budget, first, keep_last):
    g = torch.Generator().manual_seed(hkv)
    ptr = torch.tensor([sum(pages[:i]) for i in range(len(pages) + 1)], dtype=torch.int32)
    nnz = sum(pages)
    idx = torch.randperm(nnz + 5, generator=g)[:nnz].to(torch.int32)
    w = torch.exp(3 * torch.randn(hkv, nnz, generator=g))
    if kind == "equal":
        w = torch.round(w.clamp(max=1))
    elif kind == "special":
        w[torch.rand(w.shape, generator=g) < 0.2] = NAN
        w[torch.rand(w.shape, generator=g) < 0.1] = math.inf
    ref = ob.evict_pages(w, ptr, idx, budget, first, keep_last)
    got = axk.paged_evict_pages(w.to(dev), ptr.to(dev), idx.to(dev), budget, first, keep_last)
    for a, b in zip(got, ref):
        assert torch.equal(a.cpu().nan_to_num(-1.0), b.nan_to_num(-1.0))


def test_evict_a_table_with_room_to_spare(dev):
    ptr = torch.tensor([0, 10, 14], dtype=torch.int32)
    idx = torch.arange(20, dtype=torch.int32)
    w = torch.arange(40, dtype=torch.float32).view(2, 20)
    p, i, ww, f = (t.cpu() for t in axk.paged_evict_pages(w.to(dev), ptr.to(dev), idx.to(dev), 5))
    rp, ri, rw, rf = ob.evict_pages(w[:, :14].contiguous(), ptr, idx[:14], 5)
    assert torch.equal(p, rp) and torch.equal(i[:14], ri) and torch.equal(ww[:, :14], rw) and torch.equal(f[:14], rf)
    assert (i[14:] == -1).all() and not ww[:, 14:].any() and (f[14:] == -1).all()


# ---- together ----
@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
def test_decode_steps_with_eviction(dev, kv):
    """Prefilled sequences decoded for some steps: write, score, select, attend, add weights; then evicted and decoded on,
    every operator's result checked against the oracle on the state the GPU had before it."""
    page, block, hq, hkv, d, n = 32, 16, 8, 2, 128, 6
    lens = [150, 31, 96]
    c = make([x + 8 for x in lens], hq, hkv, d, page, kv)  # pages for what is to come
    cache, scale, kvs = c["cache"].to(dev), c["scale"], kv_of(c, dev)
    ptr, idx, _ = table(c, dev)
    last = torch.tensor([(x - 1) % page + 1 for x in lens], dtype=torch.int32, device=dev)
    ptr_used = torch.tensor([0] + [-(-x // page) for x in lens]).cumsum(0).int()
    rows = [c["idx"][int(c["ptr"][b]):int(c["ptr"][b + 1])].tolist() for b in range(3)]
    used = [r[:-(-x // page)] for r, x in zip(rows, lens)]
    ptr, idx = ptr_used.to(dev), torch.tensor(sum(used, []), dtype=torch.int32, device=dev)
    bounds = empty_bounds(c, block).to(dev)
    axk.paged_key_bounds(cache, bounds, ptr, idx, last, **kvs)
    w = torch.zeros(hkv, idx.numel(), device=dev)
    g = torch.Generator().manual_seed(9)
    for step in range(6):
        # the step's token: a new page where the last one is full, its weight zero
        used = [idx[int(ptr[b]):int(ptr[b + 1])].tolist() for b in range(3)]
        ws = [w[:, int(ptr[b]):int(ptr[b + 1])] for b in range(3)]
        for b in range(3):
            if int(last[b]) == page:
                fresh = next(p for p in rows[b] if p not in used[b])
                used[b].append(fresh)
                ws[b] = torch.cat([ws[b], torch.zeros(hkv, 1, device=dev)], 1)
                last[b] = 0
        last += 1
        ptr = torch.tensor([0] + [len(u) for u in used]).cumsum(0).int().to(dev)
        idx = torch.tensor(sum(used, []), dtype=torch.int32, device=dev)
        w = torch.cat(ws, 1).contiguous()
        k, v = (torch.randn(3, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
        q = (1.5 * torch.randn(3, hq, d, generator=g)).to(torch.bfloat16)
        loc = torch.tensor([[u[-1], int(last[b]) - 1] for b, u in enumerate(used)], dtype=torch.int32)
        rc, rb = ob.store(k, v, cache.cpu(), bounds.cpu(), loc, scale)
        axk.store_paged_kv_bounds(k.to(dev), v.to(dev), cache, bounds, loc.to(dev), **kvs)
        assert torch.equal(cache.cpu().view(torch.uint8), rc.view(torch.uint8)) and torch.equal(bounds.cpu(), rb)
        s = axk.paged_block_scores(q.to(dev), bounds, ptr, idx, last, page)
        blocks = axk.paged_select_blocks(s, ptr, last, page, block, n)
        assert torch.equal(blocks.cpu(), ob.select_blocks(s.cpu(), ptr.cpu(), last.cpu(), page, block, n))
        ref, rw, slack, wslack = ob.decode_blocks(q, cache.cpu(), ptr.cpu(), idx.cpu(), last.cpu(), blocks.cpu(), block,
                                                  None, w.cpu(), 0.9, scale)
        out = axk.paged_decode_blocks(q.to(dev), cache, ptr, idx, last, blocks, block, weights_in=w, weights=w, decay=0.9,
                                      **kvs)
        within(out, ref, slack + ref.abs() * 2.0 ** -8)
        within(w, rw, wslack)
        if step == 3:
            got = axk.paged_evict_pages(w, ptr, idx, 3)
            for a, b in zip(got, ob.evict_pages(w.cpu(), ptr.cpu(), idx.cpu(), 3)):
                assert torch.equal(a.cpu(), b)
            assert [int(x) for x in got[0]] == [0, 3, 5, 8]
            ptr, idx, w = got[0], got[1][:8].contiguous(), got[2][:, :8].contiguous()


def test_a_step_in_a_graph_replays_over_new_inputs(dev):
    """The whole step captured once and replayed over other queries, tokens and lengths, against eager calls; two graphs
    that share a workspace replay one after the other."""
    page, block, hq, hkv, d, n = 64, 16, 16, 2, 256, 24
    c = make([900, 3000, 65], hq, hkv, d, page)
    tab = table(c, dev)
    cache = c["cache"].to(dev).nan_to_num(0.0)
    bounds = axk.paged_key_bounds(cache, empty_bounds(c, block).to(dev), *tab)
    w = torch.zeros(hkv, tab[1].numel(), device=dev)
    ws = axk.paged_decode_blocks_workspace(3, hq, hkv, d, page, tab[1].numel(), dev, block, n, True)
    ws_all = axk.paged_decode_blocks_workspace(3, hq, hkv, d, page, tab[1].numel(), dev)
    q = c["q"].to(dev).clone()
    k, v = (torch.randn(3, hkv, d, device=dev).to(torch.bfloat16) for _ in range(2))
    loc = torch.stack([tab[1][tab[0][1:].long() - 1], tab[2] - 1], 1).contiguous()
    out, out_all = torch.empty_like(q), torch.empty_like(q)
    scores = torch.empty(hkv, tab[1].numel() * 4, device=dev)
    blocks = torch.empty(3, hkv, n, dtype=torch.int32, device=dev)

    def step(st):
        axk.store_paged_kv_bounds(k, v, st["cache"], st["bounds"], loc)
        axk.paged_block_scores(q, st["bounds"], *tab, page, output=scores)
        axk.paged_select_blocks(scores, tab[0], tab[2], page, block, n, output=blocks)
        axk.paged_decode_blocks(q, st["cache"], *tab, blocks, block, output=out, weights_in=st["w"], weights=st["w"],
                                workspace=ws)
        axk.paged_decode_blocks(q, st["cache"], *tab, output=out_all, workspace=ws_all)

    mine = dict(cache=cache, bounds=bounds, w=w)
    other = {x: t.clone() for x, t in mine.items()}
    step({x: t.clone() for x, t in mine.items()})
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(mine)
        graphs.append(graph)
    g = torch.Generator().manual_seed(3)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g).to(torch.bfloat16))
        k.copy_(torch.randn(k.shape, generator=g).to(torch.bfloat16))
        if i == 2:
            tab[2][0] -= 1  # a sequence one token shorter
        graphs[i % 2].replay()
        got = [t.clone() for t in (out, out_all, blocks, mine["w"], mine["bounds"])]
        step(other)
        torch.cuda.synchronize()
        for a, b in zip(got, (out, out_all, blocks, other["w"], other["bounds"])):
            assert torch.equal(a, b)


def test_on_a_stream_of_its_own(dev):
    c = make([500, 90], 16, 2, 128, 64)
    blocks = random_blocks(c, 32, 6).to(dev)
    args = (c["q"].to(dev), c["cache"].to(dev), *table(c, dev), blocks, 32)
    a = axk.paged_decode_blocks(*args)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        b = axk.paged_decode_blocks(*args)
    st.synchronize()
    assert torch.equal(a, b)


def test_an_empty_table(dev):
    q = torch.randn(2, 4, 64, device=dev).to(torch.bfloat16)
    cache = torch.full((3, 2, 32, 2, 64), NAN, dtype=torch.bfloat16, device=dev)
    ptr = torch.zeros(3, dtype=torch.int32, device=dev)
    idx, last = torch.empty(0, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    w = torch.empty(2, 0, device=dev)
    assert not axk.paged_decode_blocks(q, cache, ptr, idx, last, weights=w).any()
    s = axk.paged_block_scores(q, torch.zeros(3, 2, 2, 2, 64, dtype=torch.bfloat16, device=dev), ptr, idx, last, 32)
    bl = axk.paged_select_blocks(s, ptr, last, 32, 16, 4)
    assert tuple(s.shape) == (2, 0) and (bl == -1).all()
    assert not axk.paged_decode_blocks(q, cache, ptr, idx, last, bl, 16, weights=w).any()
    p, i, ww, f = axk.paged_evict_pages(w, ptr, idx, 4)
    assert not p.any() and i.numel() == ww.numel() == f.numel() == 0


# ---- what the bounds promise ----
@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("hq,hkv,d,page,block", [(6, 2, 64, 32, 16), (8, 8, 128, 96, 48), (16, 1, 256, 64, 64)])
def test_bounds_contain_the_keys_and_scores_bound_the_products(dev, kv, hq, hkv, d, page, block):
    """In every kind of cache, from the cache and at the write: lo <= key <= hi for the keys as attention reads them, and
    q . k <= score but for the roundings of the score's fp32 sum."""
    lens = [1, 16, block + 1, 2 * page + 3, 500]
    c = make(lens, hq, hkv, d, page, kv, seed=3)
    bounds = axk.paged_key_bounds(c["cache"].to(dev), empty_bounds(c, block).to(dev), *table(c, dev), **kv_of(c, dev))
    # the same keys written again, row by row
    loc = torch.tensor([[int(c["idx"][int(c["ptr"][b]) + t // page]), t % page] for b, n in enumerate(lens)
                        for t in range(n)], dtype=torch.int32)
    k = torch.randn(len(loc), hkv, d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    cache, kvs, folded = c["cache"].to(dev), kv_of(c, dev), empty_bounds(c, block).to(dev)
    axk.store_paged_kv_bounds(k.to(dev), k.to(dev), cache, folded, loc.to(dev), **kvs)
    again = dict(c, cache=cache.cpu(), scale=kvs["kv_scales"].cpu() if kv == "i8" else c["scale"])
    for x, got in ((c, bounds), (again, folded)):
        scores = axk.paged_block_scores(c["q"].to(dev), got, *table(c, dev), page).cpu().double()
        got = got.cpu()
        _, mag = ob.block_scores(c["q"], got, c["ptr"], c["idx"], c["last"], page)
        for b, n in enumerate(lens):
            key, _, _ = ob.seq_rows(x["cache"], c["ptr"], c["idx"], c["last"], b, x["scale"])
            t = torch.arange(n)
            e, s = int(c["ptr"][b]) + t // page, t % page // block
            bb = got[c["idx"][e].long(), s].double()
            assert (bb[:, :, 0] <= key).all() and (key <= bb[:, :, 1]).all()
            prod = (c["q"][b].double().view(1, hkv, hq // hkv, d) * key[:, :, None]).sum(3).amax(2)
            at = e * (page // block) + s
            assert (prod.t() <= scores[:, at] + 2 * d * 2.0 ** -24 * mag[:, at]).all()


def test_int8_scales_that_are_not_finite(dev):
    """A key that is NaN makes both bounds of its channel NaN, at the write as from the cache; infinite keys stay."""
    page, hkv, d = 32, 2, 64
    codes = torch.randint(-127, 128, (2, 2, page, hkv, d), generator=torch.Generator().manual_seed(1), dtype=torch.int8)
    codes[0, 0, 3, 0, :4] = torch.tensor([0, 5, -5, 0], dtype=torch.int8)
    scales = torch.full((2, 2, page, hkv), 0.0625, dtype=torch.bfloat16)
    scales[0, 0, 3, 0] = math.inf  # keys NaN, inf, -inf, NaN, ...
    scales[1, 0, 20, 1] = NAN
    ptr, idx, last = (torch.tensor(x, dtype=torch.int32) for x in ([0, 2], [0, 1], [page]))
    empty = torch.zeros(2, 2, hkv, 2, d, dtype=torch.bfloat16)
    ref = ob.key_bounds(codes, empty, ptr, idx, last, kv_scale=scales)
    got = axk.paged_key_bounds(codes.to(dev), empty.to(dev), ptr.to(dev), idx.to(dev), last.to(dev),
                               kv_scales=scales.to(dev)).cpu()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(0.5), ref.nan_to_num(0.5))
    assert got[0, 0, 0, :, 0].isnan().all() and got[1, 1, 1].isnan().all()
    assert got[0, 0, 0, 1, 1] == math.inf and got[0, 0, 0, 0, 2] == -math.inf
    # a row with an infinite value is stored with an infinite scale: code 0 where it was finite
    k = torch.randn(16, hkv, d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    k[5, 1, 7] = math.inf
    loc = torch.tensor([[1, t] for t in range(16)], dtype=torch.int32, device=dev)
    gc, gs, gb = codes.to(dev), scales.to(dev), empty.to(dev)
    axk.store_paged_kv_bounds(k.to(dev), k.to(dev), gc, gb, loc, kv_scales=gs)
    one = torch.tensor([0, 1], dtype=torch.int32)
    ref = ob.key_bounds(gc.cpu(), empty, one, idx[1:], torch.tensor([16], dtype=torch.int32), kv_scale=gs.cpu())
    assert torch.equal(gb[1, 0].cpu().isnan(), ref[1, 0].isnan()) and ref[1, 0].isnan().any()
    assert torch.equal(gb[1, 0].cpu().nan_to_num(0.5), ref[1, 0].nan_to_num(0.5))


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (7, 1, 128), (32, 2, 256)])
def test_scores_of_infinite_bounds(dev, hq, hkv, d):
    """max(q lo, q hi) is finite, or infinite, where one bound is infinite; NaN only where q is zero there or infinities of
    both signs meet. The other blocks of a tile and the other heads are not touched."""
    page, block = 64, 16
    c = make([500, 40], hq, hkv, d, page, seed=d)
    bounds = ob.key_bounds(c["cache"], empty_bounds(c, block), c["ptr"], c["idx"], c["last"])
    p = c["idx"].long()
    c["q"][:, :, :4] = torch.tensor([2.0, -2.0, 0.0, 1.0]).to(torch.bfloat16)
    bounds[p[0], 0, :, 0, 0] = -math.inf  # finite: the other bound decides
    bounds[p[0], 1, :, 1, 1] = math.inf   # finite
    bounds[p[0], 2, :, 1, 0] = math.inf   # +inf
    bounds[p[0], 3, :, :, 0] = -math.inf  # -inf
    bounds[p[1], 0, :, 0, 2] = -math.inf  # 0 * inf
    bounds[p[1], 1, :, 1, 0], bounds[p[1], 1, :, 1, 1] = math.inf, -math.inf
    bounds[p[1], 1, :, 0, 1] = -math.inf  # +inf twice
    bounds[p[1], 2, :, 1, 0], bounds[p[1], 2, :, :, 3] = math.inf, -math.inf  # inf - inf
    bounds[p[1], 3, 0, 0, 0] = -math.inf  # one KV head only
    ref, mag = ob.block_scores(c["q"], bounds, c["ptr"], c["idx"], c["last"], page)
    got = axk.paged_block_scores(c["q"].to(dev), bounds.to(dev), *table(c, dev), page).cpu().double()
    assert ref[0, [0, 1, 7]].isfinite().all() and ref[0, 2] == ref[0, 5] == math.inf and ref[0, 3] == -math.inf
    assert ref[0, 4].isnan() and ref[0, 6].isnan()
    there = ref.isfinite()
    assert torch.equal(got[~there].nan_to_num(0.5), ref[~there].nan_to_num(0.5))
    assert ((got - ref).abs()[there] <= (2 * d * 2.0 ** -24 * mag)[there]).all()


@pytest.mark.parametrize("weights", [False, True])
def test_lists_that_name_a_block_again(dev, weights):
    """Behind a fall of the list, or behind padding and a block that is skipped, a block may come a second time: flagged, and
    attended again."""
    c = make([300, 200], 4, 2, 64, 32)
    blocks = torch.tensor([[[0, 5, 2, 5, 7, -1], [3, 9, -1, 4, 9, 11]], [[6, 2, 6, 7, 3, 7], [1, 1, 2, 2, 12, 0]]], dtype=torch.int32)
    _, _, status = check_decode(c, dev, blocks, 16, weights=weights)
    assert status == 1
    long = blocks.repeat(1, 1, 40)  # over several pieces
    _, _, status = check_decode(c, dev, long, 16, weights=weights)
    assert status == 1
