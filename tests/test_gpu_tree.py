"""Rows appended with the rotation on the way, attention of drafted trees and the delta rule along their branches on the GPU,
against the 64-bit oracle."""
import math
import random

import pytest
import torch

import axk
from axk import configs
from oracle import paged_attn
from oracle import tree as ot

pytestmark = pytest.mark.gpu
NAN = math.nan
U = 2.0 ** -24


def random_tree(n, t, seed=0):
    rng = random.Random(seed)
    if not n:
        return [-2] * t
    return [-1] + [i - 1 if rng.random() < 0.5 else rng.randrange(-1, i) for i in range(1, n)] + [-2] * (t - n)


def chain(n, t):
    return list(range(-1, n - 1)) + [-2] * (t - n)


def within(got, ref, err, half):
    """Every value within the error bound and half a step (relative) of its own type."""
    got, ref = got.double().cpu(), ref.double()
    assert not got.isnan().any()
    tol = err * (1 + half) + ref.abs() * half
    bad = (got - ref).abs() > tol * 1.001 + 1e-37
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float(((got - ref).abs() / (tol + 1e-37)).max())}"


BF16_HALF = 2.0 ** -8


# ---- rows into the cache ----
def rope_case(rows, hq, hkv, d, rot, page, kv, table=torch.float32, norm=True, seed=0, n=300):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(rows, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16)
    pool = -(-rows // page) + 3
    at = torch.randperm(pool * page, generator=g)[:rows]
    ang = torch.rand(n, rot // 2, generator=g) * 6.28
    x = torch.randn(pool, 2, page, hkv, d, generator=g).to(torch.bfloat16)
    scales = None
    if kv == "fp8":
        x = x.to(torch.float8_e4m3fn).view(torch.uint8)
    elif kv == "i8":
        x, scales = paged_attn.quant_kv_i8(x)
    return dict(qkv=qkv, loc=torch.stack([at // page, at % page], 1).to(torch.int32), cos=ang.cos().to(table),
                sin=ang.sin().to(table), pos=torch.randint(0, n, (rows,), generator=g, dtype=torch.int32), cache=x, scales=scales,
                kn=1 + 0.2 * torch.randn(d, generator=g) if norm else None,
                qn=1 + 0.2 * torch.randn(d, generator=g) if norm else None, hq=hq, hkv=hkv, d=d, rot=rot, page=page, kv=kv)


def split(c, x):
    r, hq, hkv, d = x.shape[0], c["hq"], c["hkv"], c["d"]
    return (x[:, :hq * d].view(r, hq, d), x[:, hq * d:(hq + hkv) * d].view(r, hkv, d), x[:, (hq + hkv) * d:].view(r, hkv, d))


def check_rope(dev, c, kv_scale=4.0, queries=True, want_status=0):
    up = lambda x: None if x is None else x.to(dev)  # noqa: E731
    q, k, v = split(c, c["qkv"].to(dev))
    cache, scales = c["cache"].to(dev), up(c["scales"])
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    q_out = torch.full((q.shape[0], c["hq"], c["d"]), 7.0, dtype=torch.bfloat16, device=dev) if queries else None
    got = axk.store_paged_kv_rope(k, v, cache, up(c["loc"]), up(c["cos"]), up(c["sin"]), up(c["pos"]), k_norm=up(c["kn"]),
                                  q=q if queries else None, q_norm=up(c["qn"]) if queries else None, q_out=q_out,
                                  kv_scale=kv_scale if c["kv"] == "fp8" else None, kv_scales=scales, status=status)
    assert got is q_out and int(status) == want_status
    hq, hkv = split(c, c["qkv"])[0:2]
    vv = split(c, c["qkv"])[2]
    p = c["pos"].clamp(0, c["cos"].shape[0] - 1).long()
    cs, sn = (c["cos"][p], c["sin"][p]) if c["rot"] else (None, None)
    there = (c["pos"] >= 0) & (c["pos"] < c["cos"].shape[0])
    kept = there & (c["loc"][:, 0] >= 0) & (c["loc"][:, 0] < cache.shape[0]) & (c["loc"][:, 1] >= 0) & (c["loc"][:, 1] < c["page"])
    if queries:
        ref, err = ot.rope_rows(hq, c["qn"], cs, sn, 1e-6)
        within(q_out[there.to(dev)], ref[there], err[there], BF16_HALF)
        assert (q_out[~there.to(dev)] == 7.0).all()
    ref, err = ot.rope_rows(hkv, c["kn"], cs, sn, 1e-6)
    page, slot = c["loc"][kept, 0].long(), c["loc"][kept, 1].long()
    after, before = cache.cpu(), c["cache"]
    mask = torch.zeros(after.shape[0], after.shape[2], dtype=torch.bool)
    mask[page, slot] = True
    rest = ~mask[:, None, :, None, None].expand_as(after)
    assert torch.equal(after[rest].view(torch.uint8), before[rest].view(torch.uint8))
    k_got, v_got = after[page, 0, slot], after[page, 1, slot]
    if c["kv"] == "bf16":
        within(k_got, ref[kept], err[kept], BF16_HALF)
        assert torch.equal(v_got, vv[kept])
    elif c["kv"] == "fp8":
        x = (ref[kept] * kv_scale)
        # half a step of 2^-4 relative, or of 2^-9 absolute below the smallest normal value
        got8 = k_got.view(torch.float8_e4m3fn).double()
        assert ((got8 - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) + err[kept] * kv_scale * 2).all()
        assert torch.equal(v_got, (vv[kept].float() * kv_scale).to(torch.float8_e4m3fn).view(torch.uint8))
    else:
        s = scales.cpu()
        codes, ss = paged_attn.quant_kv_i8(vv[kept])
        assert torch.equal(v_got, codes) and torch.equal(s[page, 1, slot], ss)
        sk = s[page, 0, slot].double()
        am = ref[kept].abs().amax(-1)
        # the scale is bf16(max(amax, 1e-5) / 127): 1 / 127 and the product each rounded to bf16
        assert ((sk - am.clamp(min=1e-5) / 127).abs() <= am.clamp(min=1e-5) / 127 * 2.02 * BF16_HALF).all()
        # a code is off by half a unit, by the two roundings of 1 / s and of the product (|code| <= 129), by fp32's
        assert ((k_got.double() - ref[kept] / sk[..., None]).abs() <= 0.5 + 2.1 * BF16_HALF * 129 + 1e-3).all()
        other = s.clone()
        other[page, :, slot] = c["scales"][page, :, slot]
        assert torch.equal(other, c["scales"])
    return q_out


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("rows,hq,hkv,d,rot,page,table,norm", [
    (1, 16, 2, 256, 64, 64, torch.bfloat16, True), (16, 4, 4, 64, 64, 16, torch.float32, True),
    (37, 6, 2, 128, 128, 96, torch.float32, False), (5, 7, 7, 64, 16, 16, torch.bfloat16, False),
    (130, 32, 4, 256, 256, 256, torch.float32, True), (9, 1, 1, 128, 32, 1, torch.float32, True)])
def test_append(dev, rows, hq, hkv, d, rot, page, table, norm, kv):
    check_rope(dev, rope_case(rows, hq, hkv, d, rot, page, kv, table, norm, seed=rows))


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
def test_append_left_out_rows_and_bad_ones(dev, kv):
    c = rope_case(12, 4, 2, 128, 64, 16, kv, seed=3)
    c["loc"][2, 0] = -1        # not stored, its query is
    c["pos"][4] = -1           # no row
    c["loc"][5] = -1
    c["pos"][5] = -1
    check_rope(dev, c)
    for where, value in (("loc", (c["cache"].shape[0], 0)), ("loc", (-2, 0)), ("loc", (0, 16)), ("loc", (0, -1)),
                         ("pos", 300), ("pos", -2), ("pos", 2 ** 31 - 1)):
        x = dict(c, loc=c["loc"].clone(), pos=c["pos"].clone())
        x[where][7] = torch.tensor(value, dtype=torch.int32)
        check_rope(dev, x, want_status=1)


def test_append_without_rotation_queries_or_positions(dev):
    c = rope_case(20, 2, 2, 128, 64, 16, "bf16", seed=5)
    check_rope(dev, c, queries=False)
    q, k, v = split(c, c["qkv"].to(dev))
    cache = c["cache"].to(dev)
    axk.store_paged_kv_rope(k, v, cache, c["loc"].to(dev))  # a plain append
    ref = c["cache"].to(dev)
    axk.store_paged_kv(k.contiguous(), v.contiguous(), ref, c["loc"].to(dev))
    assert torch.equal(cache, ref)
    a = axk.store_paged_kv_rope(k, v, cache, c["loc"].to(dev), c["cos"].to(dev), c["sin"].to(dev), q=q)
    b = axk.store_paged_kv_rope(k, v, cache, c["loc"].to(dev), c["cos"].to(dev), c["sin"].to(dev),
                                torch.arange(20, dtype=torch.int32, device=dev), q=q)
    assert torch.equal(a, b)


def test_append_is_qk_norm_rope_and_store(dev):
    """The framework's separate calls round after the norm, after the rotation and when storing: within those roundings."""
    c = rope_case(33, 16, 2, 256, 64, 64, "bf16", torch.bfloat16, seed=7)
    got = check_rope(dev, c)
    q, _, _ = split(c, c["qkv"].to(dev))
    cos, sin = (c[x][c["pos"].long()].to(dev) for x in ("cos", "sin"))
    ref = axk.glue.qk_norm_rope(q.contiguous(), c["qn"].to(dev), cos, sin, 64)
    # two bf16 roundings there against one here, each at most half a step of the row's largest magnitude, sqrt(2) of it turned
    mag = ref.float().abs().amax(-1, keepdim=True)
    assert ((got.float() - ref.float()).abs() <= 4 * BF16_HALF * mag).all()


def test_append_gated_query_heads(dev):
    """q as the first halves of [q | gate] heads: a head stride of 2 D."""
    c = rope_case(6, 4, 2, 128, 64, 16, "bf16", seed=9)
    q, k, v = split(c, c["qkv"].to(dev))
    qg = torch.full((6, 4, 256), NAN, dtype=torch.bfloat16, device=dev)
    qg[..., :128] = q
    args = (c["loc"].to(dev), c["cos"].to(dev), c["sin"].to(dev), c["pos"].to(dev))
    cache = c["cache"].to(dev)
    a = axk.store_paged_kv_rope(k, v, cache, *args, q=qg[..., :128], q_norm=c["qn"].to(dev))
    b = axk.store_paged_kv_rope(k, v, cache, *args, q=q, q_norm=c["qn"].to(dev))
    assert torch.equal(a, b)


# ---- attention ----
def tree_case(lens, counts, t, hq, hkv, d, page, kv="bf16", seed=0, trees=None, extra=3):
    """Histories of lens tokens with trees of counts nodes behind them; slots that no token has hold NaN."""
    g = torch.Generator().manual_seed(seed)
    total = [x + n for x, n in zip(lens, counts)]
    pages = [-(-x // page) for x in total]
    pool = sum(pages) + extra
    idx = torch.randperm(pool, generator=g)[:sum(pages)].to(torch.int32)
    ptr = torch.tensor([sum(pages[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    last = torch.tensor([x - (p - 1) * page if p else 0 for x, p in zip(total, pages)], dtype=torch.int32)
    x = torch.randn(pool, 2, page, hkv, d, generator=g).to(torch.bfloat16)
    x[:, 0] *= torch.exp(0.5 * torch.randn(hkv, d, generator=g)).to(torch.bfloat16)
    used = torch.zeros(pool, page, dtype=torch.bool)
    for b, n in enumerate(total):
        for i in range(n):
            used[int(idx[int(ptr[b]) + i // page]), i % page] = True
    scale = None
    if kv == "fp8":
        scale = 8.0
        x = (x * scale).to(torch.float8_e4m3fn).view(torch.uint8)
        x.masked_fill_(~used[:, None, :, None, None], 0x7F)
    elif kv == "bf16":
        x.masked_fill_(~used[:, None, :, None, None], NAN)
    else:
        x, scale = paged_attn.quant_kv_i8(x)
        x = x.masked_fill(~used[:, None, :, None, None], 127)
        scale.masked_fill_(~used[:, None, :, None], NAN)
    trees = trees or [random_tree(n, t, seed * 100 + i) for i, n in enumerate(counts)]
    q = (1.5 * torch.randn(len(lens), t, hq, d, generator=g)).to(torch.bfloat16)
    return dict(q=q, cache=x, ptr=ptr, idx=idx, last=last, parents=torch.tensor(trees, dtype=torch.int32), scale=scale)


def kv_of(c, dev):
    s = c["scale"]
    return {"kv_scales": s.to(dev)} if isinstance(s, torch.Tensor) else {"kv_scale": s}


def attend(c, dev, sm_scale=None, status=None, ws=None):
    b, t, hq, d = c["q"].shape
    if ws is None:
        ws = axk.paged_tree_verify_workspace(b, t, hq, c["cache"].shape[3], d, dev)
        ws.fill_(255)  # NaNs: nothing may be read that the call has not written
    return axk.paged_tree_verify(c["q"].to(dev), c["cache"].to(dev), c["ptr"].to(dev), c["idx"].to(dev), c["last"].to(dev),
                                 c["parents"].to(dev), sm_scale=sm_scale, status=status, workspace=ws, **kv_of(c, dev),
                                 output=torch.full_like(c["q"], NAN, device=dev))


def check_tree(c, dev, sm_scale=None, want_status=0):
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = attend(c, dev, sm_scale, status)
    ref, err = ot.tree_attention(c["q"], c["cache"], c["ptr"], c["idx"], c["last"], c["parents"], sm_scale, c["scale"])
    within(out, ref, err, BF16_HALF)
    assert int(status) == want_status
    return out


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("t,hq,hkv,d,page", [(1, 16, 2, 256, 64), (3, 4, 4, 64, 16), (8, 16, 2, 256, 16), (13, 6, 2, 128, 96),
                                             (64, 7, 7, 64, 32), (33, 16, 1, 64, 16), (9, 32, 2, 128, 48), (17, 8, 2, 256, 256),
                                             (64, 4, 2, 128, 16), (5, 16, 1, 256, 32)])
def test_trees(dev, kv, t, hq, hkv, d, page):
    """Histories from none on, whole and partial tiles and pages, the longest one cut into pieces; trees of every size."""
    lens = [0, 1, page, 2 * page - 1, 16 * 37 + 5, 1500]
    counts = [t, max(1, t // 2), 1, t, (t + 1) // 2, t]
    check_tree(tree_case(lens, counts, t, hq, hkv, d, page, kv, seed=t), dev)


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
def test_no_nodes_no_pages_and_holes(dev, kv):
    trees = [[-2] * 5, [-1, -2, 0, 0, -2], [-2, -1, 1, -2, -2], [-1, 0, 1, 2, 3], [-2, -2, -2, -2, -1]]
    counts = [0, 4, 3, 5, 5]
    check_tree(tree_case([40, 33, 0, 17, 300], counts, 5, 4, 2, 128, 16, kv, trees=trees), dev)
    check_tree(tree_case([0, 0], [0, 0], 4, 4, 2, 64, 16, kv), dev)  # padded sequences: no page at all


def test_bad_parents_are_no_nodes(dev):
    trees = [[-1, 1, 0, 2], [-1, -3, 1, 0], [0, 0, -1, 2], [-1, 9, -2, 2]]
    check_tree(tree_case([20, 20, 20, 20], [4, 4, 4, 4], 4, 4, 2, 64, 16, trees=trees), dev, want_status=1)


def test_pages_outside_the_pool_and_short_caches(dev):
    c = tree_case([70, 600], [4, 4], 4, 4, 2, 64, 16)
    c["idx"][1], c["idx"][20] = -1, c["cache"].shape[0]
    check_tree(c, dev, want_status=1)
    c = tree_case([70, 3], [4, 4], 4, 4, 2, 64, 16)
    c["last"][1] = 3  # three cached tokens for four nodes
    check_tree(c, dev, want_status=1)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales_of_any_sign(dev, scale):
    c = tree_case([50, 700], [6, 6], 6, 4, 2, 64, 16)
    if scale == 3.0:  # sharp: small products, as fp32's error of a score grows with it
        c["q"] *= 0.25
    check_tree(c, dev, scale)


def test_infinite_and_nan_keys_behind_masks(dev):
    """What a node does not see leaves no trace, whatever it holds."""
    trees = [[-1, 0, 0, 1]]
    c = tree_case([30], [4], 4, 4, 2, 64, 16, trees=trees)
    where = lambda t: (int(c["idx"][t // 16]), t % 16)  # noqa: E731
    ref = attend(c, dev)
    for value in (NAN, math.inf, -math.inf, 3e38):
        p, s = where(32)  # node 2: nobody's ancestor
        x = dict(c, cache=c["cache"].clone())
        x["cache"][p, :, s] = value
        got = attend(x, dev)
        assert torch.equal(got[0, [0, 1, 3]], ref[0, [0, 1, 3]])


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
def test_nan_in_a_branch_stays_there(dev, kv):
    """A node whose value is no number makes those of its descendants none, and only those."""
    trees = [[-1, 0, 0, 1, 2, -1, 5]]
    c = tree_case([70], [7], 7, 4, 2, 128, 32, kv, trees=trees)
    ref = attend(c, dev)
    p, s = int(c["idx"][72 // 32]), 72 % 32  # node 2, ancestor of 4
    if kv == "i8":
        c["scale"][p, 1, s] = NAN
    else:
        c["cache"][p, 1, s, :, 5] = NAN if kv == "bf16" else 0x7F
    got = attend(c, dev)
    assert torch.equal(got[0, [0, 1, 3, 5, 6]], ref[0, [0, 1, 3, 5, 6]])
    assert got[0, [2, 4], :, 5].isnan().all()
    if kv != "i8":
        keep = [d for d in range(128) if d != 5]
        assert torch.equal(got[0, [2, 4]][..., keep], ref[0, [2, 4]][..., keep])


def test_chain_is_prefill(dev):
    g = torch.Generator().manual_seed(0)
    c = configs.prefill_case([12, 12], [900, 40], 8, 2, 128, 16, g, extra_pages=2)
    x = {n: c[n].to(dev) for n in ("q", "cache", "qo_indptr", "indptr", "indices", "last_page_len")}
    ref = axk.paged_prefill(*x.values())
    parents = torch.tensor([chain(12, 12)] * 2, dtype=torch.int32, device=dev)
    got = axk.paged_tree_verify(x["q"].view(2, 12, 8, 128), x["cache"], x["indptr"], x["indices"], x["last_page_len"], parents)
    # both are off by their bf16 probabilities and their own rounding
    out, err = ot.tree_attention(c["q"].view(2, 12, 8, 128), c["cache"], c["indptr"], c["indices"], c["last_page_len"],
                                 parents.cpu())
    within(ref.view_as(got), out, err, BF16_HALF)
    within(got, out, err, BF16_HALF)


@pytest.mark.parametrize("batch", [1, 63, 64, 65, 150])
def test_batches(dev, batch):
    """Sequences are looked up 64 at a time."""
    rng = random.Random(batch)
    lens = [rng.choice([0, 3, 40, 300, 800]) for _ in range(batch)]
    check_tree(tree_case(lens, [rng.randint(0, 3) for _ in lens], 3, 2, 1, 64, 16, seed=batch), dev)


def test_repeats_bit_by_bit_and_leaves_the_rest(dev):
    c = tree_case([2000, 100], [9, 4], 9, 16, 2, 256, 64)
    a = attend(c, dev)
    for _ in range(3):
        assert torch.equal(a, attend(c, dev))
    idx = torch.cat([c["idx"], torch.full((40,), 1 << 30, dtype=torch.int32)])  # a table with room to spare
    assert torch.equal(a, attend(dict(c, idx=idx), dev))


def test_offsets_past_the_table_are_clamped(dev):
    c = tree_case([100, 40], [4, 4], 4, 4, 2, 64, 16)
    ref = attend(c, dev)
    c["ptr"][2] = 1000  # the last sequence up to the table's end
    assert torch.equal(attend(c, dev), ref)


# ---- the delta rule ----
def gdn_case(bsz, t, nk, nv, counts=None, trees=None, seed=0, state_std=0.3):
    g = torch.Generator().manual_seed(seed)
    c = configs.gdn_inputs(bsz, t, g, nk=nk, nv=nv, state_std=state_std)
    c["a_log"], c["dt_bias"] = 0.5 * torch.randn(nv, generator=g), 0.5 * torch.randn(nv, generator=g)
    counts = counts or [t] + [random.Random(seed + i).randint(0, t) for i in range(1, bsz)]
    trees = trees or [random_tree(n, t, seed * 77 + i) for i, n in enumerate(counts)]
    c["parents"] = torch.tensor(trees, dtype=torch.int32)
    return c


GDN = ("q", "k", "v", "a", "b", "a_log", "dt_bias", "state", "parents")


def check_gdn(c, dev, want_status=0):
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    full = lambda x, dt: torch.full(x.shape, NAN, dtype=dt, device=dev)  # noqa: E731
    state = c["state"].to(dev)
    o, u, g = axk.gdn_tree_verify(*(state if n == "state" else c[n].to(dev) for n in GDN), output=full(c["v"], torch.bfloat16),
                                  updates=full(c["v"], torch.float32), gates=full(c["a"], torch.float32), status=status)
    (ro, ru, rg), (eo, eu, eg) = ot.gdn_tree(*(c[n] for n in GDN))
    within(g, rg, eg, U)
    within(u, ru, eu, U)
    within(o, ro, eo, BF16_HALF)
    assert torch.equal(state.cpu(), c["state"]) and int(status) == want_status
    return o, u, g


@pytest.mark.parametrize("bsz,t,nk,nv", [(1, 1, 1, 1), (1, 8, 2, 4), (3, 16, 2, 2), (2, 17, 1, 3), (2, 33, 2, 4), (1, 64, 1, 2),
                                         (40, 5, 2, 4), (33, 20, 1, 4), (34, 40, 4, 4)])
def test_gdn_trees(dev, bsz, t, nk, nv):
    """Trees of one, two and four 16-node tiles, few heads (single-wave workgroups) and many."""
    check_gdn(gdn_case(bsz, t, nk, nv, seed=t), dev)


def test_gdn_chain_is_the_recurrence(dev):
    c = gdn_case(2, 48, 2, 4, trees=[chain(48, 48)] * 2)
    o, u, g = check_gdn(c, dev)
    ro, rs = axk.gdn_recurrent(*(c[n].to(dev) for n in GDN[:-1]))
    # both outputs are within their fp32 errors of the same values, then rounded: a bf16 step apart at most
    (_, _, _), (eo, _, _) = ot.gdn_tree(*(c[n] for n in GDN))
    assert ((o.double() - ro.double()).abs().cpu() <= 2 * eo + 2.01 * BF16_HALF * ro.double().abs().cpu()).all()
    last = torch.tensor([47, 47], dtype=torch.int32, device=dev)
    s = axk.gdn_tree_commit(c["state"].to(dev), c["k"].to(dev), u, g, c["parents"].to(dev), last)
    torch.testing.assert_close(s, rs, rtol=1e-4, atol=1e-5)


def test_gdn_holes_bad_parents_and_garbage_rows(dev):
    trees = [[-2] * 6, [-1, -2, 0, 0, -2, -2], [-2, -1, 1, 1, 2, -2]]
    c = gdn_case(3, 6, 1, 2, trees=trees)
    check_gdn(c, dev)
    for n in ("q", "k", "v", "a", "b"):  # rows of no node hold anything
        for b, tree in enumerate(trees):
            for t, p in enumerate(tree):
                if p == -2:
                    c[n][b, t] = NAN
    o, u, g = (x.cpu() for x in axk.gdn_tree_verify(*(c[n].to(dev) for n in GDN)))
    assert not o.isnan().any() and not u.isnan().any() and not g.isnan().any()
    check_gdn(gdn_case(2, 4, 1, 2, trees=[[-1, 1, 0, 2], [-1, -7, 1, 0]]), dev, want_status=1)


@pytest.mark.parametrize("t", [7, 40])
@pytest.mark.parametrize("name", ["k", "v", "a", "b"])
@pytest.mark.parametrize("value", [NAN, math.inf])
def test_gdn_nan_in_a_branch_stays_there(dev, name, value, t):
    if name in "ab" and value == math.inf:
        value = -NAN
    tree = [-1, 0, 0, 1, 2, -1, 5] + [4 if i % 2 else 3 for i in range(7, t)]
    c = gdn_case(1, t, 1, 2, trees=[tree])
    ref = axk.gdn_tree_verify(*(c[n].to(dev) for n in GDN))
    c[name][0, 2, ..., -1] = value  # node 2, one channel or head
    got = axk.gdn_tree_verify(*(c[n].to(dev) for n in GDN))
    inside = [i for i, m in enumerate(ot.branches(tree)) if 2 in m]
    outside = [i for i in range(t) if i not in inside]
    for x, y in zip(got, ref):
        assert torch.equal(x[0, outside], y[0, outside])
    for x in got[:2]:
        assert x[0, inside][..., -1, -1].isnan().all()


def test_gdn_extreme_gates(dev):
    """Decays that vanish and that keep everything, and a zero state."""
    c = gdn_case(2, 20, 1, 2, trees=[chain(20, 20), random_tree(20, 20, 3)])
    c["a"][0] = 30.0
    c["a"][1] = -30.0
    c["b"][:, ::3] = 20.0
    c["b"][:, 1::3] = -20.0
    check_gdn(c, dev)
    check_gdn(gdn_case(1, 12, 1, 2, state_std=0.0), dev)


@pytest.mark.parametrize("bsz,t,nk,nv", [(1, 1, 1, 1), (3, 8, 2, 4), (5, 64, 1, 2), (2, 30, 2, 6)])
def test_commit(dev, bsz, t, nk, nv):
    c = gdn_case(bsz, t, nk, nv, counts=[t] * bsz, seed=t)
    g = torch.Generator().manual_seed(3)
    u, gt = torch.randn(c["v"].shape, generator=g), -torch.rand(c["a"].shape, generator=g) * 3
    acc = torch.tensor([t - 1] + [random.Random(i).randint(-1, t - 1) for i in range(1, bsz)], dtype=torch.int32)
    ref, err = ot.gdn_commit(c["state"], c["k"], u, gt, c["parents"], acc)
    args = [x.to(dev) for x in (c["k"], u, gt, c["parents"], acc)]
    state = c["state"].to(dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    got = axk.gdn_tree_commit(state, *args, status=status)
    within(got, ref, err, U)
    assert torch.equal(state.cpu(), c["state"])
    assert axk.gdn_tree_commit(state, *args, state_out=state) is state and torch.equal(state, got)
    assert int(status) == 0


def test_commit_of_no_node(dev):
    c = gdn_case(4, 6, 1, 2, trees=[chain(6, 6), chain(3, 6), chain(6, 6), chain(6, 6)])
    u, gt = torch.randn(c["v"].shape), -torch.rand(c["a"].shape)
    state = c["state"].to(dev)
    for acc, flagged in (([-1, 2, -1, 5], 0), ([5, 4, -1, 5], 1), ([5, 2, 6, 5], 1), ([5, 2, 5, -2], 1)):
        acc = torch.tensor(acc, dtype=torch.int32)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        got = axk.gdn_tree_commit(state, *(x.to(dev) for x in (c["k"], u, gt, c["parents"], acc)), status=status)
        ref, err = ot.gdn_commit(c["state"], c["k"], u, gt, c["parents"], acc)
        within(got, ref, err, U)
        assert int(status) == flagged
