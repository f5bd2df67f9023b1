"""Trees of drafted tokens where decays vanish, a piece of the cache holds nothing or no number for a row, and pages lie outside
the pool; on the GPU against the 64-bit oracle."""
import math

import pytest
import torch

import axk
from oracle import tree as ot

from test_gpu_tree import BF16_HALF, GDN, NAN, U, attend, chain, check_tree, gdn_case, tree_case, within

pytestmark = pytest.mark.gpu

# node 1 is followed by 3 and 6; 2, 4, 5 and the rest are other branches, in the same tile of 16 nodes and in later ones
FORGETS = [-1, 0, 0, 1, 2, -1, 3] + [5 if i % 2 else 4 for i in range(7, 40)]


def forgetting(t, value, where=1):
    """A case whose node `where` has the gate input `value`, and the same with a decay of e^-300 there: no state or update that
    it meets leaves a trace in 64 bits either (the values are below 10, a double's half step 2^-53)."""
    c = gdn_case(2, t, 1, 2, trees=[FORGETS[:t], chain(t, t)], seed=t)
    c["a_log"], c["dt_bias"] = torch.full((2,), -0.5), torch.zeros(2)
    c["a"][:, where, 1] = value
    ref = dict(c, a=c["a"].clone())
    ref["a"][:, where, 1] = 300.0 * math.exp(0.5)
    return c, ref


@pytest.mark.parametrize("value", [math.inf, 3e38, 1e20, 1e9])
@pytest.mark.parametrize("t", [7, 20, 40])
def test_a_decay_to_nothing_stays_in_its_branch(dev, t, value):
    """e^-inf is zero, as in the recurrence: the node and its descendants know nothing of what came before it, other branches are
    as they were."""
    c, finite = forgetting(t, value)
    o, u, g = (x.cpu() for x in axk.gdn_tree_verify(*(c[n].to(dev) for n in GDN)))
    (ro, ru, rg), (eo, eu, eg) = ot.gdn_tree(*(finite[n] for n in GDN))
    within(u, ru, eu, U)
    within(o, ro, eo, BF16_HALF)
    assert (g[:, 1, 1] < -5e8).all()
    g[:, 1, 1], rg[:, 1, 1], eg[:, 1, 1] = 0.0, 0.0, 0.0
    within(g, rg, eg, U)


def test_a_chain_with_a_decay_to_nothing_is_the_recurrence(dev):
    c, finite = forgetting(20, math.inf, where=9)
    c["parents"] = torch.tensor([chain(20, 20)] * 2, dtype=torch.int32)
    o = axk.gdn_tree_verify(*(c[n].to(dev) for n in GDN))[0].double().cpu()
    ro = axk.gdn_recurrent(*(c[n].to(dev) for n in GDN[:-1]))[0].double().cpu()
    finite["parents"] = c["parents"]
    eo = ot.gdn_tree(*(finite[n] for n in GDN))[1][0]
    # both are within their fp32 errors of the same values, then rounded: a bf16 step apart at most
    assert not ro.isnan().any() and ((o - ro).abs() <= 2 * eo + 2.01 * BF16_HALF * ro.abs()).all()


@pytest.mark.parametrize("name", ["a", "v"])
def test_nan_is_not_forgotten(dev, name):
    """0 times NaN: what is no number before such a decay stays none behind it, as in the recurrence."""
    c, _ = forgetting(20, math.inf, where=3)
    ref = axk.gdn_tree_verify(*(c[n].to(dev) for n in GDN))
    c[name][0, 1, 1] = NAN
    got = axk.gdn_tree_verify(*(c[n].to(dev) for n in GDN))
    inside = [t for t, m in enumerate(ot.branches(FORGETS[:20])) if 1 in m]
    outside = [t for t in range(20) if t not in inside]
    assert 3 in inside and 6 in inside
    for x, y in zip(got[:2], ref[:2]):
        assert torch.equal(x[0, outside], y[0, outside]) and torch.equal(x[1], y[1])
        assert x[0, inside, 1].isnan().all() and torch.equal(x[0, inside, 0], y[0, inside, 0])


@pytest.mark.parametrize("value", [-math.inf, -3e38, -1e20, -105.0])
def test_commit_of_a_branch_with_a_decay_to_nothing(dev, value):
    c = gdn_case(3, 20, 1, 2, trees=[chain(20, 20)] * 3, seed=3)
    g = torch.Generator().manual_seed(7)
    u, gt = torch.randn(c["v"].shape, generator=g), -torch.rand(c["a"].shape, generator=g)
    gt[0, 5, 1], gt[1, 19, 0], gt[2, 0] = value, value, value
    gt[2, 7, 0] = value
    acc = torch.tensor([19, 19, 9], dtype=torch.int32)
    finite = gt.clamp(min=-300.0)
    ref, err = ot.gdn_commit(c["state"], c["k"], u, finite, c["parents"], acc)
    got = axk.gdn_tree_commit(*(x.to(dev) for x in (c["state"], c["k"], u, gt, c["parents"], acc)))
    within(got, ref, err, U)
    u[0, 2, 1, 3], u[0, 10, 0, 4] = NAN, NAN  # before the decay, and of the other head
    bad = axk.gdn_tree_commit(*(x.to(dev) for x in (c["state"], c["k"], u, gt, c["parents"], acc)))
    assert bad[0, 1, :, 3].isnan().all() and bad[0, 0, :, 4].isnan().all()
    bad[0, 1, :, 3], bad[0, 0, :, 4] = got[0, 1, :, 3], got[0, 0, :, 4]
    assert torch.equal(bad, got)


# ---- attention ----
def where(c, b, pos):
    """(page, slot) of a cached token."""
    page = c["cache"].shape[2]
    return int(c["idx"][int(c["ptr"][b]) + pos // page]), pos % page


def put(c, b, pos, plane, value):
    """A cached row (fp8: its bytes, i8: its scale) of every head set to `value`, NaN or a number."""
    p, s = where(c, b, pos)
    if isinstance(c["scale"], torch.Tensor):
        c["scale"][p, plane, s] = value
    else:
        c["cache"][p, plane, s] = 0x7F if c["cache"].dtype is torch.uint8 else value


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("t,hq,hkv,d,hist", [(64, 4, 4, 64, 500), (64, 8, 4, 64, 500), (64, 2, 2, 128, 500),
                                             (64, 4, 2, 128, 500), (64, 16, 2, 128, 2932), (64, 2, 2, 256, 884),
                                             (64, 16, 2, 256, 2932)])
def test_a_key_that_is_no_number_behind_a_cut(dev, kv, t, hq, hkv, d, hist):
    """A row that sees nothing but one NaN score in a piece is NaN, whatever the other pieces hold; rows that do not see the key
    stay as they were. (Pieces of 128 tokens: the last one begins with node 12.)"""
    tree = chain(t, t)
    tree[50] = -1
    tree[51:] = [49 - i for i in range(t - 51)]  # nobody behind it sees node 50
    c = tree_case([hist], [t], t, hq, hkv, d, 16, kv, seed=d, trees=[tree])
    ref = attend(c, dev)
    put(c, 0, hist + 50, 0, NAN)
    got = attend(c, dev)
    assert got[0, 50].isnan().all()
    rest = [i for i in range(t) if i != 50]
    assert not ref.isnan().any() and torch.equal(got[0, rest], ref[0, rest])


@pytest.mark.parametrize("hist", [60, 500])  # whole and cut
def test_a_value_that_is_no_number_counts_whatever_its_weight(dev, hist):
    """0 times NaN: also where a whole piece's weights are zero in 32 bits."""
    c = tree_case([hist], [3], 3, 4, 2, 64, 16, trees=[[-1, 0, -1]])
    c["q"].fill_(1.0)
    c["cache"][:, 0] = 8.0
    for pos in range(32 if hist < 128 else 128):  # a pair of tiles, or a piece
        put(c, 0, pos, 0, -8.0)  # scores of -512 against 512: weights of e^-1024
    p, s = where(c, 0, 10)
    c["cache"][p, 1, s, :, 5] = NAN
    got = attend(c, dev, 1.0)
    assert got[..., 5].isnan().all()
    got[..., 5] = 0.0
    assert not got.isnan().any()


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("t,hq,hkv,d", [(4, 4, 4, 64), (20, 4, 1, 64), (6, 6, 2, 128), (20, 8, 2, 128), (20, 16, 1, 128),
                                        (5, 16, 2, 256), (20, 8, 2, 256)])
def test_pages_outside_the_pool_in_short_caches(dev, kv, t, hq, hkv, d):
    """Sequences and last pieces of one or two pairs of tiles, in which any page lies outside the pool; no row of the pool's first
    page may be read in its place."""
    for total in (t + 3, 30, 32, 50, 64, 528, 550):
        for at in sorted({0, 1, (total - 1) // 16 - 1, (total - 1) // 16}):
            if not 0 <= at <= (total - 1) // 16 or total < t:
                continue
            c = tree_case([total - t], [t], t, hq, hkv, d, 16, kv, seed=total)
            for i, pid in enumerate(c["idx"].tolist()):  # page 0 is nobody's
                if pid == 0:
                    c["idx"][i] = next(x for x in range(1, c["cache"].shape[0]) if x not in c["idx"].tolist())
                    c["cache"][c["idx"][i]] = c["cache"][0]
                    if kv == "i8":
                        c["scale"][c["idx"][i]] = c["scale"][0]
            if kv == "i8":
                c["cache"][0], c["scale"][0] = 1, NAN
            else:
                c["cache"][0] = 0x7F if kv == "fp8" else NAN
            c["idx"][at] = -1 if total % 4 else c["cache"].shape[0]
            check_tree(c, dev, want_status=1)


def pieces(dev, lens, hkv, d):
    """The pieces that a batch is cut into, by what they leave in a workspace: each row's maximum, sum and output."""
    n = len(lens)
    c = tree_case(lens, [1] * n, 1, hkv, hkv, d, 64)
    ws = axk.paged_tree_verify_workspace(n, 1, hkv, hkv, d, dev)
    ws.fill_(255)
    out = attend(c, dev, ws=ws)
    assert not out.isnan().any()
    left = int((ws[:ws.numel() // 4 * 4].view(torch.int32) != -1).sum())
    assert left % (hkv * (d + 2)) == 0
    return left // (hkv * (d + 2))


@pytest.mark.parametrize("batch", [1, 20, 40, 64, 65, 200])
def test_a_long_sequence_is_cut_beside_any_number_of_short_ones(dev, batch):
    """64 pieces of eight KV heads run at once: of 32768 tokens beside sequences of 40, the share that their work has, to within
    a factor of two (sequences of two pairs of tiles are not cut)."""
    pairs = 1025 + 2 * (batch - 1)
    assert 64 * 1025 / pairs / 2 - 1 <= pieces(dev, [32768] + [40] * (batch - 1), 8, 64) <= 64


def test_rows_past_what_a_merge_launch_holds(dev):
    """2^24 rows of nodes in a batch that is not cut."""
    few = tree_case([3, 0, 17, 40], [64, 9, 64, 30], 64, 1, 1, 64, 16)
    ref = attend(few, dev).cpu()
    n = 1 << 16  # times the four
    up = {x: few[x].to(dev) for x in ("q", "cache", "idx", "last", "parents", "ptr")}
    ptr = torch.cat([(up["ptr"][:4] + int(few["ptr"][4]) * torch.arange(n, device=dev)[:, None]).flatten().to(torch.int32),
                     torch.tensor([n * int(few["ptr"][4])], dtype=torch.int32, device=dev)])
    got = axk.paged_tree_verify(up["q"].repeat(n, 1, 1, 1), up["cache"], ptr, up["idx"].repeat(n), up["last"].repeat(n),
                                up["parents"].repeat(n, 1))
    assert torch.equal(got[:4].cpu(), ref) and torch.equal(got[-4:].cpu(), ref)
    assert (got.view(n, -1) == got[:4].view(1, -1)).all()
