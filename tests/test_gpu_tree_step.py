"""The tree operators as they are used: a step of one attention and one GDN layer from the drafted tokens to the accepted branch,
in graphs, on several streams at once, over caches longer than 32-bit offsets and over long pieces, against the 64-bit oracle."""
import math
import random

import pytest
import torch

import axk
from axk import configs
from oracle import tree as ot

from test_gpu_tree import (BF16_HALF, GDN, NAN, attend, check_gdn, check_tree, gdn_case, random_tree, tree_case,
                           within)

pytestmark = pytest.mark.gpu


def path_to(tree, node):
    out = []
    while node >= 0:
        out.append(node)
        node = tree[node]
    return out[::-1]


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
def test_step_from_drafts_to_the_accepted_branch(dev, kv):
    """Two steps: each appends the drafted rows, verifies them in both layers, accepts a node per sequence, moves the branch's
    rows to their final slots and commits the states. Afterwards the cache holds what appending the accepted tokens alone would
    hold, bit by bit, and the states are those of the recurrence over them."""
    bsz, t, hq, hkv, d, rot, page, nk, nv = 3, 9, 8, 2, 128, 64, 16, 2, 4
    g = torch.Generator().manual_seed(5)
    hist, npages = [37, 0, 100], 12  # pages a sequence
    pool = bsz * npages + 1
    pages = torch.randperm(pool, generator=g)[:bsz * npages].view(bsz, npages)
    cos, sin = torch.randn(400, rot // 2, generator=g).to(dev), torch.randn(400, rot // 2, generator=g).to(dev)
    norm = torch.rand(d, generator=g).to(dev) + 0.5
    kw = {}
    if kv == "bf16":
        cache = torch.zeros(pool, 2, page, hkv, d, dtype=torch.bfloat16, device=dev)
    elif kv == "fp8":
        cache, kw = torch.zeros(pool, 2, page, hkv, d, dtype=torch.uint8, device=dev), dict(kv_scale=8.0)
    else:
        cache = torch.zeros(pool, 2, page, hkv, d, dtype=torch.int8, device=dev)
        kw = dict(kv_scales=torch.zeros(pool, 2, page, hkv, dtype=torch.bfloat16, device=dev))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    kw["status"] = status
    slot = lambda b, pos: (int(pages[b, pos // page]), pos % page)  # noqa: E731
    draw = lambda rows, h: torch.randn(rows, h, d, generator=g).to(torch.bfloat16).to(dev)  # noqa: E731

    def append(k, v, loc, pos, **more):
        return axk.store_paged_kv_rope(k, v, cache, torch.tensor(loc, dtype=torch.int32, device=dev).view(-1, 2), cos, sin,
                                       torch.tensor(pos, dtype=torch.int32, device=dev), k_norm=norm, **more, **kw)

    kept = [(draw(n, hkv), draw(n, hkv)) for n in hist]  # every sequence's tokens so far
    for b, n in enumerate(hist):
        append(*kept[b], [slot(b, i) for i in range(n)], list(range(n)))
    gdn = configs.gdn_inputs(bsz, t, g, nk=nk, nv=nv, state_std=0.3)
    a_log, dt_bias = (0.5 * torch.randn(nv, generator=g)).to(dev), torch.randn(nv, generator=g).to(dev)
    state = gdn["state"].to(dev)
    for step in range(2):
        counts = [t, 4, 6] if step == 0 else [5, t, 1]
        trees = [random_tree(n, t, 10 * step + b) for b, n in enumerate(counts)]
        depth = [[len(path_to(tr, i)) - 1 if tr[i] != -2 else -1 for i in range(t)] for tr in trees]
        k, v, q = draw(bsz * t, hkv), draw(bsz * t, hkv), draw(bsz * t, hq)
        loc = [slot(b, hist[b] + i) if i < counts[b] else (-1, 0) for b in range(bsz) for i in range(t)]
        pos = [hist[b] + depth[b][i] if i < counts[b] else -1 for b in range(bsz) for i in range(t)]
        qr = append(k, v, loc, pos, q=q, q_norm=norm)
        total = [hist[b] + counts[b] for b in range(bsz)]
        used = [-(-x // page) for x in total]
        ptr = torch.tensor([sum(used[:b]) for b in range(bsz + 1)], dtype=torch.int32)
        idx = torch.cat([pages[b, :used[b]] for b in range(bsz)]).to(torch.int32)
        last = torch.tensor([x - (p - 1) * page for x, p in zip(total, used)], dtype=torch.int32)
        par = torch.tensor(trees, dtype=torch.int32)
        qr = torch.nan_to_num(qr).view(bsz, t, hq, d)
        out = axk.paged_tree_verify(qr, cache, ptr.to(dev), idx.to(dev), last.to(dev), par.to(dev), **kw)
        sc = kw.get("kv_scale", kw["kv_scales"].cpu() if kv == "i8" else None)
        within(out, *ot.tree_attention(qr.cpu(), cache.cpu(), ptr, idx, last, par, None, sc), BF16_HALF)
        x = {n: v.to(dev) for n, v in configs.gdn_inputs(bsz, t, g, nk=nk, nv=nv, state_std=0.3).items()}
        o, upd, gates = axk.gdn_tree_verify(x["q"], x["k"], x["v"], x["a"], x["b"], a_log, dt_bias, state, par.to(dev),
                                            status=status)
        # a node per sequence, one of them none
        accepted = [random.Random(step * 7 + b).randrange(n) for b, n in enumerate(counts)]
        accepted[step] = -1
        branch = [path_to(trees[b], accepted[b]) for b in range(bsz)]
        loc2, pos2 = [(-1, 0)] * (bsz * t), [-1] * (bsz * t)
        for b in range(bsz):
            for i, n in enumerate(branch[b]):
                loc2[b * t + n], pos2[b * t + n] = slot(b, hist[b] + i), hist[b] + i
        append(k, v, loc2, pos2)
        new = axk.gdn_tree_commit(state, x["k"], upd, gates, par.to(dev), torch.tensor(accepted, dtype=torch.int32, device=dev),
                                  status=status)
        for b in range(bsz):
            rows = torch.tensor(branch[b], dtype=torch.long, device=dev)
            if len(rows):
                one = lambda n: x[n][b:b + 1, rows].contiguous()  # noqa: E731
                ro, rs = axk.gdn_recurrent(one("q"), one("k"), one("v"), one("a"), one("b"), a_log, dt_bias, state[b:b + 1])
                torch.testing.assert_close(new[b], rs[0], rtol=1e-4, atol=1e-5)
                torch.testing.assert_close(o[b, rows].float(), ro[0].float(), rtol=4 * BF16_HALF, atol=1e-5)
            else:
                assert torch.equal(new[b], state[b])
            flat = rows + b * t
            kept[b] = (torch.cat([kept[b][0], k[flat]]), torch.cat([kept[b][1], v[flat]]))
            hist[b] += len(rows)
        state = new
    got = [[cache[slot(b, i)[0], :, slot(b, i)[1]].clone() for i in range(hist[b])] for b in range(bsz)]
    cache.zero_()
    for b in range(bsz):
        append(*kept[b], [slot(b, i) for i in range(hist[b])], list(range(hist[b])))
        for i in range(hist[b]):
            assert torch.equal(got[b][i], cache[slot(b, i)[0], :, slot(b, i)[1]])
    assert int(status) == 0


def test_captured_and_replayed(dev):
    """A step's operators in one graph, replayed with other inputs and the program's own work between; two graphs that share a
    workspace, replayed one after the other."""
    c1, c2 = tree_case([900, 40], [9, 4], 9, 16, 2, 256, 64), tree_case([300, 1200], [5, 9], 9, 16, 2, 256, 64, seed=3)
    gd = gdn_case(2, 9, 2, 4, seed=3)
    ws = axk.paged_tree_verify_workspace(2, 9, 16, 2, 256, dev)
    acc = torch.tensor([3, -1], dtype=torch.int32, device=dev)

    def step(c, x):
        out = axk.paged_tree_verify(c["q"], c["cache"], c["ptr"], c["idx"], c["last"], c["parents"], workspace=ws)
        o, u, g = axk.gdn_tree_verify(*(x[n] for n in GDN))
        return out, o, u, g, axk.gdn_tree_commit(x["state"], x["k"], u, g, x["parents"], acc)

    cases = [{n: v.to(dev) for n, v in c.items() if isinstance(v, torch.Tensor)} for c in (c1, c2)]
    x = {n: gd[n].to(dev) for n in GDN}
    step(cases[0], x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(c, x))
        graphs.append(graph)
    for i in range(4):
        for c in cases:
            c["q"].copy_(torch.roll(c["q"], 1, -1))
            c["parents"].copy_(torch.tensor([random_tree(9, 9, i), random_tree(4, 9, i)], dtype=torch.int32))
        x["v"].mul_(1.25)
        for graph, out in zip(graphs, outs):
            for y in out:
                y.fill_(NAN)
            graph.replay()
        torch.cuda.synchronize()
        for c, out in zip(cases, outs):
            for y, ref in zip(out, step(c, x)):
                assert torch.equal(y, ref)
        torch.cuda.synchronize()


def test_two_streams_at_once(dev):
    """Calls on two streams, each with its workspace, interleaved; inputs made on another stream than the calls'."""
    cs = [tree_case([5000], [8], 8, 16, 2, 256, 64, seed=i) for i in range(2)]
    refs = [attend(c, dev) for c in cs]
    on = [{n: v.to(dev) for n, v in c.items() if isinstance(v, torch.Tensor)} for c in cs]
    ws = [axk.paged_tree_verify_workspace(1, 8, 16, 2, 256, dev) for _ in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x = on[i]
                outs[i].append(axk.paged_tree_verify(x["q"], x["cache"], x["ptr"], x["idx"], x["last"], x["parents"],
                                                     workspace=ws[i]))
    torch.cuda.synchronize()
    for ref, out in zip(refs, outs):
        assert all(torch.equal(ref, o) for o in out)


@pytest.mark.parametrize("kv,hq,hkv,d", [("bf16", 16, 2, 256), ("fp8", 16, 2, 256), ("i8", 16, 2, 128), ("bf16", 8, 1, 64),
                                         ("fp8", 8, 1, 128), ("i8", 16, 1, 256)])
@pytest.mark.parametrize("t", [2, 12, 40])
def test_long_pieces(dev, kv, hq, hkv, d, t):
    """Pieces of many whole pairs, pages of 16 tokens (64 at a time are at hand), and pages outside the pool inside them."""
    c = tree_case([9000, 4100, 30], [t, (t + 1) // 2, 1], t, hq, hkv, d, 16, kv, seed=t)
    check_tree(c, dev)
    c["idx"][[3, 200, 201, 420, 650]] = torch.tensor([-1, 1 << 30, -7, c["cache"].shape[0], -1], dtype=torch.int32)
    check_tree(c, dev, want_status=1)


@pytest.mark.parametrize("kv", ["bf16", "fp8", "i8"])
@pytest.mark.parametrize("t,hq,hkv,d", [(16, 16, 2, 64), (16, 8, 1, 128), (25, 5, 1, 128), (8, 16, 2, 256), (8, 8, 1, 64),
                                        (64, 4, 1, 64), (64, 16, 4, 128), (43, 3, 1, 256)])
@pytest.mark.parametrize("lens", [[500, 33], [40, 0, 9]])
def test_row_blocks_filled_to_the_last_row(dev, kv, t, hq, hkv, d, lens):
    """Every row of a block is a node's: 64, 125 to 129 and 256 of them; in several pieces and in one."""
    check_tree(tree_case(lens, [t] * len(lens), t, hq, hkv, d, 16, kv, seed=t), dev)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("t,hq,d", [(12, 16, 128), (12, 4, 128), (12, 16, 256), (40, 16, 64), (40, 16, 128), (16, 16, 64)])
def test_nan_and_infinite_values_behind_a_long_history(dev, kv, t, hq, d):
    """Values of nodes that are no numbers, where a sequence is cut into pieces and the nodes lie in several pages: the rows that
    see them get them, no other row does."""
    c = tree_case([6001, 700], [t, t], t, hq, 2, d, 16, kv, seed=1, trees=[random_tree(t, t, 4), random_tree(t, t, 9)])
    ref = attend(c, dev).cpu()
    bad = {}
    for b, length in enumerate((6001, 700)):
        for n, val in ((2, math.inf), (7, NAN)):
            pos = length + n
            p = int(c["idx"][int(c["ptr"][b]) + pos // 16])
            c["cache"][p, 1, pos % 16, 0, 5] = 0x7F if kv == "fp8" else val
            bad[b, n] = NAN if kv == "fp8" else val
    got = attend(c, dev).cpu()
    g = hq // 2
    for b in range(2):
        for n in range(t):
            seen = set(path_to(c["parents"][b].tolist(), n))
            hit = [v for (bb, m), v in bad.items() if bb == b and m in seen]
            col = got[b, n, :g, 5]
            if not hit:
                assert torch.equal(got[b, n], ref[b, n])
            elif any(math.isnan(v) for v in hit):
                assert torch.isnan(col).all()
            else:
                assert (col == math.inf).all()
            if hit:
                rest = torch.ones(hq, d, dtype=torch.bool)
                rest[:g, 5] = False
                assert torch.equal(got[b, n][rest], ref[b, n][rest])


@pytest.mark.parametrize("kv", ["bf16", "i8"])
def test_pools_past_32_bit_offsets(dev, kv):
    """Pages behind the first 4 GiB of a pool, appended to and attended."""
    hkv, d, page, t, hq = 4, 256, 256, 5, 8
    per = 2 * page * hkv * d * (2 if kv == "bf16" else 1)
    pool = (5 << 30) // per
    c = tree_case([700], [t], t, hq, hkv, d, page, kv, seed=2, extra=0)
    n = c["cache"].shape[0]
    cache = torch.empty((pool, *c["cache"].shape[1:]), dtype=c["cache"].dtype, device=dev)
    cache[pool - n:] = c["cache"].to(dev)
    idx = (c["idx"] + (pool - n)).to(dev)
    kw = {}
    if kv == "i8":
        scales = torch.empty((pool, *c["scale"].shape[1:]), dtype=torch.bfloat16, device=dev)
        scales[pool - n:] = c["scale"].to(dev)
        kw = dict(kv_scales=scales)
    # the drafted rows once more, at their places: the pool's last pages change, and nothing else
    k, v = torch.randn(t, hkv, d).to(torch.bfloat16).to(dev), torch.randn(t, hkv, d).to(torch.bfloat16).to(dev)
    loc = torch.tensor([[pool - n + int(c["idx"][(700 + i) // page]), (700 + i) % page] for i in range(t)], dtype=torch.int32)
    axk.store_paged_kv_rope(k, v, cache, loc.to(dev), **kw)
    out = axk.paged_tree_verify(c["q"].to(dev), cache, c["ptr"].to(dev), idx, c["last"].to(dev), c["parents"].to(dev), **kw)
    small = dict(c, cache=cache[pool - n:].cpu())
    if kv == "i8":
        small["scale"] = scales[pool - n:].cpu()
    assert not torch.equal(small["cache"], c["cache"])
    within(out, *ot.tree_attention(c["q"], small["cache"], c["ptr"], c["idx"], c["last"], c["parents"], None, small["scale"]),
           BF16_HALF)


@pytest.mark.parametrize("bsz,t,nk,nv", [(33, 5, 2, 8), (257, 16, 1, 1), (2, 16, 16, 32)])
def test_gdn_many_heads(dev, bsz, t, nk, nv):
    """Short trees of more heads than single-wave workgroups are taken for, and of as many as they are."""
    check_gdn(gdn_case(bsz, t, nk, nv, seed=t), dev)


@pytest.mark.parametrize("batch,longest", [(90, 200), (200, 2500), (256, 60), (257, 60), (700, 12)])
def test_large_batches(dev, batch, longest):
    """Sequences left whole because they are even, cut although they are many, and too many to be cut."""
    rng = random.Random(batch)
    lens = [longest] + [rng.randint(longest // 2, longest) if batch < 100 else rng.randint(0, 40) for _ in range(batch - 1)]
    check_tree(tree_case(lens, [rng.randint(0, 2) for _ in lens], 2, 4, 2, 64, 16, seed=batch), dev)


def test_no_rows_and_one_node(dev):
    """Nothing to append; a batch of nodes alone, without history; a chain of one."""
    cache = torch.zeros(2, 2, 16, 1, 64, dtype=torch.bfloat16, device=dev)
    none = torch.zeros(0, 1, 64, dtype=torch.bfloat16, device=dev)
    loc = torch.zeros(0, 2, dtype=torch.int32, device=dev)
    assert axk.store_paged_kv_rope(none, none, cache, loc, q=none).shape == (0, 1, 64)
    check_tree(tree_case([0, 0, 1], [1, 0, 1], 1, 1, 1, 64, 16, trees=[[-1], [-2], [-1]]), dev)
    gd = gdn_case(1, 1, 1, 1, trees=[[-1]])
    _, u, g = check_gdn(gd, dev)
    _, s = axk.gdn_recurrent(*(gd[n].to(dev) for n in GDN[:-1]))
    got = axk.gdn_tree_commit(gd["state"].to(dev), gd["k"].to(dev), u, g, gd["parents"].to(dev),
                              torch.zeros(1, dtype=torch.int32, device=dev))
    torch.testing.assert_close(got, s, rtol=1e-5, atol=1e-6)
