"""What pins the oracle of the drafted trees (CPU)."""
import math
import random

import pytest
import torch

from axk import configs
from oracle import gdn as ogdn
from oracle import paged_attn
from oracle import tree as ot


def random_tree(n, t, seed=0):
    rng = random.Random(seed)
    return [-1] + [i - 1 if rng.random() < 0.5 else rng.randrange(-1, i) for i in range(1, n)] + [-2] * (t - n) if n else [-2] * t


def chain(n, t):
    return list(range(-1, n - 1)) + [-2] * (t - n)


def test_branches():
    assert ot.branches([-1, 0, 0, 2, -1, 4]) == [[0], [0, 1], [0, 2], [0, 2, 3], [4], [4, 5]]
    assert ot.branches([-1, -2, 1, 0, 9, -5, 3]) == [[0], [], [], [0, 3], [], [], [0, 3, 6]]
    assert ot.bad_tree([-1, -2, 1]) and ot.bad_tree([0]) and ot.bad_tree([-3]) and not ot.bad_tree([-1, -2, 0])
    assert ot.node_count([-1, -2, 0, -2]) == 3 and ot.node_count([-2, -2]) == 0


def test_chain_attention_is_prefill():
    g = torch.Generator().manual_seed(0)
    c = configs.prefill_case([5, 1, 7], [40, 1, 21], 6, 2, 64, 16, g, extra_pages=2)
    q = torch.zeros(3, 7, 6, 64, dtype=torch.bfloat16)
    for b, n in enumerate(c["qlens"]):
        q[b, :n] = c["q"][int(c["qo_indptr"][b]):][:n]
    parents = torch.tensor([chain(n, 7) for n in c["qlens"]])
    got, _ = ot.tree_attention(q, c["cache"], c["indptr"], c["indices"], c["last_page_len"], parents, c["scale"])
    ref = paged_attn.paged_prefill(c["q"], c["cache"], c["qo_indptr"], c["indptr"], c["indices"], c["last_page_len"], c["scale"])
    for b, n in enumerate(c["qlens"]):
        torch.testing.assert_close(got[b, :n], ref[int(c["qo_indptr"][b]):][:n].double(), rtol=1e-5, atol=1e-5)
        assert not got[b, n:].any()


def test_every_branch_attends_as_its_own_chain():
    """The branch's rows moved behind the history, in order, and attended as a chain."""
    g = torch.Generator().manual_seed(1)
    hist, n, page = 19, 9, 16
    tree = random_tree(n, n, 3)
    c = configs.paged_case([hist + n], 4, 2, 64, page, g)
    q = torch.randn(1, n, 4, 64, generator=g).to(torch.bfloat16)
    got, _ = ot.tree_attention(q, c["cache"], c["indptr"], c["indices"], c["last_page_len"], torch.tensor([tree]))
    where = lambda t: (int(c["indices"][t // page]), t % page)  # noqa: E731
    for t, mine in enumerate(ot.branches(tree)):
        cache = c["cache"].clone()
        for i, m in enumerate(mine):
            (p0, s0), (p1, s1) = where(hist + m), where(hist + i)
            cache[p1, :, s1] = c["cache"][p0, :, s0]
        total = hist + len(mine)
        pages = -(-total // page)
        ref = paged_attn.paged_prefill(q[0, mine], cache, [0, len(mine)], [0, pages], c["indices"][:pages],
                                       [total - (pages - 1) * page], 0.125)
        torch.testing.assert_close(got[0, t], ref[-1].double(), rtol=1e-5, atol=1e-5)


def test_gdn_chain_is_the_recurrence():
    g = torch.Generator().manual_seed(2)
    c = configs.gdn_inputs(2, 6, g, nk=2, nv=4)
    c["a_log"], c["dt_bias"] = torch.randn(4, generator=g), torch.randn(4, generator=g)
    names = ("q", "k", "v", "a", "b", "a_log", "dt_bias", "state")
    parents = torch.tensor([chain(6, 6)] * 2)
    (o, u, gt), _ = ot.gdn_tree(*(c[x] for x in names), parents)
    ref, state = ogdn.gdn_fp32(*(c[x] for x in names))
    torch.testing.assert_close(o.float(), ref, rtol=1e-5, atol=1e-6)
    got, _ = ot.gdn_commit(c["state"], c["k"], u.float(), gt.float(), parents, torch.tensor([5, 5]))
    torch.testing.assert_close(got.float(), state, rtol=1e-5, atol=1e-6)


def test_every_gdn_branch_is_its_own_chain():
    g = torch.Generator().manual_seed(3)
    n = 8
    c = configs.gdn_inputs(1, n, g, nk=1, nv=2)
    tree = random_tree(n, n, 5)
    names = ("q", "k", "v", "a", "b")
    rest = (c["a_log"], c["dt_bias"], c["state"])
    parents = torch.tensor([tree])
    (o, u, gt), _ = ot.gdn_tree(*(c[x] for x in names), *rest, parents)
    for t, mine in enumerate(ot.branches(tree)):
        ref, state = ogdn.gdn_fp32(*(c[x][:, mine] for x in names), *rest)
        torch.testing.assert_close(o[0, t].float(), ref[0, -1], rtol=1e-5, atol=1e-6)
        got, _ = ot.gdn_commit(c["state"], c["k"], u.float(), gt.float(), parents, torch.tensor([t]))
        torch.testing.assert_close(got.float(), state, rtol=1e-5, atol=1e-6)


def test_commit_of_nothing_keeps_the_state():
    g = torch.Generator().manual_seed(4)
    state, k = torch.randn(3, 2, 128, 128, generator=g), torch.randn(3, 4, 1, 128, generator=g)
    u, gt = torch.randn(3, 4, 2, 128, generator=g), -torch.rand(3, 4, 2, generator=g)
    parents = torch.tensor([chain(4, 4), chain(2, 4), chain(4, 4)])
    got, _ = ot.gdn_commit(state, k, u, gt, parents, torch.tensor([-1, 3, 9]))
    assert torch.equal(got, state.double())


@pytest.mark.parametrize("rot", [16, 64])
def test_rotations(rot):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(7, 3, 64, generator=g)
    one, zero = torch.ones(7, rot // 2), torch.zeros(7, rot // 2)
    assert torch.equal(ot.rope_rows(x, None, one, zero, 1e-6)[0], x.double())
    a, b = torch.rand(7, rot // 2, generator=g).double(), torch.rand(7, rot // 2, generator=g).double()
    once = ot.rope_rows(ot.rope_rows(x, None, a.cos(), a.sin(), 0)[0], None, b.cos(), b.sin(), 0)[0]
    both = ot.rope_rows(x, None, (a + b).cos(), (a + b).sin(), 0)[0]
    torch.testing.assert_close(once, both)
    torch.testing.assert_close(once.norm(dim=-1), x.double().norm(dim=-1))
    half = rot // 2  # channel 0 against channel rot / 2, a quarter turn
    y = ot.rope_rows(x, None, zero, one, 0)[0]
    assert torch.equal(y[..., 0], -x[..., half].double()) and torch.equal(y[..., half], x[..., 0].double())
    assert torch.equal(y[..., rot:], x[..., rot:].double())


def test_norm():
    x = torch.tensor([[[3.0, 4.0] + [0.0] * 62]])
    w = torch.full((64,), 2.0)
    y, _ = ot.rope_rows(x, w, None, None, 0.0)
    assert math.isclose(float(y[0, 0, 1]), 2 * 4 / math.sqrt(25 / 64), rel_tol=1e-12)
