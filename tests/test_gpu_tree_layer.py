"""A GDN layer's tree step from its convolution on: every node's window of inputs gathered along its branch, the delta rule in both
orders of value heads, and the accepted branch's states, against the layer's operators over each branch as a chain."""
import pytest
import torch

import axk
from axk import configs
from axk.layer import v_tiled

from test_gpu_tree import BF16_HALF, random_tree
from test_gpu_tree_step import path_to

pytestmark = pytest.mark.gpu
K = 4  # taps of the convolution


def windows(parents, start, steps):
    """Entries of [conv state | nodes] in which the `steps` inputs that end at entry `start` [B, N] lie, oldest first."""
    nodes = parents.long()
    before = torch.where(nodes >= -1, nodes + K - 1, 0)  # the entry before each node's
    before = torch.cat([torch.arange(-1, K - 2, device=parents.device).clamp(min=0).expand(len(nodes), -1), before], 1)
    out = [start]
    for _ in range(steps - 1):
        out.insert(0, before.gather(1, out[0]))
    return torch.stack(out, 2)


@pytest.mark.parametrize("t,nk,nv", [(9, 2, 4), (33, 2, 6), (1, 1, 1)])
def test_gdn_layer_from_its_convolution_on(dev, t, nk, nv):
    bsz, c = 3, (2 * nk + nv) * 128
    g = torch.Generator().manual_seed(t)
    trees = [random_tree(n, t, 3 * t + i) for i, n in enumerate([t, max(1, t // 2), t])]
    accepted = [t - 1, -1, t // 2]
    x = torch.randn(bsz, t, c, generator=g).to(torch.bfloat16).to(dev)
    w = (0.5 * torch.randn(c, K, generator=g)).to(torch.bfloat16).to(dev)
    conv = torch.randn(bsz, K - 1, c, generator=g).to(torch.bfloat16).to(dev)
    d = {n: v.to(dev) for n, v in configs.gdn_inputs(bsz, t, g, nk=nk, nv=nv, state_std=0.3).items()}
    a_log, dt_bias = (0.5 * torch.randn(nv, generator=g)).to(dev), torch.randn(nv, generator=g).to(dev)
    parents = torch.tensor(trees, dtype=torch.int32, device=dev)
    acc = torch.tensor(accepted, dtype=torch.int32, device=dev)

    # every node is a sequence of one row, its state the three inputs before it on its branch
    ext = torch.cat([conv, x], 1)
    at = windows(parents, torch.arange(K - 1, K - 1 + t, device=dev).expand(bsz, -1).contiguous(), K)[:, :, :K - 1]
    pick = lambda e: ext.gather(1, e.reshape(bsz, -1, 1).expand(-1, -1, c)).view(-1, K - 1, c)  # noqa: E731
    y = axk.glue.causal_conv1d_silu(x.view(bsz * t, 1, c), w, pick(at))[0].view(bsz, t, c)
    new_conv = pick(windows(parents, acc.long()[:, None] + K - 1, K)[:, :, 1:])
    q, k, v = (z.reshape(bsz, t, -1, 128).contiguous() for z in y.split([nk * 128, nk * 128, nv * 128], 2))
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out, upd, gates = axk.gdn_tree_verify(q, k, v, d["a"], d["b"], a_log, dt_bias, d["state"], parents, status=status)
    new = axk.gdn_tree_commit(d["state"], k, upd, gates, parents, acc, status=status)

    for b, tree in enumerate(trees):
        for n in sorted({0, t // 3, t - 1, max(accepted[b], 0)}):
            if tree[n] == -2:
                continue
            rows = torch.tensor(path_to(tree, n), device=dev)
            yb, cs = axk.glue.causal_conv1d_silu(x[b:b + 1, rows].contiguous(), w, conv[b:b + 1])
            assert torch.equal(y[b, rows], yb[0])
            one = lambda z: z[b:b + 1, rows].contiguous()  # noqa: E731
            qb, kb, vb = (z.reshape(1, len(rows), -1, 128).contiguous()
                          for z in yb.split([nk * 128, nk * 128, nv * 128], 2))
            ro, rs = axk.gdn_recurrent(qb, kb, vb, one(d["a"]), one(d["b"]), a_log, dt_bias, d["state"][b:b + 1])
            torch.testing.assert_close(out[b, rows].float(), ro[0].float(), rtol=4 * BF16_HALF, atol=1e-5)
            if n == accepted[b]:
                assert torch.equal(new_conv[b], cs[0])
                torch.testing.assert_close(new[b], rs[0], rtol=1e-4, atol=1e-5)
        if accepted[b] < 0:
            assert torch.equal(new_conv[b], conv[b]) and torch.equal(new[b], d["state"][b])

    # the same layer with its value heads in the tiled order: q and k repeated to a head each
    tiled = lambda z, dim: v_tiled(z, dim, nk, nv, 1)  # noqa: E731
    qr, kr = (z.repeat(1, 1, nv // nk, 1) for z in (q, k))
    to, tu, tg = axk.gdn_tree_verify(qr, kr, tiled(v, 2), tiled(d["a"], 2), tiled(d["b"], 2), tiled(a_log, 0), tiled(dt_bias, 0),
                                     tiled(d["state"], 1), parents, status=status)
    for got, ref in ((to, out), (tu, upd), (tg, gates)):
        assert torch.equal(got, tiled(ref, 2))
    assert torch.equal(axk.gdn_tree_commit(tiled(d["state"], 1), kr, tu, tg, parents, acc, status=status), tiled(new, 1))
    assert int(status) == 0
