"""Oracle: verifying a tree of drafted tokens (CPU, 64 bits, test infrastructure only).

Trees, caches, page tables and argument meaning as include/axk.h describes them. Every function also returns a bound of the
rounding errors that the arithmetic it allows can make (fp32 sums, exponentials and products; bf16 probabilities; the final
rounding to the output's type is left to the caller). Pinned by tests/test_oracle_tree.py: a chain's attention is
paged_attn.paged_prefill and its recurrence gdn.gdn_fp32, every branch of a tree is the chain of its nodes, the state after a
branch is that chain's state, rows rotated by zero angles are the rows, and rotations keep lengths and compose.
"""
from __future__ import annotations

import math

import torch

from .paged_attn import seq_lens
from .paged_blocks import seq_rows

U = 2.0 ** -24  # half a step of fp32


def branches(parents) -> list[list[int]]:
    """For each node of one tree its ancestors and itself, the first ancestor first; [] where it is no node."""
    out: list[list[int]] = []
    for t, p in enumerate(parents):
        if p == -1:
            out.append([t])
        elif 0 <= p < t and out[p]:
            out.append(out[p] + [t])
        else:
            out.append([])
    return out


def bad_tree(parents) -> bool:
    """Whether some entry is neither a node nor -2."""
    return any(p != -2 and not b for p, b in zip(parents, branches(parents)))


def node_count(parents) -> int:
    return max([t + 1 for t, p in enumerate(parents) if p != -2], default=0)


# ---- rows into the cache ----
def rope_rows(x, w, cos, sin, eps: float):
    """x [rows, heads, D] normalised by w (or None) and rotated by cos, sin [rows, rot / 2] (or None), and its error bound."""
    d = x.shape[-1]
    y = x.double()
    err = torch.zeros_like(y)
    if w is not None:
        # the mean's D + 2 roundings count half behind the root, then the root, the quotient and two products
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
        err = y.abs() * U * (d / 2 + 8)
    if cos is None:
        return y, err
    half = cos.shape[-1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    lo, hi = y[..., :half], y[..., half:2 * half]
    elo, ehi = err[..., :half], err[..., half:2 * half]
    out = torch.cat([lo * c - hi * s, hi * c + lo * s, y[..., 2 * half:]], -1)
    mag = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1)
    e = torch.cat([elo * c.abs() + ehi * s.abs(), ehi * c.abs() + elo * s.abs()], -1)
    return out, torch.cat([e + 3 * U * mag, err[..., 2 * half:]], -1)


# ---- attention ----
def tree_attention(q, cache, indptr, indices, last, parents, sm_scale=None, kv_scale=None):
    """(out f64 [B, T, HQ, D], error bound): node t over the history, its ancestors and itself."""
    bsz, t_all, hq, d = q.shape
    hkv, page = cache.shape[3], cache.shape[2]
    group = hq // hkv
    sm_scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    out = torch.zeros(bsz, t_all, hq, d, dtype=torch.float64)
    slack = torch.zeros_like(out)
    for b, length in enumerate(seq_lens(indptr, last, page)):
        tree = parents[b].tolist()
        n = node_count(tree)
        base = length - n
        if base < 0:
            continue
        k, v, good = seq_rows(cache, indptr, indices, last, b, kv_scale)
        for t, mine in enumerate(branches(tree)):
            if not mine:
                continue
            rows = torch.cat([torch.arange(base), torch.tensor([base + i for i in mine])])
            rows = rows[good[rows]]
            if not len(rows):
                continue
            for h in range(hkv):
                g = slice(h * group, (h + 1) * group)
                x, kk, vv = q[b, t, g].double(), k[rows, h], v[rows, h]
                s = x @ kk.t() * sm_scale
                p = torch.softmax(s, 1)
                # a score is off by its sum's roundings and by the exponential's argument's
                off = U * (d + 8) * abs(sm_scale) * (x.abs() @ kk.abs().t()) + 4 * U * (s.abs() + s.abs().amax(1, keepdim=True))
                rel = 2 * off.amax(1, keepdim=True) + U * (len(rows) + 64)
                out[b, t, g] = p @ vv
                slack[b, t, g] = (2.0 ** -8 + rel) * (p @ vv.abs())
    return out, slack


# ---- the delta rule ----
def _branch_sums(g, tree):
    """[T]: the sum of g over each node's branch."""
    return torch.stack([g[m].sum(0) if m else torch.zeros_like(g[0]) for m in tree])


def gdn_tree(q, k, v, a, b, a_log, dt_bias, state, parents):
    """((out, updates, gates) f64, their error bounds): gdn.gdn_fp32's step from the parent's state, node by node."""
    bsz, t_all, nv, _ = v.shape
    per = nv // k.shape[2]
    unit = lambda x: (x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + 1e-6)).repeat_interleave(per, 2)  # noqa: E731
    qn, kn = unit(q) * 128 ** -0.5, unit(k)
    x = a.double() + dt_bias.double()
    g_all = -torch.exp(a_log.double()) * torch.nn.functional.softplus(x)
    beta = torch.sigmoid(b.double())
    out = torch.zeros(bsz, t_all, nv, 128, dtype=torch.float64)
    upd, gates = torch.zeros_like(out), torch.zeros(bsz, t_all, nv, dtype=torch.float64)
    e_out, e_upd, e_gate = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(gates)
    for i in range(bsz):
        tree = branches(parents[i].tolist())
        after: dict[int, torch.Tensor] = {}
        for t, mine in enumerate(tree):
            if not mine:
                continue
            s = (after[mine[-2]] if len(mine) > 1 else state[i].double()) * torch.exp(g_all[i, t])[:, None, None]
            u = (v[i, t].double() - torch.einsum("hk,hkv->hv", kn[i, t], s)) * beta[i, t][:, None]
            s = s + kn[i, t][:, :, None] * u[:, None]
            after[t] = s
            out[i, t], upd[i, t], gates[i, t] = torch.einsum("hk,hkv->hv", qn[i, t], s), u, g_all[i, t]
            e_gate[i, t] = U * (16 * g_all[i, t].abs() + 4 * torch.exp(a_log.double()) * x[i, t].abs())
        # the errors of the closed form (I + A) u = rhs: each entry of rhs, A and the outputs' weights is a product of sums of
        # up to 128 terms with norms, a sigmoid and an exponential, off by c of its terms' magnitudes; what they leave in u goes
        # through |(I + A)^-1|
        sums = _branch_sums(gates[i], tree)
        live = torch.tensor([bool(m) for m in tree])
        sees = torch.zeros(t_all, t_all, dtype=torch.bool)
        for t, mine in enumerate(tree):
            sees[t, mine] = True
        for h in range(nv):
            c = U * (256 + 8 * float(sums[:, h].abs().max()))
            w = torch.where(sees, torch.exp(sums[:, None, h] - sums[None, :, h]), 0.0)
            kk, qk = kn[i, :, h].abs() @ kn[i, :, h].abs().t(), qn[i, :, h].abs() @ kn[i, :, h].abs().t()
            dec, be, sa = torch.exp(sums[:, h])[:, None], beta[i, :, h][:, None], state[i, h].double().abs()
            strict = w * be * (1 - torch.eye(t_all, dtype=torch.float64))
            ua = upd[i, :, h].abs()
            inv = torch.linalg.inv(torch.eye(t_all, dtype=torch.float64) + strict * (kn[i, :, h] @ kn[i, :, h].t())).abs()
            eu = inv @ (c * (be * (v[i, :, h].double().abs() + dec * (kn[i, :, h].abs() @ sa)) + strict * kk @ ua + ua))
            e_upd[i, :, h] = eu * live[:, None]
            e_out[i, :, h] = (c * (dec * (qn[i, :, h].abs() @ sa) + (w * qk) @ ua) + (w * qk) @ eu) * live[:, None]
    return (out, upd, gates), (e_out, e_upd, e_gate)


def gdn_commit(state, k, updates, gates, parents, accepted):
    """(state after each tree's accepted node f64, error bound)."""
    out = state.double()
    err = torch.zeros_like(out)
    nv = state.shape[1]
    kn = k.double() / torch.sqrt(k.double().square().sum(-1, keepdim=True) + 1e-6)
    kn = kn.repeat_interleave(nv // k.shape[2], 2)
    for b, n in enumerate(accepted.tolist()):
        tree = branches(parents[b].tolist())
        mine = tree[n] if 0 <= n < len(tree) else []
        mag = out[b].abs()
        for i in mine:
            e = torch.exp(gates[b, i].double())[:, None, None]
            add = kn[b, i][:, :, None] * updates[b, i].double()[:, None]
            out[b] = out[b] * e + add
            mag = mag * e + add.abs()
        total = gates[b, mine].double().sum(0).abs().max() if mine else 0.0
        err[b] = U * (len(mine) + 80 + float(total)) * mag if mine else 0.0
    return out, err
