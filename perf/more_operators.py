"""The measured work of verifying trees of drafted tokens in a hybrid model: the rows of keys and values written into a
paged cache with the position rotation applied on the way, attention of the drafted nodes over the cached history and
their own ancestors, the Gated DeltaNet (GDN) recurrence along every branch of the tree, and the state brought to the
node that was accepted.

A sequence's tree is a row of `parents`: node t's parent is a node before it, -1 stands for the last token of the
history and -2 for no node (rows behind a smaller tree). Node t's key and value lie in the cache behind the history, in
the nodes' order. A case is a dict of plain values whose "kind" names the operator:
  append  k, v rows of fused projections -> norm and rotation -> the cache; the queries rotated in the same call
  tree    attention of every node over the history, its ancestors and itself
  gdn     the delta rule along every branch: outputs, the nodes' state updates and decays; the state itself stays
  commit  the state after the accepted node's branch
"own" chooses between the plain forms (elementary torch operations) and the framework's operators.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
INF = float("inf")
KV_SCALE = 8.0  # an FP8 cache holds e4m3(x * KV_SCALE)
EPS = 1e-6
THETA = 1e7


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
        # One decode step's rows of 16 sequences, queries and keys normalised: a latency-bound call made once a layer.
        {"name": "append_b16", "kind": "append", "kv": "bf16", "rows": 16, "far": 16384, "hq": 16, "hkv": 2, "d": 256,
         "rot": 64, "page": 64, "norm": True, "queries": True, "skip": 0, "table": "bf16"},
        # The accepted branches of 8 drafted trees of 16 nodes written to their places in an FP8 cache: keys and values
        # only, most rows left out.
        {"name": "append_accepted_fp8", "kind": "append", "kv": "fp8", "rows": 128, "far": 131072, "hq": 32, "hkv": 4,
         "d": 256, "rot": 64, "page": 256, "norm": True, "queries": False, "skip": 96, "table": "f32"},
        # A 4096-token prompt chunk, the whole head rotated: bound by memory traffic.
        {"name": "append_chunk4096", "kind": "append", "kv": "bf16", "rows": 4096, "far": 32768, "hq": 32, "hkv": 8,
         "d": 128, "rot": 128, "page": 64, "norm": False, "queries": True, "skip": 0, "table": "f32"},
        # One user's draft of 8 nodes over an ordinary history.
        {"name": "tree_b1_t8", "kind": "tree", "kv": "bf16", "batch": 1, "lo": 5003, "hi": 5003, "nodes": 8, "hq": 16,
         "hkv": 2, "d": 256, "page": 64},
        # A serving step: 16 uneven sequences of an FP8 cache with up to 13 nodes each.
        {"name": "tree_fp8_b16_t13", "kind": "tree", "kv": "fp8", "batch": 16, "lo": 1024, "hi": 16384, "nodes": 13,
         "hq": 16, "hkv": 2, "d": 256, "page": 64},
        # The same for 4 sequences of an INT8 cache and smaller heads.
        {"name": "tree_i8_b4_t24", "kind": "tree", "kv": "int8", "batch": 4, "lo": 2048, "hi": 8192, "nodes": 24,
         "hq": 32, "hkv": 8, "d": 128, "page": 16},
        # Wide drafts over long histories: 64 nodes x 8 query heads share every cached row, bound by the matrix cores.
        {"name": "tree_b8_t64_long", "kind": "tree", "kv": "bf16", "batch": 8, "lo": 32768, "hi": 32768, "nodes": 64,
         "hq": 32, "hkv": 4, "d": 256, "page": 256},
        # One sequence's draft through a GDN layer: 32 states of 64 KiB.
        {"name": "gdn_b1_t8", "kind": "gdn", "batch": 1, "nodes": 8, "nk": 16, "nv": 32},
        # The widest drafts.
        {"name": "gdn_b8_t64", "kind": "gdn", "batch": 8, "nodes": 64, "nk": 16, "nv": 32},
        # A full batch: 67 MB of states read once.
        {"name": "gdn_b32_t16", "kind": "gdn", "batch": 32, "nodes": 16, "nk": 16, "nv": 32},
        # One sequence's states brought to its accepted node.
        {"name": "commit_b1_t8", "kind": "commit", "batch": 1, "nodes": 8, "nk": 16, "nv": 32},
        # A full batch's states, in place.
        {"name": "commit_b32_t16", "kind": "commit", "batch": 32, "nodes": 16, "nk": 16, "nv": 32},
    ]


def _log(rng, lo, hi):
    """An integer spread over [lo, hi] by its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "tree", "tree", "tree", "gdn", "gdn", "commit"])
    if kind in ("gdn", "commit"):
        nk, nv = rng.choice([(16, 32), (16, 32), (16, 48), (2, 4), (4, 4), (16, 16)])
        nodes = _log(rng, 1, 64)
        return {"kind": kind, "batch": _log(rng, 1, max(1, min(64, 32 * 32 * 16 // (nv * max(nodes, 16))))),
                "nodes": nodes, "nk": nk, "nv": nv}
    kv = rng.choice(["bf16", "fp8", "int8"])
    hq, hkv, d = rng.choice([(16, 2, 256), (32, 4, 256), (16, 4, 256), (8, 2, 128), (32, 8, 128), (6, 2, 128),
                             (16, 1, 64), (7, 7, 64)])
    page = rng.choice([16, 64, 256, 96])
    if kind == "append":
        rows = _log(rng, 1, 4096 * 32 * 128 // (hq * d))
        return {"kind": kind, "kv": "fp8" if kv == "int8" else kv, "rows": rows, "far": _log(rng, 2048, 131072), "hq": hq,
                "hkv": hkv, "d": d, "rot": rng.choice([x for x in (16, 32, 64, 128, 256) if x <= d]), "page": page,
                "norm": rng.random() < 0.5, "queries": rng.random() < 0.6,
                "skip": rng.choice([0, 0, _log(rng, 1, rows) // 2]), "table": rng.choice(["bf16", "f32"])}
    batch, nodes = _log(rng, 1, 64), _log(rng, 1, 64)
    hi = _log(rng, 1, max(1, min(131072, 8 * 32768 * 4 * 256 // (batch * hkv * d),
                                 8 * 32768 * 64 * 32 * 256 // (batch * nodes * hq * d))))
    return {"kind": kind, "kv": kv, "batch": batch, "lo": max(0, hi // 8 - 1), "hi": hi, "nodes": nodes, "hq": hq,
            "hkv": hkv, "d": d, "page": page}


def _lens(case):
    """The history of each sequence in tokens, spread over [lo, hi] by the case's own sizes."""
    rng = random.Random(case["batch"] * 1000003 + case["lo"] * 1009 + case["hi"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def _counts(case):
    """The nodes of each sequence: the first has them all, the others at least half."""
    rng = random.Random(case["batch"] * 7001 + case["nodes"])
    most = case["nodes"]
    return [most] + [rng.randint((most + 1) // 2, most) for _ in range(case["batch"] - 1)]


def _cdiv(a, b):
    return -(-a // b)


def _tree(rng, n, most):
    """n nodes as a drafter lays them out, parents first: half of them extend the node before, -2 behind them."""
    p = [-1] + [t - 1 if rng.random() < 0.5 else rng.randrange(-1, t) for t in range(1, n)]
    return p + [-2] * (most - n)


def _branch(parents, t):
    """Node t and its ancestors, the first ancestor first."""
    out = []
    while t >= 0:
        out.append(t)
        t = parents[t]
    return out[::-1]


def work(case):
    kind = case["kind"]
    if kind == "append":
        kept = case["rows"] - case["skip"]
        size = 1 if case["kv"] == "fp8" else 2
        heads = case["hq"] if case["queries"] else 0
        table = case["rot"] * (2 if case["table"] == "bf16" else 4)
        live = case["rows"] if case["queries"] else kept
        return {"bytes": 2 * kept * case["hkv"] * case["d"] * (2 + size) + 4 * case["rows"] * heads * case["d"]
                + live * (table + 12), "flops": 6.0 * (kept * case["hkv"] + case["rows"] * heads) * case["d"]}
    counts = _counts(case)
    if kind == "tree":
        lens, d = _lens(case), case["d"]
        size = 2 if case["kv"] == "bf16" else 1
        row = 2 * case["hkv"] * (d * size + (2 if case["kv"] == "int8" else 0))
        return {"bytes": sum(x + n for x, n in zip(lens, counts)) * row + 4 * sum(counts) * case["hq"] * d,
                "flops": 4.0 * case["hq"] * d * sum(n * x + n * (n + 1) // 2 for x, n in zip(lens, counts))}
    nv, nk, nodes = case["nv"], case["nk"], sum(counts)
    states = case["batch"] * nv * 128 * 128
    if kind == "gdn":
        return {"bytes": 4 * states + nodes * (2 * 2 * nk * 128 + 2 * nv * 128 + 4 * nv + nv * 128 * (2 + 4) + 4 * nv),
                "flops": 4.0 * nodes * nv * 128 * 128 + 4.0 * nv * 128 * sum(n * n for n in counts)}
    return {"bytes": 8 * states + nodes // 2 * (nv * 128 * 4 + nk * 128 * 2 + 4 * nv),
            "flops": 2.0 * states + 1.0 * nodes * nv * 128 * 128}


# ---- inputs ----
def _table(pages, gen, extra=3):
    """indptr, indices of sequences of so many pages each, and the pool they lie in, in random order."""
    nnz = sum(pages)
    pool = nnz + extra
    indptr = torch.tensor([0] + [sum(pages[:i + 1]) for i in range(len(pages))], dtype=torch.int32, device=DEV)
    indices = torch.randperm(pool, generator=gen, device=DEV)[:nnz].to(torch.int32)
    return indptr, indices, pool


def _cache(pool, page, hkv, d, kv, gen):
    """A KV pool: keys with channels of uneven size, as projections give them, and values of one size; its scales."""
    x = torch.randn(pool, 2, page, hkv, d, generator=gen, device=DEV, dtype=torch.bfloat16)
    x[:, 0] *= torch.exp(0.5 * torch.randn(hkv, d, generator=gen, device=DEV)).to(torch.bfloat16)
    if kv == "bf16":
        return x, None
    if kv == "fp8":
        return (x * KV_SCALE).to(torch.float8_e4m3fn).view(torch.uint8), None
    s = (x.abs().amax(-1).clamp(min=1e-5) / 127).to(torch.bfloat16)
    return (x / s[..., None]).round().clamp(-128, 127).to(torch.int8), s


def _values(x, scales, kv):
    """What attention reads for stored values x, in 32 bits."""
    if kv == "bf16":
        return x.float()
    return x.view(torch.float8_e4m3fn).float() / KV_SCALE if kv == "fp8" else x.float() * scales.float()[..., None]


def _trees(case, seed):
    rng = random.Random(seed * 131 + 7)
    return [_tree(rng, n, case["nodes"]) for n in _counts(case)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 7919 + 17)
    kind = case["kind"]
    st = {"case": case, "kind": kind}

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)

    if kind == "append":
        rows, hq, hkv, d, page = case["rows"], case["hq"], case["hkv"], case["d"], case["page"]
        # one projection's rows [q | k | v], as a fused weight gives them: the operands are views of it
        qkv = randn(rows, (hq + 2 * hkv) * d)
        st["q"] = qkv[:, :hq * d].view(rows, hq, d) if case["queries"] else None
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].view(rows, hkv, d)
        st["v"] = qkv[:, (hq + hkv) * d:].view(rows, hkv, d)
        pool = _cdiv(rows, page) + 16
        st["cache"] = _cache(pool, page, hkv, d, case["kv"], gen)[0]
        st["kv_scale"] = KV_SCALE if case["kv"] == "fp8" else None
        at = torch.randperm(pool * page, generator=gen, device=DEV)[:rows]
        if rows >= 512:  # a prompt chunk fills whole pages
            first = torch.randperm(pool, generator=gen, device=DEV)[:_cdiv(rows, page)]
            at = (first[:, None] * page + torch.arange(page, device=DEV)).flatten()[:rows]
        st["loc"] = torch.stack([at // page, at % page], 1).to(torch.int32).contiguous()
        st["rows"] = None
        if case["skip"]:  # rows that are not stored, and those that are
            order = torch.randperm(rows, generator=gen, device=DEV)
            st["loc"][order[:case["skip"]]] = -1
            st["rows"] = order[case["skip"]:].sort().values
        st["positions"] = torch.randint(0, case["far"], (rows,), generator=gen, device=DEV, dtype=torch.int32)
        inv = THETA ** -(torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV) / case["rot"])
        angle = torch.arange(case["far"], dtype=torch.float64, device=DEV)[:, None] * inv
        kept = torch.bfloat16 if case["table"] == "bf16" else torch.float32
        st["cos"], st["sin"] = angle.cos().to(kept), angle.sin().to(kept)
        st["q_norm"] = st["k_norm"] = None
        if case["norm"]:
            st["k_norm"] = 1.0 + 0.1 * randn(d, dtype=torch.float32)
            st["q_norm"] = 1.0 + 0.1 * randn(d, dtype=torch.float32) if case["queries"] else None
        return st
    trees = _trees(case, seed)
    batch, nodes = case["batch"], case["nodes"]
    st["parents"] = torch.tensor(trees, dtype=torch.int32, device=DEV)
    if kind == "tree":
        lens, counts, page = _lens(case), _counts(case), case["page"]
        total = [x + n for x, n in zip(lens, counts)]
        pages = [_cdiv(x, page) for x in total]
        st["indptr"], st["indices"], pool = _table(pages, gen)
        st["last"] = torch.tensor([x - (p - 1) * page for x, p in zip(total, pages)], dtype=torch.int32, device=DEV)
        st["most"] = max(total)
        st["cache"], st["scales"] = _cache(pool, page, case["hkv"], case["d"], case["kv"], gen)
        st["q"] = randn(batch, nodes, case["hq"], case["d"]) * 2
        st["scale"] = 1.0 / math.sqrt(case["d"])
        return st
    nk, nv = case["nk"], case["nv"]
    st["k"] = randn(batch, nodes, nk, 128)
    st["state"] = 0.3 * randn(batch, nv, 128, 128, dtype=torch.float32)
    if kind == "gdn":
        st["q"], st["v"] = randn(batch, nodes, nk, 128), randn(batch, nodes, nv, 128)
        st["a"], st["b"] = randn(batch, nodes, nv), randn(batch, nodes, nv)
        st["a_log"] = 0.5 * randn(nv, dtype=torch.float32)
        st["dt_bias"] = 0.5 * randn(nv, dtype=torch.float32)
        return st
    # what the verify step left: updates and log decays of every node, zero where there is none
    there = (st["parents"] >= -1)[:, :, None]
    st["updates"] = randn(batch, nodes, nv, 128, dtype=torch.float32) * there[..., None]
    st["gates"] = -torch.nn.functional.softplus(randn(batch, nodes, nv, dtype=torch.float32)) * there
    rng = random.Random(seed * 31 + 5)
    st["accepted"] = torch.tensor([rng.randrange(-1, n) if i else n - 1 for i, n in enumerate(_counts(case))],
                                  dtype=torch.int32, device=DEV)
    return st


# ---- one pass ----
def run(st):
    if own:
        return _run_own(st)
    return {"append": _append, "tree": _attend, "gdn": _gdn, "commit": _commit}[st["kind"]](st)


def _run_own(st):
    axk, kind = _axk(), st["kind"]
    if kind == "append":
        q = axk.store_paged_kv_rope(st["k"], st["v"], st["cache"], st["loc"], st["cos"], st["sin"], st["positions"],
                                    k_norm=st["k_norm"], q=st["q"], q_norm=st["q_norm"], eps=EPS,
                                    kv_scale=st["kv_scale"])
        return _stored(st) if q is None else {"q": q, **_stored(st)}
    if kind == "tree":
        return axk.paged_tree_verify(st["q"], st["cache"], st["indptr"], st["indices"], st["last"], st["parents"],
                                     sm_scale=st["scale"], kv_scale=KV_SCALE if st["case"]["kv"] == "fp8" else None,
                                     kv_scales=st["scales"])
    if kind == "gdn":
        out, updates, gates = axk.gdn_tree_verify(st["q"], st["k"], st["v"], st["a"], st["b"], st["a_log"],
                                                  st["dt_bias"], st["state"], st["parents"])
        return {"out": out, "updates": updates, "gates": gates}
    return axk.gdn_tree_commit(st["state"], st["k"], st["updates"], st["gates"], st["parents"], st["accepted"],
                               state_out=st["state"])


def _stored(st):
    """The cache as the values its bytes stand for."""
    return {"cache": st["cache"] if st["case"]["kv"] == "bf16" else st["cache"].view(torch.float8_e4m3fn)}


# ---- the plain forms ----
def _rotated(x, w, cos, sin):
    """x [rows, heads, D] normalised by w (if any) and rotated, in 32 bits."""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    half = cos.shape[-1]
    c, s = cos.float()[:, None], sin.float()[:, None]
    lo, hi = x[..., :half], x[..., half:2 * half]
    return torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., 2 * half:]], -1)


def _append(st):
    case, cache = st["case"], st["cache"]
    pos = st["positions"].long()
    cos, sin = st["cos"][pos], st["sin"][pos]
    page, slot = st["loc"][:, 0].long(), st["loc"][:, 1].long()
    rows = slice(None) if st["rows"] is None else st["rows"]
    flat = cache.view(-1, *cache.shape[-2:])
    at = 2 * page * case["page"] + slot
    for plane, x in ((0, _rotated(st["k"], st["k_norm"], cos, sin)), (1, st["v"].float())):
        if case["kv"] == "fp8":
            x = (x * KV_SCALE).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            x = x.to(torch.bfloat16)
        flat[(at + plane * case["page"])[rows]] = x[rows]
    if st["q"] is None:
        return _stored(st)
    return {"q": _rotated(st["q"], st["q_norm"], cos, sin).to(torch.bfloat16), **_stored(st)}


def _sees(parents):
    """[B, T, T]: whether node j is node t or an ancestor of it; nodes that are none see nothing."""
    b, t = parents.shape
    there = parents >= -1
    sees = torch.diag_embed(there)
    at = parents.long()
    for _ in range(t):
        if t == 1:
            break
        step = (torch.arange(t, device=parents.device) == at[..., None]) & (at >= 0)[..., None]
        sees = sees | step
        at = torch.where(at >= 0, torch.gather(parents.long(), 1, at.clamp(min=0)), -1)
    return sees, there


def _attend(st):
    case, parents = st["case"], st["parents"]
    page, hkv, kv = case["page"], case["hkv"], case["kv"]
    b, t, hq, d = st["q"].shape
    sees, there = _sees(parents)
    n = there.sum(1)
    out = torch.empty(b, t, hq, d, dtype=torch.bfloat16, device=DEV)
    pages = (st["indptr"][1:] - st["indptr"][:-1]).long()
    total = torch.where(pages > 0, (pages - 1) * page + st["last"].long(), 0)
    tok = torch.arange(st["most"], device=DEV)
    entry = (st["indptr"][:-1].long()[:, None] + tok // page).clamp(max=st["indices"].numel() - 1)
    some = max(1, int(2e9) // (st["most"] * hkv * max(d, t * (hq // hkv)) * 4))
    for b0 in range(0, b, some):
        s_ = slice(b0, min(b, b0 + some))
        at = st["indices"].long()[entry[s_]]
        k, v = (_values(st["cache"][at, i, tok % page], None if st["scales"] is None else st["scales"][at, i, tok % page], kv)
                .permute(0, 2, 1, 3) for i in (0, 1))  # [b, HKV, most, D]
        q = st["q"][s_].float().view(-1, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(-1, hkv, t * (hq // hkv), d)
        s = torch.matmul(q, k.transpose(2, 3)) * st["scale"]
        node = tok[None] - (total - n)[s_, None]  # the node a cached token is, if any
        row = sees[s_].gather(2, node.clamp(0, t - 1)[:, None].expand(-1, t, -1))
        ok = (tok[None] < total[s_, None])[:, None] & there[s_][:, :, None] & ((node < 0)[:, None] | row)
        ok = ok[:, None, :, None].expand(-1, hkv, -1, hq // hkv, -1).reshape(-1, hkv, t * (hq // hkv), st["most"])
        s = torch.where(ok, s, -INF)
        p = torch.exp(s - s.amax(3, keepdim=True).clamp(min=-3e38))
        sum_ = p.sum(3, keepdim=True)
        v = torch.where((tok[None] < total[s_, None])[:, None, :, None], v, 0.0)
        o = torch.matmul(p, v) / torch.where(sum_ > 0, sum_, 1.0)
        out[s_] = o.view(-1, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(-1, t, hq, d).to(torch.bfloat16)
    return out


def _unit(x):
    x = x.float()
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _gdn(st):
    parents = st["parents"].long()
    b, t, nv, _ = st["v"].shape
    rep = nv // st["k"].shape[2]
    there = parents >= -1
    q, k = (_unit(x).repeat_interleave(rep, 2) for x in (st["q"], st["k"]))
    q = q * 128 ** -0.5
    x = st["a"].float() + st["dt_bias"]
    g = -torch.exp(st["a_log"]) * (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    beta = torch.sigmoid(st["b"].float())
    # the state after every node, the one before the tree first
    states = torch.empty(t + 1, b, nv, 128, 128, device=DEV)
    states[0] = st["state"]
    at = torch.arange(b, device=DEV)
    out = torch.empty(b, t, nv, 128, dtype=torch.bfloat16, device=DEV)
    updates = torch.empty(b, t, nv, 128, device=DEV)
    for i in range(t):
        s = states[(parents[:, i] + 1).clamp(min=0), at] * torch.exp(g[:, i])[..., None, None]
        u = (st["v"][:, i].float() - torch.matmul(k[:, i, :, None], s)[:, :, 0]) * beta[:, i, :, None]
        s = s + k[:, i, :, :, None] * u[:, :, None]
        states[i + 1] = s
        live = there[:, i, None, None]
        out[:, i] = torch.where(live, torch.matmul(q[:, i, :, None], s)[:, :, 0], 0.0).to(torch.bfloat16)
        updates[:, i] = torch.where(live, u, 0.0)
    return {"out": out, "updates": updates, "gates": torch.where(there[..., None], g, 0.0)}


def _commit(st):
    parents, state = st["parents"], st["state"]
    b, t, nv, _ = st["updates"].shape
    sees, there = _sees(parents)
    node = st["accepted"].long()
    path = torch.where((node >= 0)[:, None], sees[torch.arange(b, device=DEV), node.clamp(min=0)], False)
    g = torch.where(path[..., None], st["gates"], 0.0)
    left = g.double().flip(1).cumsum(1).flip(1).float()  # the decay from before each node on
    w = torch.where(path[..., None], torch.exp(left - g), 0.0)  # what is left of a node's own update
    k = _unit(st["k"]).repeat_interleave(nv // st["k"].shape[2], 2)
    added = torch.matmul((k * w[..., None]).permute(0, 2, 3, 1), st["updates"].permute(0, 2, 1, 3))
    state.mul_(torch.exp(left[:, 0])[..., None, None]).add_(added)
    return state


# ---- the definitions, in 64 bits, one sequence or row at a time ----
def _read(x, scale, kv):
    """Stored values in 64 bits; an E4M3 byte by its fields."""
    if kv == "bf16":
        return x.double()
    if kv == "int8":
        return x.double() * scale.double()[..., None]
    x = x.long()
    sign, e, m = 1.0 - 2.0 * (x >> 7).double(), (x >> 3) & 15, (x & 7).double()
    return sign * torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m / 512) / KV_SCALE


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        half, d = case["rot"] // 2, case["d"]

        def turned(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + EPS) * w.double()
            # a pair of channels as one complex number, turned by the row's angle
            z = torch.complex(x[..., :half], x[..., half:2 * half])
            at = st["positions"].long()
            z = z * torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]
            return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

        size = KV_SCALE if case["kv"] == "fp8" else 1.0
        cache = st["cache"].double() if case["kv"] == "bf16" else _read(st["cache"], None, "fp8") * KV_SCALE
        k, v = turned(st["k"], st["k_norm"]) * size, st["v"].double() * size
        rows = slice(None) if st["rows"] is None else st["rows"]
        page, slot = st["loc"][rows, 0].long(), st["loc"][rows, 1].long()
        cache[page, 0, slot] = k[rows]
        cache[page, 1, slot] = v[rows]
        return {"cache": cache} if st["q"] is None else {"q": turned(st["q"], st["q_norm"]), "cache": cache}
    trees, counts = _trees(case, seed), _counts(case)
    if kind == "tree":
        page, hkv, d = case["page"], case["hkv"], case["d"]
        group = case["hq"] // hkv
        ptr = st["indptr"].tolist()
        out = torch.zeros(case["batch"], case["nodes"], case["hq"], d, dtype=torch.float64, device=DEV)
        for b, (x, n) in enumerate(zip(_lens(case), counts)):
            ids = st["indices"][ptr[b]:ptr[b + 1]].long()
            rows = torch.arange(x + n, device=DEV)
            hide = torch.full((n, x + n), -INF, dtype=torch.float64, device=DEV)
            hide[:, :x] = 0
            for t in range(n):
                hide[t, [x + j for j in _branch(trees[b], t)]] = 0
            for h in range(hkv):
                k, v = (_read(st["cache"][ids[rows // page], i, rows % page, h],
                              None if st["scales"] is None else st["scales"][ids[rows // page], i, rows % page, h],
                              case["kv"]) for i in (0, 1))
                for g in range(h * group, (h + 1) * group):
                    p = torch.softmax(st["q"][b, :n, g].double() @ k.t() * st["scale"] + hide, 1)
                    out[b, :n, g] = p @ v
        return out
    nv, nk = case["nv"], case["nk"]
    head = torch.arange(nv, device=DEV) // (nv // nk)
    k = st["k"].double()
    k = (k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6))[:, :, head]
    if kind == "commit":
        state = st["state"].double()
        for b, n in enumerate(st["accepted"].tolist()):
            for i in _branch(trees[b], n):
                state[b] = state[b] * torch.exp(st["gates"][b, i].double())[:, None, None] \
                    + k[b, i][:, :, None] * st["updates"][b, i].double()[:, None]
        return state
    q = st["q"].double()
    q = (q / torch.sqrt(q.square().sum(-1, keepdim=True) + 1e-6) / math.sqrt(128))[:, :, head]
    g = -torch.exp(st["a_log"].double()) * torch.nn.functional.softplus(st["a"].double() + st["dt_bias"].double())
    beta = torch.sigmoid(st["b"].double())
    out = torch.zeros(*st["v"].shape, dtype=torch.float64, device=DEV)
    updates, gates = torch.zeros_like(out), torch.zeros_like(g)
    for b, n in enumerate(counts):
        after = []
        for i in range(n):
            s = (st["state"][b].double() if trees[b][i] < 0 else after[trees[b][i]]) * torch.exp(g[b, i])[:, None, None]
            u = beta[b, i][:, None] * (st["v"][b, i].double() - (k[b, i][:, :, None] * s).sum(1))
            s = s + k[b, i][:, :, None] * u[:, None]
            after.append(s)
            out[b, i], updates[b, i], gates[b, i] = (q[b, i][:, :, None] * s).sum(1), u, g[b, i]
    return {"out": out, "updates": updates, "gates": gates}
