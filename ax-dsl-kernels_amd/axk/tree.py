"""Verifying a tree of drafted tokens on gfx950, in the attention and the GDN layers of a hybrid model.

parents int32 [B, T], T <= 64, is the tree of each sequence: a node's parent before it, -1 for the last token of the history,
-2 for no node (rows behind a smaller tree; their outputs are zero). One step over a paged cache and GDN states is::

    q = store_paged_kv_rope(k, v, kv_cache, loc, cos, sin, positions, k_norm=kn, q=q, q_norm=qn)  # attention layers
    out = paged_tree_verify(q.view(B, T, HQ, D), kv_cache, indptr, indices, last, parents)
    out, updates, gates = gdn_tree_verify(q, k, v, a, b, a_log, dt_bias, state, parents)          # GDN layers

with node t's rows in the cache behind the history, in the nodes' order, at position history + its depth. When a branch has
been accepted, its rows go to their final places, and the states to its last node::

    store_paged_kv_rope(k, v, kv_cache, final_loc, cos, sin, positions, k_norm=kn)  # page -1: rows that are not kept
    gdn_tree_commit(state, k, updates, gates, parents, accepted, state_out=state)

The GDN calls take q, k and v behind the layer's causal convolution, contiguous. Along a tree a node's window holds the inputs
before it on its branch, not in the rows before: causal_conv1d_silu computes it with every node as a sequence of one row,
x.view(B * T, 1, C), and as its state the K - 1 inputs before the node, gathered from [conv state | x] along its parents; those up
to the accepted node are the next conv state. Value head h reads key head h // (NV // NK), the "grouped" order, as in
gdn_recurrent. In a layer of the "tiled" order (the default of axk.layer), where it reads head h % NK, q and k are passed repeated
to NV heads: q.repeat(1, 1, NV // NK, 1). The calls of whole layers, attn_layer_verify and gdn_layer_verify, verify chains.

Caches are those of paged_decode (bf16), paged_decode_fp8 (u8 / float8_e4m3fn with ``kv_scale``) and paged_decode_i8 (int8 with
``kv_scales``), page tables theirs too. Nothing is read back to the host, so a step can be captured in a HIP graph. Contract
violations raise ValueError; what only the device sees (a bad parent, page, slot, position) sets ``status`` (int32 [1]) to 1.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .blocks import _cache, _call, _status, _table

_BF16, _F32, _I32, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
_DT_BF16, _DT_F32 = _lib.DT_BF16, _lib.DT_F32


def _rows(t: torch.Tensor, name: str, rows: int, heads: int, d: int):
    """(pointer, row stride, head stride) of a bf16 [rows, heads, d] operand whose channels are contiguous."""
    if t.shape != (rows, heads, d) or t.dtype is not _BF16:
        raise ValueError(f"{name} must be bf16 [{rows}, {heads}, {d}], got {list(t.shape)} {t.dtype}")
    ld, hd, one = t.stride()
    if rows < 2:
        ld = 0
    if heads < 2:
        hd = 0
    if one != 1 or ld % 8 or hd % 8 or ld < 0 or hd < 0:
        raise ValueError(f"{name} needs contiguous channels and row and head strides of multiples of 8, got {t.stride()}")
    return t.data_ptr(), ld, hd


def _norm(w, name: str, d: int):
    if w is not None and (w.dtype is not _F32 or w.shape != (d,) or not w.is_contiguous()):
        raise ValueError(f"{name} must be contiguous float32 [{d}]")


def _parents(parents, b: int, t: int) -> None:
    if parents.dtype is not _I32 or parents.shape != (b, t) or not parents.is_contiguous():
        raise ValueError(f"parents must be contiguous int32 [{b}, {t}]")


def store_paged_kv_rope(
    k: torch.Tensor,
    v: torch.Tensor,
    kv_cache: torch.Tensor,
    cache_location: torch.Tensor,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    k_norm: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    q_norm: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    q_out: Optional[torch.Tensor] = None,
    kv_scale: Optional[float] = None,
    status: Optional[torch.Tensor] = None,
    kv_scales: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """k, v [rows, HKV, D] bf16 into the cache at cache_location[r] = (page, slot) (int32 [rows, 2]; page -1: not stored), and
    q [rows, HQ, D] bf16, if given, into q_out (returned), in one launch. q and k are normalised on the way by q_norm / k_norm
    f32 [D] (the qk_norm_rope operator's norm; None: not) and their first rot = 2 cos.shape[1] channels rotated, halves
    against each other, by row positions[r] (int32 [rows]; -1: no row, nothing is written; None: row r) of the tables cos, sin
    [N, rot / 2], both bf16 or both f32; rot a multiple of 16; no tables: no rotation. Computed in fp32 and rounded once, to
    bf16, E4M3 of x * kv_scale or int8 codes. k, v and q may be views with row and head strides. Distinct locations."""
    kind, stored, p, page, hkv, d = _cache(kv_cache, kv_scale, kv_scales)
    if k.dim() != 3:
        raise ValueError(f"k must be bf16 [rows, {hkv}, {d}]")
    rows = k.shape[0]
    kp, vp = _rows(k, "k", rows, hkv, d), _rows(v, "v", rows, hkv, d)
    if cache_location.dtype is not _I32 or cache_location.shape != (rows, 2) or not cache_location.is_contiguous():
        raise ValueError(f"cache_location must be contiguous int32 [{rows}, 2]")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    n, rot, table = 0, 0, _DT_BF16
    if cos is not None:
        if (cos.dim() != 2 or sin.shape != cos.shape or sin.dtype is not cos.dtype or cos.dtype not in (_BF16, _F32)
                or not cos.is_contiguous() or not sin.is_contiguous()):
            raise ValueError("cos and sin must be contiguous [N, rot / 2], both bfloat16 or both float32")
        n, rot = cos.shape[0], 2 * cos.shape[1]
        table = _DT_BF16 if cos.dtype is _BF16 else _DT_F32
        if rot > d or rot % 16:
            raise ValueError(f"cos has {rot // 2} columns: rot must be a multiple of 16, at most {d}")
        if rot and (n < 1 or (positions is None and n < rows)):
            raise ValueError(f"cos and sin hold {n} positions" + ("" if positions is not None else f" for {rows} rows"))
    if positions is not None and (positions.dtype is not _I32 or positions.shape != (rows,) or not positions.is_contiguous()):
        raise ValueError(f"positions must be contiguous int32 [{rows}]")
    _norm(k_norm, "k_norm", d)
    _norm(q_norm, "q_norm", d)
    _status(status)
    hq, qp = 0, (None, 0, 0)
    if q is not None:
        if q.dim() != 3 or q.shape[1] < 1:
            raise ValueError(f"q must be bf16 [{rows}, HQ, {d}]")
        hq = q.shape[1]
        qp = _rows(q, "q", rows, hq, d)
        if q_out is None:
            q_out = q.new_empty((rows, hq, d))
        elif q_out.shape != (rows, hq, d) or q_out.dtype is not _BF16 or not q_out.is_contiguous():
            raise ValueError(f"q_out must be contiguous bf16 [{rows}, {hq}, {d}]")
    elif q_norm is not None or q_out is not None:
        raise ValueError("q_norm and q_out need q")
    if rows:
        _call("axk_paged_kv_write_rope" + kind,
              (k, v, kv_cache, kv_scales, cache_location, cos, sin, positions, k_norm, q, q_norm, q_out, status),
              *qp, *kp, *vp, _lib.ptr(q_norm), _lib.ptr(k_norm), _lib.ptr(cos), _lib.ptr(sin), table, n, _lib.ptr(positions),
              cache_location.data_ptr(), _lib.ptr(q_out), kv_cache.data_ptr(), *stored, rows, hq, hkv, d, rot,
              page, p, eps, _lib.ptr(status))
    return q_out


def paged_tree_verify_workspace(batch: int, nodes: int, num_qo_heads: int, num_kv_heads: int, head_dim: int,
                                device) -> torch.Tensor:
    """A byte buffer large enough for paged_tree_verify with this configuration. It carries nothing from call to call; calls
    that may run at the same time (streams, graphs replayed side by side) need one each."""
    n = _lib.load().axk_paged_tree_verify_workspace_size(batch, nodes, num_qo_heads, num_kv_heads, head_dim)
    return torch.empty(n, dtype=_U8, device=device)


def paged_tree_verify(
    q: torch.Tensor,
    kv_cache: torch.Tensor,
    indptr: torch.Tensor,
    indices: torch.Tensor,
    last_page_len: torch.Tensor,
    parents: torch.Tensor,
    sm_scale: Optional[float] = None,
    output: Optional[torch.Tensor] = None,
    kv_scale: Optional[float] = None,
    workspace: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
    kv_scales: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Every drafted node attends its sequence's history, its ancestors and itself: q [B, T, HQ, D] bf16, parents int32 [B, T].
    The page table covers the history and the n nodes of the sequence (up to the last that is one), whose K / V are its last n
    cached tokens in the nodes' order. Returns bf16 [B, T, HQ, D], zeros where there is no node. A chain (-1, 0, 1, ..) gives
    paged_prefill's rows."""
    b = _table(indptr, last_page_len, indices)
    kind, stored, p, page, hkv, d = _cache(kv_cache, kv_scale, kv_scales)
    shape = q.shape
    if len(shape) != 4 or shape[0] != b or shape[3] != d or q.dtype is not _BF16 or not q.is_contiguous():
        raise ValueError(f"q must be contiguous bf16 [{b}, T, HQ, {d}]")
    t, hq = shape[1], shape[2]
    if t < 1 or t > 64:
        raise ValueError(f"{t} nodes: a tree has 1 to 64")
    if hkv < 1 or hq < 1 or hq % hkv or hq // hkv > 16:
        raise ValueError(f"num_qo_heads {hq} must be a multiple (<= 16x) of num_kv_heads {hkv}")
    if page < 16 or page % 16 or page > 4096:
        raise ValueError(f"page_size {page} must be a multiple of 16, at most 4096")
    _parents(parents, b, t)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(d)
    if output is None:
        output = torch.empty_like(q)
    elif output.shape != shape or output.dtype is not _BF16 or not output.is_contiguous():
        raise ValueError(f"output must be contiguous bf16 {list(shape)}")
    _status(status)
    if workspace is None:
        workspace = paged_tree_verify_workspace(b, t, hq, hkv, d, q.device)
    elif workspace.dtype is not _U8 or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous uint8")
    _call("axk_paged_tree_verify" + kind,
          (q, kv_cache, kv_scales, indptr, indices, last_page_len, parents, output, status, workspace), q.data_ptr(),
          kv_cache.data_ptr(), *stored, indptr.data_ptr(), indices.data_ptr(), last_page_len.data_ptr(), parents.data_ptr(),
          output.data_ptr(), indices.numel(), b, t, hq, hkv, d, page, p, sm_scale, _lib.ptr(status), workspace.data_ptr(),
          workspace.numel())
    return output


def _gdn_heads(k: torch.Tensor, nv: int):
    if k.dim() != 4 or k.shape[3] != 128 or k.dtype is not _BF16 or not k.is_contiguous():
        raise ValueError("k must be contiguous bf16 [B, T, NK, 128]")
    b, t, nk, _ = k.shape
    if b < 1 or t < 1 or t > 64:
        raise ValueError(f"{t} nodes of {b} sequences: a tree has 1 to 64")
    if nk < 1 or nv < 1 or nv % nk:
        raise ValueError(f"{nv} value heads must be a multiple of {nk} key heads")
    return b, t, nk


def _made(x, name: str, like: torch.Tensor, dtype, shape):
    if x is None:
        return like.new_empty(shape, dtype=dtype)
    if x.dtype is not dtype or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} {list(shape)}")
    return x


def gdn_tree_verify(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    a_log: torch.Tensor,
    dt_bias: torch.Tensor,
    state: torch.Tensor,
    parents: torch.Tensor,
    output: Optional[torch.Tensor] = None,
    updates: Optional[torch.Tensor] = None,
    gates: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
):
    """gdn_recurrent along every branch of the trees: q, k [B, T, NK, 128] bf16; v [B, T, NV, 128] bf16; a, b [B, T, NV] bf16;
    a_log, dt_bias [NV] f32; state [B, NV, 128, 128] f32, the state before the trees, only read; parents int32 [B, T]; all
    contiguous, value heads in the grouped order (the module's head says what a layer of the other order passes). Returns
    (output bf16 [B, T, NV, 128], updates f32 [B, T, NV, 128], gates f32 [B, T, NV]): every node's output, its rank-1 update
    and log decay (may be -inf), which gdn_tree_commit takes; zeros where there is no node."""
    if v.dim() != 4 or v.dtype is not _BF16 or not v.is_contiguous():
        raise ValueError("v must be contiguous bf16 [B, T, NV, 128]")
    nv = v.shape[2]
    bsz, t, nk = _gdn_heads(k, nv)
    if v.shape != (bsz, t, nv, 128):
        raise ValueError(f"v must be contiguous bf16 [{bsz}, {t}, NV, 128]")
    if q.shape != k.shape or q.dtype is not _BF16 or not q.is_contiguous():
        raise ValueError(f"q must be contiguous bf16 {list(k.shape)}")
    for name, x in (("a", a), ("b", b)):
        if x.shape != (bsz, t, nv) or x.dtype is not _BF16 or not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous bf16 [{bsz}, {t}, {nv}]")
    for name, x in (("a_log", a_log), ("dt_bias", dt_bias)):
        if x.shape != (nv,) or x.dtype is not _F32 or not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 [{nv}]")
    if state.shape != (bsz, nv, 128, 128) or state.dtype is not _F32 or not state.is_contiguous():
        raise ValueError(f"state must be contiguous float32 [{bsz}, {nv}, 128, 128]")
    _parents(parents, bsz, t)
    output = _made(output, "output", v, _BF16, v.shape)
    updates = _made(updates, "updates", v, _F32, v.shape)
    gates = _made(gates, "gates", v, _F32, a.shape)
    _status(status)
    _call("axk_gdn_tree_verify", (q, k, v, a, b, a_log, dt_bias, state, parents, output, updates, gates, status),
          q.data_ptr(), k.data_ptr(), v.data_ptr(), a.data_ptr(), b.data_ptr(), a_log.data_ptr(), dt_bias.data_ptr(),
          state.data_ptr(), parents.data_ptr(), output.data_ptr(), updates.data_ptr(), gates.data_ptr(), bsz, t, nk, nv, 128,
          128, _lib.ptr(status))
    return output, updates, gates


def gdn_tree_commit(
    state: torch.Tensor,
    k: torch.Tensor,
    updates: torch.Tensor,
    gates: torch.Tensor,
    parents: torch.Tensor,
    accepted: torch.Tensor,
    state_out: Optional[torch.Tensor] = None,
    status: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The state after node accepted[b] (int32 [B]; -1: none, the state as it was) of each tree, from gdn_tree_verify's k and
    parents and the updates and gates that it returned. Returns state_out f32 [B, NV, 128, 128]; pass state_out=state to
    update the state in place."""
    if state.dim() != 4 or state.dtype is not _F32 or not state.is_contiguous():
        raise ValueError("state must be contiguous float32 [B, NV, 128, 128]")
    nv = state.shape[1]
    b, t, nk = _gdn_heads(k, nv)
    if state.shape != (b, nv, 128, 128):
        raise ValueError(f"state must be contiguous float32 [{b}, NV, 128, 128]")
    if updates.shape != (b, t, nv, 128) or updates.dtype is not _F32 or not updates.is_contiguous():
        raise ValueError(f"updates must be contiguous float32 [{b}, {t}, {nv}, 128]")
    if gates.shape != (b, t, nv) or gates.dtype is not _F32 or not gates.is_contiguous():
        raise ValueError(f"gates must be contiguous float32 [{b}, {t}, {nv}]")
    _parents(parents, b, t)
    if accepted.shape != (b,) or accepted.dtype is not _I32 or not accepted.is_contiguous():
        raise ValueError(f"accepted must be contiguous int32 [{b}]")
    state_out = _made(state_out, "state_out", state, _F32, state.shape)
    _status(status)
    _call("axk_gdn_tree_commit", (state, k, updates, gates, parents, accepted, state_out, status), state.data_ptr(),
          k.data_ptr(), updates.data_ptr(), gates.data_ptr(), parents.data_ptr(), accepted.data_ptr(), state_out.data_ptr(), b,
          t, nk, nv, 128, 128, _lib.ptr(status))
    return state_out
