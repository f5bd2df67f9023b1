"""Refusals of the tree operators, before anything is launched (CPU): the C entries' status codes, with pointers that are never
followed, and the Python layer's ValueErrors."""
import ctypes

import pytest
import torch

import axk
from axk import _lib

NULL, SHAPE, ALIGN, DTYPE, ALIAS, WORKSPACE = 1, 2, 3, 4, 5, 6
BF16, F32, E4M3 = _lib.DT_BF16, _lib.DT_F32, _lib.DT_FP8E4M3
I32, BF, F = torch.int32, torch.bfloat16, torch.float32


def at(mib, off=0):
    return ctypes.c_void_p((mib << 20) + off)


def rope(q=at(1), ldq=256, hdq=64, k=at(2), ldk=128, hdk=64, v=at(3), ldv=128, hdv=64, qn=at(4), kn=at(5), cos=at(6), sin=at(7),
         tab=F32, n=100, pos=at(8), loc=at(9), out=at(10), cache=at(16), dt=BF16, scale=1.0, rows=3, hq=4, hkv=2, d=64, rot=32,
         page=32, pages=8, status=None):
    return _lib.load().axk_paged_kv_write_rope(q, ldq, hdq, k, ldk, hdk, v, ldv, hdv, qn, kn, cos, sin, tab, n, pos, loc, out,
                                               cache, dt, scale, rows, hq, hkv, d, rot, page, pages, 1e-6, status, None)


def rope_i8(cache=at(16), scales=at(20), **kw):
    a = dict(q=at(1), k=at(2), v=at(3), qn=at(4), kn=at(5), loc=at(9), out=at(10), **kw)
    return _lib.load().axk_paged_kv_write_rope_i8(a["q"], 256, 64, a["k"], 128, 64, a["v"], 128, 64, a["qn"], a["kn"], at(6),
                                                  at(7), F32, 100, at(8), a["loc"], a["out"], cache, scales, 3, 4, 2, 64, 32,
                                                  32, 8, 1e-6, None, None)


def tree(q=at(1), cache=at(16), dt=BF16, scale=1.0, ptr=at(4), idx=at(5), last=at(6), par=at(7), out=at(8), nnz=64, batch=2,
         t=4, hq=4, hkv=2, d=64, page=32, pages=8, status=None, ws=at(64), nbytes=1 << 28):
    return _lib.load().axk_paged_tree_verify(q, cache, dt, scale, ptr, idx, last, par, out, nnz, batch, t, hq, hkv, d, page,
                                             pages, 0.125, status, ws, nbytes, None)


def tree_i8(cache=at(16), scales=at(20), out=at(8)):
    return _lib.load().axk_paged_tree_verify_i8(at(1), cache, scales, at(4), at(5), at(6), at(7), out, 64, 2, 4, 4, 2, 64, 32, 8,
                                                0.125, None, at(64), 1 << 28, None)


GDN = ("q", "k", "v", "a", "b", "a_log", "dt_bias", "state", "parents", "out", "updates", "gates")


def gdn(batch=2, t=4, nk=2, nv=4, dk=128, dv=128, status=None, **kw):
    p = [kw.get(n, at(2 * i + 1)) for i, n in enumerate(GDN)]
    return _lib.load().axk_gdn_tree_verify(*p, batch, t, nk, nv, dk, dv, status, None)


COMMIT = ("state", "k", "updates", "gates", "parents", "accepted", "state_out")


def commit(batch=2, t=4, nk=2, nv=4, dk=128, dv=128, status=None, **kw):
    p = [kw.get(n, at(4 * i + 1)) for i, n in enumerate(COMMIT)]
    return _lib.load().axk_gdn_tree_commit(*p, batch, t, nk, nv, dk, dv, status, None)


@pytest.mark.parametrize("kw,want", [
    *[({n: None}, NULL) for n in ("q", "k", "v", "cos", "sin", "loc", "out", "cache")],
    (dict(hq=0), NULL), (dict(rows=-1), SHAPE), (dict(rows=(1 << 24) + 1), SHAPE), (dict(hq=-1), SHAPE), (dict(hkv=0), SHAPE),
    (dict(d=96), SHAPE), (dict(rot=24), SHAPE), (dict(rot=80), SHAPE), (dict(rot=-16), SHAPE), (dict(page=0), SHAPE),
    (dict(pages=0), SHAPE), (dict(pages=1 << 31), SHAPE), (dict(n=0), SHAPE), (dict(pos=None, n=2), SHAPE),
    (dict(dt=F32), DTYPE), (dict(tab=E4M3), DTYPE), (dict(dt=E4M3, scale=3.0), SHAPE), (dict(dt=E4M3, scale=0.0), SHAPE),
    (dict(ldq=-8), SHAPE), (dict(ldk=(1 << 32) + 8), SHAPE), (dict(ldv=100), ALIGN), (dict(hdk=4), ALIGN),
    *[({n: at(i, o)}, ALIGN) for n, i, o in (("q", 1, 8), ("k", 2, 8), ("v", 3, 8), ("cos", 6, 8), ("sin", 7, 8), ("qn", 4, 4),
                                             ("kn", 5, 8), ("cache", 16, 8), ("out", 10, 8), ("loc", 9, 2), ("pos", 8, 1),
                                             ("status", 11, 2))],
    (dict(out=at(1)), ALIAS), (dict(out=at(3, 512)), ALIAS), (dict(cache=at(2)), ALIAS), (dict(out=at(16, 4096)), ALIAS),
    (dict(status=at(9)), ALIAS), (dict(out=at(6)), ALIAS), (dict(rows=1 << 24, hq=4096, d=256), SHAPE)])
def test_append_refuses(kw, want):
    assert rope(**kw) == want


def test_append_of_no_rows_and_int8():
    assert rope(rows=0) == 0
    assert rope_i8(scales=None) == NULL
    assert rope_i8(scales=at(20, 1)) == ALIGN
    assert rope_i8(scales=at(16, 64)) == ALIAS
    assert rope_i8(scales=at(1)) == ALIAS


@pytest.mark.parametrize("kw,want", [
    *[({n: None}, NULL) for n in ("q", "cache", "ptr", "idx", "last", "par", "out")],
    (dict(batch=0), SHAPE), (dict(t=0), SHAPE), (dict(t=65), SHAPE), (dict(hq=3), SHAPE), (dict(hq=0), SHAPE),
    (dict(hkv=0), SHAPE), (dict(hq=34), SHAPE), (dict(d=96), SHAPE), (dict(page=24), SHAPE), (dict(page=8192), SHAPE),
    (dict(pages=0), SHAPE), (dict(nnz=-1), SHAPE), (dict(nnz=1 << 28), SHAPE), (dict(batch=(1 << 20) + 1), SHAPE),
    (dict(dt=F32), DTYPE), (dict(dt=E4M3, scale=-2.0), SHAPE), (dict(dt=E4M3, scale=6.0), SHAPE),
    *[({n: at(i, o)}, ALIGN) for n, i, o in (("q", 1, 8), ("cache", 16, 8), ("out", 8, 4), ("ptr", 4, 2), ("idx", 5, 2),
                                             ("last", 6, 2), ("par", 7, 2), ("status", 9, 1))],
    (dict(ws=None), WORKSPACE), (dict(nbytes=0), WORKSPACE), (dict(ws=at(64, 128)), WORKSPACE),
    (dict(out=at(1)), ALIAS), (dict(out=at(16)), ALIAS), (dict(ws=at(1)), ALIAS), (dict(ws=at(8)), ALIAS),
    (dict(status=at(7, 4)), ALIAS)])
def test_tree_refuses(kw, want):
    assert tree(**kw) == want


def test_tree_int8_and_workspace_size():
    assert tree_i8(scales=None) == NULL
    assert tree_i8(scales=at(20, 1)) == ALIGN
    assert tree_i8(out=at(20)) == ALIAS
    size = _lib.load().axk_paged_tree_verify_workspace_size
    need = size(2, 4, 4, 2, 64)
    assert 0 < need < 1 << 28 and tree(nbytes=need - 1) == WORKSPACE
    for bad in ((0, 4, 4, 2, 64), (2, 0, 4, 2, 64), (2, 65, 4, 2, 64), (2, 4, 3, 2, 64), (2, 4, 4, 2, 80)):
        assert size(*bad) == 0
    # nothing is cut where the sequences fill the device by themselves
    assert size(4096, 64, 512, 512, 256) == 0


def test_a_batch_that_is_not_cut_needs_no_merge():
    """2^24 rows of nodes were taken for more than a merge launch holds, but such a batch makes none. (The check of overlaps comes
    behind that of sizes, and nothing is launched.)"""
    assert tree(batch=1 << 18, t=64, hq=1, hkv=1, nnz=0, out=at(1)) == ALIAS
    assert tree(batch=256, t=64, hq=4096, hkv=256, nnz=1 << 20, out=at(1)) == ALIAS
    assert tree(batch=1 << 20, t=64, hq=16 * 64, hkv=64, nnz=0, out=at(1)) == SHAPE  # 2^29 workgroups


@pytest.mark.parametrize("kw,want", [
    *[({n: None}, NULL) for n in GDN],
    (dict(batch=0), SHAPE), (dict(t=0), SHAPE), (dict(t=65), SHAPE), (dict(nk=3), SHAPE), (dict(nk=0), SHAPE), (dict(nv=0), SHAPE),
    (dict(dk=64), SHAPE), (dict(dv=256), SHAPE), (dict(batch=1 << 19), SHAPE),
    (dict(q=at(1, 8)), ALIGN), (dict(k=at(3, 8)), ALIGN), (dict(state=at(15, 4)), ALIGN), (dict(updates=at(21, 4)), ALIGN),
    (dict(parents=at(17, 2)), ALIGN), (dict(status=at(30, 1)), ALIGN),
    (dict(out=at(5)), ALIAS), (dict(updates=at(15)), ALIAS), (dict(gates=at(21)), ALIAS), (dict(status=at(17)), ALIAS)])
def test_gdn_refuses(kw, want):
    assert gdn(**kw) == want


@pytest.mark.parametrize("kw,want", [
    *[({n: None}, NULL) for n in COMMIT],
    (dict(batch=0), SHAPE), (dict(t=65), SHAPE), (dict(nv=3), SHAPE), (dict(dk=64), SHAPE),
    (dict(state=at(1, 8)), ALIGN), (dict(updates=at(9, 8)), ALIGN), (dict(accepted=at(21, 2)), ALIGN),
    (dict(state_out=at(1, 65536)), ALIAS), (dict(state_out=at(9)), ALIAS), (dict(status=at(21)), ALIAS)])
def test_commit_refuses(kw, want):
    assert commit(**kw) == want


def raises(what, f, *args, **kw):
    with pytest.raises(ValueError, match=what):
        f(*args, **kw)


def test_append_arguments():
    k, v, cache = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF), torch.zeros(4, 2, 16, 2, 64, dtype=BF)
    loc, tab, q = torch.zeros(3, 2, dtype=I32), torch.zeros(9, 16), torch.zeros(3, 4, 64, dtype=BF)
    f = axk.store_paged_kv_rope
    raises("k must", f, k.view(3, 128), v, cache, loc)
    raises("k must", f, k.float(), v, cache, loc)
    raises("v must", f, k, v[:2], cache, loc)
    raises("contiguous channels", f, k, torch.zeros(3, 64, 2, dtype=BF).transpose(1, 2), cache, loc)
    raises("strides", f, torch.zeros(3, 2, 68, dtype=BF)[..., :64], v, cache, loc)
    raises("cache_location", f, k, v, cache, loc.long())
    raises("cache_location", f, k, v, cache, loc[:2])
    raises("go together", f, k, v, cache, loc, tab)
    raises("cos and sin must", f, k, v, cache, loc, tab, tab.bfloat16())
    raises("cos and sin must", f, k, v, cache, loc, tab.half(), tab.half())
    raises("multiple of 16", f, k, v, cache, loc, tab[:, :12].contiguous(), tab[:, :12].contiguous())
    raises("at most 64", f, k, v, cache, loc, torch.zeros(9, 40), torch.zeros(9, 40))
    raises("positions", f, k, v, cache, loc, tab[:2], tab[:2])
    raises("0 positions", f, k, v, cache, loc, tab[:0], tab[:0], torch.zeros(3, dtype=I32))
    raises("positions must", f, k, v, cache, loc, tab, tab, torch.zeros(2, dtype=I32))
    raises("k_norm", f, k, v, cache, loc, k_norm=torch.zeros(64, dtype=BF))
    raises("need q", f, k, v, cache, loc, q_norm=torch.zeros(64))
    raises("need q", f, k, v, cache, loc, q_out=q)
    raises("q must", f, k, v, cache, loc, q=q[:2])
    raises("q_out", f, k, v, cache, loc, q=q, q_out=q.float())
    raises(None, f, k, v, cache.view(torch.int8), loc)  # int8 without its scales
    raises(None, f, k, v, cache[0], loc)


def test_tree_arguments():
    q, cache = torch.zeros(2, 3, 4, 64, dtype=BF), torch.zeros(4, 2, 16, 2, 64, dtype=BF)
    table = [torch.tensor([0, 1, 2], dtype=I32), torch.tensor([0, 1], dtype=I32), torch.tensor([5, 5], dtype=I32)]
    par = torch.full((2, 3), -2, dtype=I32)
    f = axk.paged_tree_verify
    raises("q must", f, q[0], cache, *table, par)
    raises("q must", f, q[:1], cache, *table, par)
    raises("q must", f, q.float(), cache, *table, par)
    raises("q must", f, q.transpose(1, 2), cache, *table, par)
    raises("1 to 64", f, q[:, :0], cache, *table, par)
    raises("1 to 64", f, torch.zeros(2, 65, 4, 64, dtype=BF), cache, *table, par)
    raises("multiple", f, q[:, :, :3].contiguous(), cache, *table, par)
    raises("page_size", f, q, torch.zeros(4, 2, 24, 2, 64, dtype=BF), *table, par)
    raises("parents", f, q, cache, *table, par.long())
    raises("parents", f, q, cache, *table, par[:, :2])
    raises("output", f, q, cache, *table, par, output=q[:1])
    raises("workspace", f, q, cache, *table, par, workspace=torch.zeros(8))
    raises("status", f, q, cache, *table, par, status=torch.zeros(1))


def test_gdn_arguments():
    k, v, a = torch.zeros(2, 3, 2, 128, dtype=BF), torch.zeros(2, 3, 4, 128, dtype=BF), torch.zeros(2, 3, 4, dtype=BF)
    h, state, par = torch.zeros(4), torch.zeros(2, 4, 128, 128), torch.full((2, 3), -2, dtype=I32)
    good = dict(q=k, k=k, v=v, a=a, b=a, a_log=h, dt_bias=h, state=state, parents=par)
    for name, bad in (("v", v.float()), ("v", v[:1]), ("k", k[..., :64]), ("k", k[:, :, :0]), ("q", k[:1]), ("q", k.float()),
                      ("a", a[:1]), ("b", a.float()), ("a_log", h.double()), ("dt_bias", h[:3]), ("state", state[:1]),
                      ("state", state.bfloat16()), ("state", state.transpose(2, 3)), ("parents", par[:1]), ("output", v.float()),
                      ("updates", v), ("gates", a), ("status", h)):
        with pytest.raises(ValueError):
            axk.gdn_tree_verify(**{**good, name: bad})
    many = torch.zeros(1, 65, 2, 128, dtype=BF)
    with pytest.raises(ValueError, match="1 to 64"):
        axk.gdn_tree_verify(**{**good, "k": many})
    u, g, acc = torch.zeros(2, 3, 4, 128), torch.zeros(2, 3, 4), torch.zeros(2, dtype=I32)
    good = dict(state=state, k=k, updates=u, gates=g, parents=par, accepted=acc)
    for name, bad in (("state", state[:1]), ("state", state[0]), ("k", k[:, :2]), ("updates", u.bfloat16()), ("gates", g[:1]),
                      ("parents", par.long()), ("accepted", acc[:1]), ("accepted", acc.long()), ("state_out", state[:1]),
                      ("status", h)):
        with pytest.raises(ValueError):
            axk.gdn_tree_commit(**{**good, name: bad})
