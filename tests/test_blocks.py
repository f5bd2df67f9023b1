"""Refusals of the block operators, before anything is launched (CPU): the C entries' status codes, with pointers that are
never followed, and the Python layer's ValueErrors."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import axk
from axk import _lib

NULL, SHAPE, ALIGN, DTYPE, ALIAS, WORKSPACE = 1, 2, 3, 4, 5, 6
BF16, E4M3 = _lib.DT_BF16, _lib.DT_FP8E4M3


def at(mib, off=0):
    return ctypes.c_void_p((mib << 20) + off)


def write(k=at(1), v=at(2), cache=at(16), dt=BF16, scale=1.0, bounds=at(3), loc=at(4), rows=2, hkv=2, d=64, page=32,
          block=16, pages=8):
    return _lib.load().axk_paged_kv_write_bounds(k, v, cache, dt, scale, bounds, loc, rows, hkv, d, page, block, pages,
                                                 None, None)


def bounds_(cache=at(16), dt=BF16, scale=1.0, bounds=at(3), ptr=at(4), idx=at(5), last=at(6), nnz=8, batch=2, hkv=2, d=64,
            page=32, block=16, pages=8):
    return _lib.load().axk_paged_key_bounds(cache, dt, scale, bounds, ptr, idx, last, None, nnz, batch, hkv, d, page,
                                            block, pages, None, None)


def scores(q=at(1), bounds=at(3), ptr=at(4), idx=at(5), last=at(6), out=at(7), nnz=8, batch=2, hq=4, hkv=2, d=64, page=32,
           block=16, pages=8):
    return _lib.load().axk_paged_block_scores(q, bounds, ptr, idx, last, out, nnz, batch, hq, hkv, d, page, block, pages,
                                              None, None)


def select(sc=at(1), ptr=at(4), last=at(6), out=at(7), nnz=8, batch=2, hkv=2, page=32, block=16, n=4, first=1, keep=1):
    return _lib.load().axk_paged_select_blocks(sc, ptr, last, out, nnz, batch, hkv, page, block, n, first, keep, None)


def decode(q=at(1), cache=at(16), dt=BF16, scale=1.0, ptr=at(4), idx=at(5), last=at(6), blocks=at(7), block=16, n=4,
           out=at(8), win=None, wout=None, nnz=8, batch=2, hq=4, hkv=2, d=64, page=32, pages=8, ws=at(32), bytes_=1 << 24):
    return _lib.load().axk_paged_decode_blocks(q, cache, dt, scale, ptr, idx, last, blocks, block, n, out, win, wout, 1.0,
                                               nnz, batch, hq, hkv, d, page, pages, 0.125, None, ws, bytes_, None)


def evict(w=at(1), ptr=at(2), idx=at(3), optr=at(4), oidx=at(5), ow=at(6), freed=at(7), nnz=8, batch=2, hkv=2, budget=4,
          first=1, keep=1):
    return _lib.load().axk_paged_evict_pages(w, ptr, idx, optr, oidx, ow, freed, nnz, batch, hkv, budget, first, keep,
                                             None)


def write_i8(cache=at(16), scales=at(24), bounds=at(3), rows=2, d=64, hkv=2):
    return _lib.load().axk_paged_kv_write_bounds_i8(at(1), at(2), cache, scales, bounds, at(4), rows, hkv, d, 32, 16, 8, None,
                                                    None)


def bounds_i8(scales=at(24), bounds=at(3), d=64):
    return _lib.load().axk_paged_key_bounds_i8(at(16), scales, bounds, at(4), at(5), at(6), None, 8, 2, 2, d, 32, 16, 8,
                                               None, None)


def decode_i8(scales=at(24), out=at(8), ws=at(32), d=64):
    return _lib.load().axk_paged_decode_blocks_i8(at(1), at(16), scales, at(4), at(5), at(6), None, 0, 0, out, None, None,
                                                  1.0, 8, 2, 4, 2, d, 32, 8, 0.125, None, ws, 1 << 24, None)


@pytest.mark.parametrize("call,code", [
    (lambda: write_i8(scales=None), NULL), (lambda: write_i8(scales=at(24, 1)), ALIGN), (lambda: write_i8(scales=at(16)), ALIAS),
    (lambda: write_i8(bounds=at(24)), ALIAS), (lambda: write_i8(d=80), SHAPE), (lambda: write_i8(rows=1 << 15), SHAPE),
    (lambda: bounds_i8(scales=None), NULL), (lambda: bounds_i8(bounds=at(24)), ALIAS), (lambda: bounds_i8(d=512), SHAPE),
    (lambda: decode_i8(scales=None), NULL), (lambda: decode_i8(scales=at(24, 1)), ALIGN), (lambda: decode_i8(ws=None), WORKSPACE),
    (lambda: decode_i8(out=at(16)), ALIAS),
    (lambda: write(k=None), NULL), (lambda: write(bounds=None), NULL), (lambda: write(loc=None), NULL),
    (lambda: write(d=96), SHAPE), (lambda: write(page=24), SHAPE), (lambda: write(block=24), SHAPE),
    (lambda: write(page=48, block=32), SHAPE), (lambda: write(page=8192, block=16), SHAPE),
    (lambda: write(hkv=0), SHAPE), (lambda: write(pages=0), SHAPE), (lambda: write(rows=-1), SHAPE), (lambda: write(rows=16385), SHAPE),
    (lambda: write(dt=_lib.DT_F16), DTYPE), (lambda: write(dt=E4M3, scale=3.0), SHAPE),
    (lambda: write(dt=E4M3, scale=float("nan")), SHAPE), (lambda: write(k=at(1, 8)), ALIGN),
    (lambda: write(bounds=at(3, 2)), ALIGN), (lambda: write(bounds=at(16)), ALIAS), (lambda: write(k=at(16)), ALIAS),
    (lambda: bounds_(cache=None), NULL), (lambda: bounds_(idx=None), NULL), (lambda: bounds_(batch=0), SHAPE),
    (lambda: bounds_(nnz=-1), SHAPE), (lambda: bounds_(nnz=(1 << 28) + 1, page=64), SHAPE), (lambda: bounds_(d=32), SHAPE),
    (lambda: bounds_(dt=_lib.DT_U8), DTYPE), (lambda: bounds_(dt=E4M3, scale=0.0), SHAPE),
    (lambda: bounds_(cache=at(16, 8)), ALIGN), (lambda: bounds_(bounds=at(16, 4096)), ALIAS),
    (lambda: scores(out=None), NULL), (lambda: scores(q=None), NULL), (lambda: scores(hq=3), SHAPE),
    (lambda: scores(hq=34), SHAPE), (lambda: scores(hq=0), SHAPE), (lambda: scores(block=0), SHAPE),
    (lambda: scores(q=at(1, 2)), ALIGN), (lambda: scores(out=at(1)), ALIAS), (lambda: scores(out=at(3)), ALIAS),
    (lambda: select(sc=None), NULL), (lambda: select(out=None), NULL), (lambda: select(n=0), SHAPE),
    (lambda: select(n=1), SHAPE), (lambda: select(first=-1), SHAPE), (lambda: select(first=4), SHAPE),
    (lambda: select(block=48), SHAPE), (lambda: select(out=at(1)), ALIAS),
    (lambda: decode(q=None), NULL), (lambda: decode(blocks=None), NULL), (lambda: decode(n=0), SHAPE),
    (lambda: decode(n=-1), SHAPE), (lambda: decode(win=at(9)), NULL), (lambda: decode(hq=5), SHAPE),
    (lambda: decode(hq=34), SHAPE), (lambda: decode(block=8), SHAPE), (lambda: decode(dt=_lib.DT_F32), DTYPE),
    (lambda: decode(dt=E4M3, scale=6.0), SHAPE), (lambda: decode(q=at(1, 8)), ALIGN), (lambda: decode(out=at(8, 4)), ALIGN),
    (lambda: decode(wout=at(9), ws=None), WORKSPACE), (lambda: decode(wout=at(9), bytes_=64), WORKSPACE),
    (lambda: decode(wout=at(9), ws=at(32, 128)), WORKSPACE), (lambda: decode(blocks=None, n=0, ws=None), WORKSPACE),
    (lambda: decode(out=at(1)), ALIAS), (lambda: decode(out=at(16)), ALIAS),
    (lambda: decode(win=at(9), wout=at(9, 4)), ALIAS), (lambda: decode(wout=at(8)), ALIAS),
    (lambda: decode(wout=at(32)), ALIAS), (lambda: decode(win=at(32), wout=at(9)), ALIAS),
    (lambda: evict(w=None), NULL), (lambda: evict(freed=None), NULL), (lambda: evict(batch=0), SHAPE),
    (lambda: evict(budget=1), SHAPE), (lambda: evict(keep=0), SHAPE), (lambda: evict(first=-1), SHAPE),
    (lambda: evict(oidx=at(3)), ALIAS), (lambda: evict(ow=at(1)), ALIAS), (lambda: evict(freed=at(5)), ALIAS),
    (lambda: evict(optr=at(2)), ALIAS), (lambda: evict(oidx=at(5, 2)), ALIGN),
])
def test_entries_refuse_before_a_launch(call, code):
    assert call() == code


def test_workspace_size():
    size = _lib.load().axk_paged_decode_blocks_workspace_size
    assert size(2, 4, 2, 64, 32, 8, 16, 4, 0) == 0  # one piece a row: written directly
    assert size(2, 4, 2, 64, 32, 8, 16, 4, 1) > 0
    assert size(2, 4, 2, 64, 32, 8, 16, 0, 0) > 0   # every block: rows of several pieces
    assert size(2, 5, 2, 64, 32, 8, 16, 0, 1) == 0  # refused shape
    assert size(2, 4, 2, 96, 32, 8, 16, 0, 1) == 0
    # listed blocks: the size follows the list, not the cache
    assert size(2, 4, 2, 64, 32, 1 << 16, 16, 512, 1) == size(2, 4, 2, 64, 32, 8, 16, 512, 1)


def table(b=2, nnz=4):
    return torch.tensor([0] + [nnz] * b, dtype=torch.int32), torch.zeros(nnz, dtype=torch.int32), \
        torch.ones(b, dtype=torch.int32)


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


CACHE = bf(4, 2, 32, 2, 64)
BOUNDS = bf(4, 2, 2, 2, 64)
U8 = torch.zeros(4, 2, 32, 2, 64, dtype=torch.uint8)


@pytest.mark.parametrize("call,match", [
    (lambda t: axk.store_paged_kv_bounds(bf(2, 2, 64), bf(2, 2, 64), U8, BOUNDS, torch.zeros(2, 2, dtype=torch.int32)),
     "kv_scale"),
    (lambda t: axk.store_paged_kv_bounds(bf(2, 2, 64), bf(2, 2, 64), CACHE, BOUNDS, torch.zeros(2, 2, dtype=torch.int32),
                                         kv_scale=8.0), "kv_scale"),
    (lambda t: axk.store_paged_kv_bounds(bf(2, 2, 64), bf(2, 2, 64), CACHE.to(torch.int16), BOUNDS,
                                         torch.zeros(2, 2, dtype=torch.int32)), "bfloat16, u8"),
    (lambda t: axk.store_paged_kv_bounds(bf(2, 2, 64), bf(2, 2, 64), CACHE.to(torch.int8), BOUNDS,
                                         torch.zeros(2, 2, dtype=torch.int32)), "kv_scales"),
    (lambda t: axk.paged_key_bounds(CACHE.to(torch.int8), BOUNDS, *t, kv_scales=bf(4, 2, 32, 3)), "kv_scales"),
    (lambda t: axk.paged_key_bounds(CACHE, BOUNDS, *t, kv_scales=bf(4, 2, 32, 2)), "INT8"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), CACHE.to(torch.int8), *t, kv_scale=8.0, kv_scales=bf(4, 2, 32, 2)),
     "FP8"),
    (lambda t: axk.store_paged_kv_bounds(bf(2, 2, 64), bf(2, 2, 64), CACHE, BOUNDS, torch.zeros(3, 2, dtype=torch.int32)),
     "cache_location"),
    (lambda t: axk.store_paged_kv_bounds(bf(2, 3, 64), bf(2, 3, 64), CACHE, BOUNDS, torch.zeros(2, 2, dtype=torch.int32)),
     "k and v"),
    (lambda t: axk.paged_key_bounds(CACHE, bf(4, 3, 2, 2, 64), *t), "bounds"),
    (lambda t: axk.paged_key_bounds(CACHE, bf(4, 4, 2, 2, 64), *t), "block_size"),
    (lambda t: axk.paged_key_bounds(CACHE, BOUNDS.float(), *t), "bounds"),
    (lambda t: axk.paged_key_bounds(CACHE[:, :, :16], BOUNDS, *t), "contiguous"),
    (lambda t: axk.paged_key_bounds(CACHE, BOUNDS, t[0][:2], t[1], t[2]), "indptr"),
    (lambda t: axk.paged_key_bounds(CACHE, BOUNDS, *t, start=torch.zeros(2)), "start"),
    (lambda t: axk.paged_key_bounds(CACHE, BOUNDS, *t, status=torch.zeros(1)), "status"),
    (lambda t: axk.paged_block_scores(bf(3, 4, 64), BOUNDS, *t, 32), "q must"),
    (lambda t: axk.paged_block_scores(bf(2, 5, 64), BOUNDS, *t, 32), "num_qo_heads"),
    (lambda t: axk.paged_block_scores(bf(2, 4, 64), BOUNDS, *t, 33), "bounds"),
    (lambda t: axk.paged_block_scores(bf(2, 4, 64), BOUNDS, *t, 32, output=torch.zeros(2, 7)), "output"),
    (lambda t: axk.paged_select_blocks(torch.zeros(2, 8), t[0], t[2], 32, 16, 1), "num_select"),
    (lambda t: axk.paged_select_blocks(torch.zeros(2, 7), t[0], t[2], 32, 16, 4), "scores"),
    (lambda t: axk.paged_select_blocks(torch.zeros(2, 8).double(), t[0], t[2], 32, 16, 4), "scores"),
    (lambda t: axk.paged_select_blocks(torch.zeros(2, 8), t[0], t[2], 32, 24, 4), "block_size"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), CACHE, *t, blocks=torch.zeros(2, 2, 4, dtype=torch.int32)),
     "block_size"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), CACHE, *t, blocks=torch.zeros(2, 2, 4), block_size=16), "blocks"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), CACHE, *t, weights_in=torch.zeros(2, 4)), "weights_in without"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), CACHE, *t, weights=torch.zeros(2, 5)), "weights"),
    (lambda t: axk.paged_decode_blocks(bf(2, 34, 64), CACHE, *t), "num_qo_heads"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 128), CACHE, *t), "q must"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), U8, *t, kv_scale=5.0), "power of two"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), CACHE, *t, workspace=torch.zeros(4)), "workspace"),
    (lambda t: axk.paged_evict_pages(torch.zeros(2, 4), t[0], t[1], 1), "budget"),
    (lambda t: axk.paged_evict_pages(torch.zeros(2, 4), t[0], t[1], 4, keep_last=0), "budget"),
    (lambda t: axk.paged_evict_pages(torch.zeros(2, 3), t[0], t[1], 4), "weights"),
    (lambda t: axk.paged_evict_pages(torch.zeros(2, 4), t[0].long(), t[1], 4), "indptr"),
    # host tensors, with nothing else wrong
    (lambda t: axk.paged_evict_pages(torch.zeros(2, 4), t[0], t[1], 4), "device tensors"),
    (lambda t: axk.paged_decode_blocks(bf(2, 4, 64), CACHE, *t), "device tensors"),
])
def test_python_layer_raises_value_error(call, match):
    with pytest.raises(ValueError, match=match):
        call(table())


@pytest.mark.parametrize("call", [
    # a launch holds fewer than 2^32 threads: 256 a block of bounds, 64 for 16 blocks' scores of a head, 256 or 1024 a
    # selected row, 256 a piece of a decode and a part of its merge
    lambda: bounds_(nnz=1 << 24, page=16, block=16),
    lambda: bounds_(nnz=1 << 20, page=256, block=16),
    lambda: scores(nnz=1 << 20, hq=1024, hkv=1024, page=16, block=16),
    lambda: select(nnz=4096, batch=1 << 20, hkv=4),
    lambda: select(nnz=8, batch=1 << 20, hkv=16),
    lambda: decode(batch=1 << 16, hq=16, hkv=16, n=1 << 13),
    lambda: decode(batch=1 << 20, hq=16, hkv=16, n=1),
    lambda: decode(batch=1 << 20, hq=256, hkv=16, d=256, blocks=None, n=0),
])
def test_launches_that_do_not_fit_are_refused(call):
    assert call() == SHAPE


def test_workspace_of_a_launch_that_does_not_fit():
    size = _lib.load().axk_paged_decode_blocks_workspace_size
    assert size(1 << 16, 16, 16, 64, 32, 8, 16, 1 << 13, 0) == 0
    assert size(1 << 10, 16, 16, 64, 32, 8, 16, 1 << 13, 0) > 0


W = dict(wout=at(9))


@pytest.mark.parametrize("call", [
    # the tables that a call reads, or that its second kernel reads again, under what it writes
    lambda: write(loc=at(16)), lambda: write(loc=at(3)),
    lambda: bounds_(ptr=at(3)), lambda: bounds_(idx=at(3, 16)), lambda: bounds_(last=at(3)),
    lambda: bounds_with_start(at(3)),
    lambda: scores(out=at(4)), lambda: scores(out=at(5)), lambda: scores(out=at(6)),
    lambda: select(out=at(4)), lambda: select(out=at(6)),
    lambda: decode(out=at(4, 8)), lambda: decode(out=at(5)), lambda: decode(out=at(6)), lambda: decode(out=at(7)),
    lambda: decode(wout=at(4)), lambda: decode(wout=at(5)), lambda: decode(wout=at(6)), lambda: decode(wout=at(7)),
    lambda: decode(ws=at(4), **W), lambda: decode(ws=at(5), **W), lambda: decode(ws=at(6), **W), lambda: decode(ws=at(7), **W),
    lambda: decode(out=at(10), win=at(10), **W),
    lambda: decode_i8(out=at(24)), lambda: decode_i8(ws=at(24)),
    lambda: write_i8(scales=at(4)),
])
def test_overlapping_arrays_are_refused(call):
    assert call() == ALIAS


def bounds_with_start(start):
    return _lib.load().axk_paged_key_bounds(at(16), BF16, 1.0, at(3), at(4), at(5), at(6), start, 8, 2, 2, 64, 32, 16, 8,
                                            None, None)


def test_import_beside_a_torch_that_was_built_without_a_gpu():
    """Such a torch lacks the stream functions of its extension module: the codecs and configs import all the same."""
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]: delattr(torch._C, n)\n"
            "import axk\n"
            "from axk import configs\n"
            "print(axk.quantize_nvfp4(torch.ones(16, 32))[0].shape, len(dir(configs)) > 0)\n")
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(axk.__file__))))
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, timeout=300)
    assert got.returncode == 0, got.stderr
