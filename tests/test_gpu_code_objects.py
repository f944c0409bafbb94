"""A deployment of the library and the main code object alone: the context and the dense path work, and
the calls that need another code object say which file they miss."""
import ctypes as C
import os
import shutil

import numpy as np
import pytest

import velokv
from velokv import _capi

pytestmark = pytest.mark.gpu
PKG = os.path.dirname(_capi.LIB_PATH)
BESIDE = {"velokv_sparse_gfx950.co": "vk_sparse_merge", "velokv_logits_gfx950.co": "vk_logprob_part_q0"}


def library(folder):
    """The library as it is loaded from `folder`, which holds a copy of it."""
    L = C.CDLL(shutil.copy(_capi.LIB_PATH, folder))
    for name, argtypes in _capi.PROTOTYPES.items():
        getattr(L, name).argtypes = argtypes
        getattr(L, name).restype = _capi.RESTYPES.get(name, C.c_int)
    L.vk_last_error.restype = C.c_char_p
    return L


@pytest.mark.parametrize("own_path", [False, True])
@pytest.mark.parametrize("there", [[], ["velokv_sparse_gfx950.co"], ["velokv_logits_gfx950.co"]])
def test_main_code_object_alone(ctx, tmp_path, there, own_path):
    L, main = library(tmp_path), "velokv_gfx950.co"
    path = os.path.join(PKG, main).encode() if own_path else None
    for name in there + ([] if own_path else [main]):
        shutil.copy(os.path.join(PKG, name), tmp_path)
    h = C.c_void_p()
    assert L.vk_ctx_create(0, path, C.byref(h)) == _capi.OK, L.vk_last_error()
    for file, kernel in BESIDE.items():
        rc = L.vk_kernel_launch_check(h, kernel.encode(), 256, None)
        assert rc == (_capi.OK if file in there else _capi.ERR_NOT_WIRED)
        assert rc == _capi.OK or file.encode() in L.vk_last_error()
    x = ctx.upload(np.array([[1, 3, 2]], np.float32))
    ids, top = ctx.upload(np.full(1, -7, np.int32)), ctx.alloc(4)
    a = _capi.LogprobArgs(x.ptr, velokv.DT_F32, 0, 1, 3, 0.0, None, 0, None, None, ids.ptr, top.ptr, 1, None, 0)
    rc = L.vk_token_logprobs(h, C.byref(a), None)
    ctx.sync()
    assert (rc, ids.download((1,), np.int32)[0]) == ((_capi.OK, 1) if "velokv_logits_gfx950.co" in there else (_capi.ERR_NOT_WIRED, -7))
    # the dense path: a slot mapping of its own table
    d, pool = _capi.PoolDesc(1, 4, 16, 1, 128, velokv.KV_F16, 1, 4), C.c_void_p()
    assert L.vk_pool_create(h, C.byref(d), C.byref(pool)) == _capi.OK
    pages, at, out = (C.c_uint32 * 2)(3, 1), ctx.upload(np.array([0, 17], np.int32)), ctx.alloc(16)
    assert L.vk_bind_slot(pool, 0, pages, 2) == _capi.OK
    rows = ctx.upload(np.zeros(2, np.int32))
    assert L.vk_slot_mapping(h, pool, None, 0, rows.ptr, at.ptr, 2, out.ptr, None) == _capi.OK
    assert L.vk_stream_sync(h, None) == _capi.OK
    assert out.download((2,), np.int64).tolist() == [48, 17]
    assert L.vk_pool_destroy(pool) == _capi.OK and L.vk_ctx_destroy(h) == _capi.OK


def test_main_code_object_missing(ctx, tmp_path):
    """Without the main code object there is no context."""
    L, h = library(tmp_path), C.c_void_p()
    for name in BESIDE:
        shutil.copy(os.path.join(PKG, name), tmp_path)
    assert L.vk_ctx_create(0, None, C.byref(h)) == _capi.ERR_NOT_WIRED and not h
    assert b"velokv_gfx950.co" in L.vk_last_error()
