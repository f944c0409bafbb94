"""Sparse decode and log probabilities without a GPU: null handles and arguments are errors, not faults."""
import ctypes as C
import os
import re
import subprocess

import pytest

import velokv
from velokv import _capi


def test_null_handles_and_arguments():
    lib, n = _capi.lib(), C.c_uint64()
    a, b = _capi.SparseArgs(), _capi.LogprobArgs()
    assert lib.vk_index_create(None, None, None) == velokv.ERR_NOT_WIRED
    assert lib.vk_index_update(None, None, 0, None, 0, None, None, None, 0, 0, 0, None) == velokv.ERR_NOT_WIRED
    assert lib.vk_index_read(None, None, 0, None, 0, None, None, None) == velokv.ERR_NOT_WIRED
    for call in (lib.vk_select_pages, lib.vk_sparse_decode, lib.vk_select_decode):
        assert call(None, None, C.byref(a), None) == velokv.ERR_NOT_WIRED
    assert lib.vk_token_logprobs(None, C.byref(b), None) == velokv.ERR_NOT_WIRED
    assert lib.vk_index_destroy(None) == _capi.OK
    assert lib.vk_index_bytes(None, C.byref(n)) == velokv.ERR_BAD_ARG
    assert lib.vk_sparse_workspace(None, C.byref(a), C.byref(n)) == velokv.ERR_BAD_ARG
    assert lib.vk_token_logprobs_workspace(None, C.byref(b), C.byref(n)) == velokv.ERR_BAD_ARG
    assert b"null" in lib.vk_last_error()


def test_verify_result_without_log_probabilities():
    assert velokv.TreeVerifyResult([1, 2]).logprobs == []


@pytest.mark.parametrize("name", ["sparse", "logits"])
def test_kernels_use_no_scratch_memory(name):
    """No kernel of the two code objects spills a register or keeps anything in scratch memory."""
    co = _capi.CODE_OBJECT_PATH.replace("velokv_gfx950", f"velokv_{name}_gfx950")
    readelf = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-readelf")
    if not (os.path.exists(co) and os.path.exists(readelf)):
        pytest.skip("no built code object or no llvm-readelf")
    notes = subprocess.run([readelf, "--notes", co], capture_output=True, text=True, check=True).stdout
    found = re.findall(r"\.(private_segment_fixed_size|vgpr_spill_count):\s+(\d+)", notes)
    assert found and all(int(n) == 0 for _, n in found)
