"""Limits of the arguments of sparse decode and of the log probabilities, without a GPU: the library's own
checks over a context and a pool made by hand (tests/csrc/args_check.cpp)."""
import os
import shutil
import subprocess

import numpy as np
import pytest

import velokv
from velokv import _capi

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

pytestmark = pytest.mark.skipif(shutil.which("g++") is None or not os.path.exists(_capi.LIB_PATH), reason="g++ or the library not found")


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    """ask(*words): (status, bytes, message)."""
    exe, lib = str(tmp_path_factory.mktemp("args") / "args_check"), os.path.dirname(_capi.LIB_PATH)
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "velo-core_amd", "csrc"), os.path.join(HERE, "csrc", "args_check.cpp"), "-o", exe,
                    os.path.join(lib, "libvelokv.so"), f"-L{ROCM}/lib", "-lamdhip64", f"-Wl,-rpath,{lib}:{ROCM}/lib"], check=True)

    def run(*words):
        r = subprocess.run([exe, *map(str, words)], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stdout + r.stderr
        rc, n, message = r.stdout.split(" ", 2)
        return int(rc), int(n), message.strip()
    return run


def test_scale_of_logits(ask):
    """The kernels take the scale times log2(e) in fp32: where that is infinite a row's largest logit would
    meet 0 * infinity."""
    log2e, up = np.float32(1.4426950408889634), np.float32(np.inf)
    last = np.float32(np.float64(np.finfo(np.float32).max) / np.float64(log2e))
    with np.errstate(over="ignore"):
        while np.isfinite(np.nextafter(last, up) * log2e):
            last = np.nextafter(last, up)
        while not np.isfinite(last * log2e):
            last = np.nextafter(last, -up)
        first = np.nextafter(last, up)
    for ok in (0.0, 1e-45, 1.0, last):
        assert ask("scale", repr(float(ok)))[0] == _capi.OK, ok
    for bad in (first, np.finfo(np.float32).max, np.inf, np.nan, -1.0):
        rc, _, message = ask("scale", repr(float(bad)))
        assert rc == velokv.ERR_BAD_ARG and "scale" in message, bad


def test_length_of_a_list(ask):
    """The kernels count a list's entries in 32 bits and step past its end by up to a workgroup: indices of a
    list near 2^31 entries would wrap to before its start."""
    for n in (1, 512, 1 << 20, 1 << 30):
        assert ask("list", n, 0, 1000)[0] == _capi.OK, n
    for n in ((1 << 30) + 1, 2 ** 31 - 513, 2 ** 31 - 512, 2 ** 31 - 1):
        rc, _, message = ask("list", n, 1, 1000)
        assert rc == velokv.ERR_UNSUPPORTED and str(n) in message, n
