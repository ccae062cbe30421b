"""CPU check of how uploaded weights are replaced (csrc/gx_upload.h, run by upload_emu.cpp): in place when the call
returns, and on any failure the ones before stay."""
import ctypes
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
OK, NOMEM, TIMEOUT, DEVICE = 0, -2, -3, -4


@pytest.fixture(scope="module")
def replace(tmp_path_factory):
    so = tmp_path_factory.mktemp("up") / "up.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", str(HERE / "upload_emu.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))

    def call(alloc=0, copy=-1, answer=OK, remove=0):
        out, live, in_use = (ctypes.c_uint8 * 12)(), ctypes.c_int(), ctypes.c_int()
        r = lib.replace_twice(alloc, copy, answer, remove, out, ctypes.byref(live), ctypes.byref(in_use))
        assert in_use.value == 0
        return r, bytes(out), live.value
    return call


def test_new_weights_are_in_place_when_the_call_returns(replace):
    assert replace() == (OK, b"\2\2\2\2\xee\xee\xee\xee\2\2\2\2", 1)
    assert replace(remove=1) == (OK, bytes(12), 0)


@pytest.mark.parametrize("fault,answer", [(dict(alloc=1), NOMEM), (dict(copy=0), DEVICE), (dict(copy=1), DEVICE),
                                          (dict(answer=DEVICE), DEVICE), (dict(answer=-9), -9)])
def test_a_failed_call_leaves_the_old_weights(replace, fault, answer):
    assert replace(**fault) == (answer, bytes([1] * 12), 1)


def test_a_timeout_frees_nothing_that_a_copy_may_write(replace):
    assert replace(answer=TIMEOUT) == (TIMEOUT, bytes([1] * 12), 2)
    assert replace(answer=TIMEOUT, remove=1) == (TIMEOUT, bytes([1] * 12), 1)
