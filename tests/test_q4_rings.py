"""CPU check of the rings of the 4-bit batch product (csrc/gx_q4_tc.h, walked through by ring_emu.cpp): whatever
order copies land in and warps run in, every unit is decoded and multiplied from its own bytes."""
import ctypes
import subprocess
from pathlib import Path

import pytest

from gyro_moe import abi

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    so = tmp_path_factory.mktemp("ring") / "ring.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", str(HERE / "ring_emu.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.ring_walk.argtypes = [ctypes.c_uint32, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_uint64, ctypes.c_uint64]
    return lib.ring_walk


@pytest.mark.parametrize("kind", [abi.GX_Q4_0, abi.GX_Q4_1])
@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("tokens", [16, 32, 64])
def test_units_are_read_as_they_were_copied(walk, kind, bf16, tokens):
    for total in (1, 2, 3, 7, 40):
        for slow in [0] + [1 << u for u in range(min(total, 16))] + [0x5555, 0x2492, 0x8421]:
            for seed in range(20):
                assert walk(kind, bf16, tokens, total, slow, seed) == 0, (total, slow, seed)
