"""The counter that the CTAs of a divided item share (plugins_b200/csrc/exl3_parts.h), compiled for the host: whoever gives up, the
last part finds all arrived, and the item is written by none unless every part brought its own."""
import ctypes
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = r"""
#include "exl3_parts.h"
extern "C" uint32_t arrival(int brought) { return exl3::part_arrival(brought != 0); }
extern "C" int arrived(uint32_t n, int parts) { return exl3::parts_arrived(n, parts); }
extern "C" int whole(uint32_t n) { return exl3::parts_whole(n); }
extern "C" int most() { return exl3::kMaxParts; }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("parts")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "plugins_b200", "csrc"),
                           str(d / "shim.cpp"), "-o", str(d / "shim.so")])
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.arrival.restype = ctypes.c_uint32
    lib.arrived.argtypes, lib.whole.argtypes = [ctypes.c_uint32, ctypes.c_int], [ctypes.c_uint32]
    return lib


def arrive(lib, brought):
    """Parts arriving one after another -> (which of them was last, whether it writes)."""
    counter, last = 0, []
    for i, b in enumerate(brought):
        counter += lib.arrival(int(b))
        assert counter < 2 ** 32
        if lib.arrived(counter, len(brought)):
            last.append((i, bool(lib.whole(counter))))
            counter = 0
    assert counter == 0  # as the next launch expects it
    return last


@pytest.mark.parametrize("parts", range(1, 9))
def test_the_last_part_writes_what_all_have_brought(lib, parts):
    for brought in itertools.product((True, False), repeat=parts):
        assert arrive(lib, brought) == [(parts - 1, all(brought))]


def test_as_many_parts_as_a_grid_has(lib):
    for parts in (148, lib.most()):
        for brought in ([True] * parts, [False] * parts, [True] * (parts - 1) + [False], [False] + [True] * (parts - 1)):
            assert arrive(lib, brought) == [(parts - 1, all(brought))]
