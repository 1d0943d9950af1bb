"""Index arithmetic of the attention kernels (zillaphp_b200/csrc/kv_attend.cuh), compiled for the host and called on the CPU at
values that no GPU run should be given."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from zillaphp_b200 import build

SOURCE = """
#include "kv_attend.cuh"
extern "C" int noted_slots(int note, int splits) { return zb::kv::noted_slots(note, splits); }
extern "C" int slots_of(int keys, int chunk) { return zb::kv::slots_of(keys, chunk); }
extern "C" int slot_end(int begin, int chunk, int len) { return zb::kv::slot_end(begin, chunk, len); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_plan")
    (d / "plan.cu").write_text(SOURCE)
    subprocess.run([build._nvcc(), *build.ARCH, *build.NVCC_FLAGS, "-I" + build.CSRC, "-shared", str(d / "plan.cu"), "-o", str(d / "plan.so")],
                   check=True, capture_output=True)
    return C.CDLL(str(d / "plan.so"))


def test_slots_of_an_item_that_was_not_noted(lib):
    """A kernel whose wait ran out leaves the word as it was: the join stays within the prefix's slots, and keeps every note."""
    nan = int(np.full(1, np.nan, np.float32).view(np.int32)[0])
    for splits in (1, 2, 7, 148):
        assert [lib.noted_slots(n, splits) for n in range(splits + 1)] == list(range(splits + 1))
        for junk in (splits + 1, nan, 2 ** 31 - 1, -1, -2 ** 31, int(np.float32(-1.5).view(np.int32))):
            assert 0 <= lib.noted_slots(junk, splits) <= splits, junk


def test_slots_near_31_bits(lib):
    """Slots that cover the keys, each once, also where a slot's end or keys + chunk pass 31 bits."""
    for len_ in (0, 1, 63, 64, 65, 1000, 2 ** 30, 2 ** 31 - 5000, 2 ** 31 - 4097):
        for chunk in (64, 256, 64 * 201_000, 64 * 25_800_000, 64 * ((2 ** 31 - 4097 + 63) // 64)):
            n = lib.slots_of(len_, chunk)
            assert n == -(-len_ // chunk)
            for slot in {0, 1, n // 2, max(0, n - 2), max(0, n - 1)}:
                begin = slot * chunk
                if slot < max(n, 1):
                    assert lib.slot_end(begin, chunk, len_) == min(begin + chunk, len_)
            # a row that sees fewer keys than the sequence has: its slots end with its keys
            assert lib.slot_end(64, chunk, 10) == 10
