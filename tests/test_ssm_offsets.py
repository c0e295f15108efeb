"""Offsets that the chunked scan forms (pe_ranges.h, the header that it includes,
built here for the CPU) at the widest token strides that it takes."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "pto-einsum_amd", "csrc")


@pytest.fixture(scope="module")
def ranges(tmp_path_factory):
    d = tmp_path_factory.mktemp("offsets")
    src, lib = d / "offsets.cpp", d / "liboffsets.so"
    src.write_text('#include "pe_ranges.h"\nextern "C" {\n'
                   "int64_t step_offset(int i, int stride) { return pe::step_offset(i, stride); }\n"
                   "int64_t stride_end() { return pe::kScanStrideEnd; }\n}\n")
    # -fwrapv: 32-bit products wrap, as they do on the GPU.
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o", str(lib)],
                   check=True)
    lib = ctypes.CDLL(str(lib))
    lib.step_offset.restype = lib.stride_end.restype = ctypes.c_int64
    return lib


@pytest.mark.parametrize("i", [0, 127, 128, 255, 383])
def test_step_sizes_lie_where_their_tokens_do(ranges, i):
    end = ranges.stride_end()
    for stride in (1, 5592405, 5700000, 8388608, 9000001, end - 1):
        assert ranges.step_offset(i, stride) == i * stride


def test_rows_of_a_chunk_lie_within_32_bits(ranges):
    """64 rows of two bytes an element or 32 of four, eight elements before and 256
    after each row's start."""
    end = ranges.stride_end()
    assert (63 * (end - 1) + 256 + 16) * 2 < 2 ** 32 and (31 * (end - 1) + 256 + 16) * 4 < 2 ** 32
    assert 63 * (end - 1) + 256 + 16 < 2 ** 31
