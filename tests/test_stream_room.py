"""csrc/stream_room.h on the CPU: what a stream owns where device memory is short.  The attention's 32 MiB never cost the GEMMs
their 16."""
import ctypes
import os
import shutil
import subprocess

import pytest

from helpers import ROOT

DRIVER = """
#include "stream_room.h"
#include <set>
using namespace mi;
// `most`: bytes that an allocation may have, `all`: that they may have together; out: bytes of the workspace and of the sums that the stream
// has, bytes allocated and not released, allocations asked for
extern "C" void room(long long most, long long all, int clears, long long* out) {
    static char memory[4];
    long long used = 0, sizes[4] = {}, asked = 0;
    const StreamRoom r = make_stream_room(
        [&](size_t bytes) -> void* {
            const long long n = static_cast<long long>(bytes);
            if (n > most || used + n > all) return nullptr;
            used += n;
            sizes[asked] = n;
            return memory + asked++;
        },
        [&](void* p) { return p && clears; }, [&](void* p) { used -= sizes[static_cast<char*>(p) - memory]; });
    out[0] = r.workspace ? sizes[static_cast<char*>(r.workspace) - memory] : 0;
    out[1] = r.sums ? sizes[static_cast<char*>(r.sums) - memory] : 0;
    out[2] = used;
    out[3] = asked;
}
"""
GEMM, SUMS = (16 << 20) + 16384 * 4, 32 << 20


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_what_a_stream_owns(tmp_path):
    src, so = tmp_path / "room.cpp", str(tmp_path / "room.so")
    src.write_text(DRIVER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "adreno-llms_amd", "csrc"), "-o", so, str(src)])
    lib = ctypes.CDLL(so)

    def room(most, everything, clears=1):
        out = (ctypes.c_longlong * 4)()
        lib.room(ctypes.c_longlong(most), ctypes.c_longlong(everything), clears, out)
        return list(out)[:3]

    assert room(1 << 40, 1 << 40) == [GEMM, SUMS, GEMM + SUMS]
    assert room(1 << 40, GEMM + SUMS - 1) == [GEMM, 0, GEMM]               # short of the second alone
    assert room(SUMS - 1, 1 << 40) == [GEMM, 0, GEMM]
    assert room(GEMM - 1, 1 << 40) == [0, 0, 0] and room(0, 0) == [0, 0, 0]
    assert room(1 << 40, 1 << 40, clears=0) == [0, 0, 0]                   # and nothing is left behind
