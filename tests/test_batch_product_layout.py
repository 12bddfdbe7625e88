"""Where the products of many tokens put what they read 16 bytes at a time: items and turn buffers in LDS, and what the adapters' ranks receive in the
library's scratch -- compiled here, no GPU."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import test_batch_plan as tp
from test_build_resources import CSRC, HIPCC

LDS = """
#include "%s/prefill.hip"
namespace l2 {
static_assert(sizeof(Items) %% 16 == 0, "items stand behind each other");
static_assert(offsetof(Items, tokens) %% 16 == 0, "an item's tokens are stored as 16 bytes");
template <int MT, int WN>
constexpr bool turn_buffers_are_aligned()
{
    using Lds = GemmLds<MT, WN, 4 / WN>;
    static_assert(Lds::kRed %% 16 == 0 && Lds::kTurnAt %% 16 == 0, "16 bytes of LDS at a time");
    static_assert(Lds::kTurnAt >= Lds::kRed + MT * static_cast<int>(sizeof(Items)) && Lds::kRowsBytes >= Lds::kTurnAt + 8 * 1024, "apart");
    return true;
}
static_assert(turn_buffers_are_aligned<1, 4>() && turn_buffers_are_aligned<2, 4>() && turn_buffers_are_aligned<3, 4>() &&
              turn_buffers_are_aligned<4, 4>() && turn_buffers_are_aligned<1, 2>() && turn_buffers_are_aligned<2, 2>() &&
              turn_buffers_are_aligned<1, 1>());
} // namespace l2
"""


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="hipcc not found")
def test_lds_that_is_read_16_bytes_at_a_time(tmp_path):
    (tmp_path / "lds.hip").write_text(LDS % CSRC)
    out = subprocess.run([HIPCC, "--offload-arch=gfx950", "-std=c++17", "--cuda-host-only", "-fsyntax-only", "-I", CSRC, str(tmp_path / "lds.hip")],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-3000:]


SCRATCH = tp.SOURCE.split('#include "batch_plan.hpp"')[0] + """
#include "batch_product_plan.hpp"
extern "C" int scratch(size_t operands, int tokens, const int* ranks, int n, size_t* out)
{
    const l2::LowScratch s = l2::low_scratch(operands, tokens, ranks, n);
    for (int i = 0; i < n; ++i)
        out[2 * i] = s.low[i], out[2 * i + 1] = s.info[i];
    out[8] = s.bytes;
    return sizeof(l2::TokenAdapter);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_what_the_ranks_receive_lies_on_its_multiples(tmp_path):
    """Odd numbers of tokens, of one and of several tensors with adapters and without: 64 bytes of 16 ranks are one piece, and no two
    tensors' overlap."""
    (tmp_path / "scratch.cpp").write_text(SCRATCH)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-Wno-unused-function", "-shared", "-fPIC", "-I", CSRC, "-I",
                           os.path.join(tp.ROOT, "include"), str(tmp_path / "scratch.cpp"), "-o", str(tmp_path / "scratch.so")])
    lib = C.CDLL(str(tmp_path / "scratch.so"))
    lib.scratch.argtypes = [C.c_size_t, C.c_int, C.POINTER(C.c_int), C.c_int, C.POINTER(C.c_size_t)]
    out = (C.c_size_t * 9)()
    for operands in (0, 4096, 5 * 8192):
        for tokens in (1, 3, 33, 48, 49, 101, 4095, 4096):
            for ranks in ([16], [0], [8, 16, 16], [16, 0, 64], [128, 8, 0, 24], [0, 0, 0, 0], [40, 40]):
                info = lib.scratch(operands, tokens, (C.c_int * len(ranks))(*ranks), len(ranks), out)
                assert info == 8
                pieces = []
                for i, r in enumerate(ranks):
                    blocks = tokens * -(-r // 16)
                    assert out[2 * i] % 64 == 0 and out[2 * i + 1] % info == 0, (operands, tokens, ranks, i)
                    pieces += [(out[2 * i], blocks * 64), (out[2 * i + 1], blocks * info)]
                at = operands
                for start, size in sorted(p for p in pieces if p[1]):
                    assert start == at, (operands, tokens, ranks)
                    at += size
                assert at == out[8]
