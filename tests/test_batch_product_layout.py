"""Where the products of many tokens put what they read 16 bytes at a time: items and turn buffers in LDS, and what the adapters' ranks receive in the
library's scratch -- compiled here, no GPU."""
import os
import shutil
import subprocess

import pytest

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
