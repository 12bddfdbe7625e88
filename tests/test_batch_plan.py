"""Host side of the operators of a step of several requests (csrc/batch_plan.hpp, plain host code, compiled here): what the
entry points refuse, and how the attention is cut into pieces -- no GPU."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from managedllama2_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "managedllama2_amd", "csrc")
SOURCE = """
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include "llama2_hip.h"
static char message[512];
namespace l2 {
inline int ceil_div(int a, int b) { return (a + b - 1) / b; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool overlap(const void* a, size_t na, const void* b, size_t nb)
{
    auto pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    return pa < pb + nb && pb < pa + na;
}
inline int fail(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(message, sizeof(message), fmt, ap);
    va_end(ap);
    return code;
}
}
#define L2_CHECK(cond, ...) do { if (!(cond)) return ::l2::fail(LLAMA2_ERR_INVALID_ARGUMENT, __VA_ARGS__); } while (0)
#include "batch_plan.hpp"
extern "C" {
const char* last() { return message; }
int tables(const llama2_batch* b, const int* cached, const int* counts, const int* free_blocks, int n_free, const int* taken,
           int* new_taken, int block_size)
{
    return l2::check_batch_tables(b, cached, counts, free_blocks, n_free, taken, new_taken, block_size);
}
int rope(const llama2_half* o, const llama2_half* q, const llama2_half* k, const llama2_half* v, const llama2_half* gq,
         const llama2_half* gk, const llama2_batch* b, const llama2_paged_cache* c, int h, int so, int sq, int skv, float eps, float theta)
{
    return l2::check_batch_rope(o, q, k, v, gq, gk, b, c, h, so, sq, skv, eps, theta);
}
int attention(const llama2_half* o, const llama2_half* q, const llama2_batch* b, const llama2_paged_cache* c, int h, int so, int sq,
              float scale)
{
    return l2::check_batch_attention(o, q, b, c, h, so, sq, scale);
}
int fits(const llama2_batch* b, int n_kv_heads, int group, int max_rows)
{
    return l2::check_batch_attn_plan(l2::batch_attn_plan(*b, n_kv_heads, group, max_rows, 256), b->n_tokens, n_kv_heads * group, n_kv_heads);
}
unsigned divide(unsigned n, int d) // as a kernel does
{
    const l2::Divisor by = l2::divisor(d);
    return static_cast<unsigned>((static_cast<unsigned long long>(2 * n) * by.m) >> 32) >> by.shift;
}
void plan(const llama2_batch* b, int n_kv_heads, int group, int max_rows, int* out)
{
    const l2::BatchAttnPlan p = l2::batch_attn_plan(*b, n_kv_heads, group, max_rows, 256);
    out[0] = static_cast<int>(p.kernel), out[1] = p.shared_tiles, out[2] = p.shared_splits, out[3] = p.shared_piece;
    out[4] = p.own_tiles, out[5] = p.own_splits, out[6] = p.own_piece, out[7] = p.own_prefix;
}
}
"""

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
MIB = 1 << 20
INVALID, UNSUPPORTED = capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("plan")
    (out / "plan.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-I",
                           os.path.join(ROOT, "include"), str(out / "plan.cpp"), "-o", str(out / "plan.so")])
    lib = C.CDLL(str(out / "plan.so"))
    for ours, name in (("tables", "llama2_batch_tables"), ("rope", "llama2_batch_qk_norm_rope"), ("attention", "llama2_batch_attention")):
        getattr(lib, ours).argtypes = capi._SIGNATURES[name]
    lib.plan.argtypes = [C.POINTER(capi.Batch), C.c_int, C.c_int, C.c_int, C.POINTER(C.c_int)]
    lib.fits.argtypes = [C.POINTER(capi.Batch), C.c_int, C.c_int, C.c_int]
    lib.last.restype = C.c_char_p
    return lib


def batch(**other):  # addresses are only compared, never followed
    f = dict(block_tables=1 * MIB, lengths=2 * MIB, query_starts=3 * MIB, positions=4 * MIB, slots=5 * MIB, prefix_table=6 * MIB,
             n_requests=4, n_tokens=9, table_stride=10, prefix_length=20, max_length=160)
    f.update(other)
    return capi.Batch(**f)


def cache(**other):
    f = dict(key=100 * MIB, value=200 * MIB, block_stride=0, n_blocks=50, block_size=16, n_kv_heads=2, head_size=128)
    f.update(other)
    return capi.PagedCache(**f)


def test_structs_are_laid_out_as_in_the_header(lib, tmp_path):
    (tmp_path / "size.c").write_text('#include "llama2_hip.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){printf("%zu %zu '
                                     '%zu %zu", sizeof(llama2_batch), sizeof(llama2_paged_cache), offsetof(llama2_batch, max_length), '
                                     'offsetof(llama2_paged_cache, head_size)); return 0;}')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "size.c"), "-o", str(tmp_path / "size")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "size")]).split()]
    assert got == [C.sizeof(capi.Batch), C.sizeof(capi.PagedCache), capi.Batch.max_length.offset, capi.PagedCache.head_size.offset]


TABLES = dict(cached=10 * MIB, counts=11 * MIB, free_blocks=12 * MIB, n_free=7, taken=13 * MIB, new_taken=14 * MIB, block_size=16)


def call_tables(lib, b, **other):
    a = dict(TABLES, **other)
    return lib.tables(b, a["cached"], a["counts"], a["free_blocks"], a["n_free"], a["taken"], a["new_taken"], a["block_size"])


def test_tables_refusals(lib):
    assert call_tables(lib, batch()) == 0
    assert call_tables(lib, batch(prefix_table=None, max_length=0)) == 0  # neither is read
    assert call_tables(lib, batch(), free_blocks=None, n_free=0) == 0
    assert call_tables(lib, batch(lengths=10 * MIB), new_taken=13 * MIB) == 0  # in place
    for name in ("block_tables", "lengths", "query_starts", "positions", "slots"):
        assert call_tables(lib, batch(**{name: None})) == INVALID, name
        assert call_tables(lib, batch(**{name: getattr(batch(), name) + 2})) == INVALID, name
    for name in ("cached", "counts", "free_blocks", "taken", "new_taken"):
        assert call_tables(lib, batch(), **{name: None}) == INVALID, name
        assert call_tables(lib, batch(), **{name: TABLES[name] + 1}) == INVALID, name
    for name, values in dict(n_requests=(0, -1, (1 << 20) + 1), n_tokens=(0, -5, (1 << 20) + 1), prefix_length=(-1,),
                             table_stride=(0, -1, 0x7FFFFFFF // 16)).items():
        for v in values:
            assert call_tables(lib, batch(**{name: v})) == INVALID, (name, v)
    for v in (0, 4, 7, 12, 24, 2048, -16):
        assert call_tables(lib, batch(), block_size=v) == INVALID, v
        assert b"block_size" in lib.last()
    assert call_tables(lib, batch(), n_free=-1) == INVALID
    assert lib.tables(None, *TABLES.values()) == INVALID
    # overlaps: outputs with each other, outputs with inputs (but for the two that may be updated in place)
    assert call_tables(lib, batch(slots=4 * MIB + 8 * 4)) == INVALID
    assert call_tables(lib, batch(positions=12 * MIB + 24)) == INVALID
    assert call_tables(lib, batch(lengths=11 * MIB)) == INVALID
    assert call_tables(lib, batch(lengths=10 * MIB + 4)) == INVALID
    assert call_tables(lib, batch(), new_taken=10 * MIB + 12) == INVALID
    assert call_tables(lib, batch(block_tables=12 * MIB - 4 * 10 * 4 + 4)) == INVALID


ROPE = dict(o=300 * MIB, q=310 * MIB, k=320 * MIB, v=330 * MIB, gq=340 * MIB, gk=341 * MIB, heads=8, so=1024, sq=1024, skv=256, eps=1e-5,
            theta=1e4)


def call_rope(lib, b, c, **other):
    a = dict(ROPE, **other)
    return lib.rope(a["o"], a["q"], a["k"], a["v"], a["gq"], a["gk"], b, c, a["heads"], a["so"], a["sq"], a["skv"], a["eps"], a["theta"])


def test_rope_refusals(lib):
    assert call_rope(lib, batch(), cache()) == 0
    assert call_rope(lib, batch(block_tables=None, query_starts=None, lengths=None), cache(), gq=None, gk=None) == 0
    fused = dict(q=310 * MIB, k=310 * MIB + 2048, v=310 * MIB + 2560, sq=1536, skv=1536)
    assert call_rope(lib, batch(), cache(), **fused) == 0
    assert call_rope(lib, batch(), cache(), **dict(fused, o=310 * MIB, so=1536)) == 0  # in place
    assert call_rope(lib, batch(), cache(), **dict(fused, o=310 * MIB, so=1024)) == INVALID
    assert call_rope(lib, batch(), cache(), **dict(fused, o=310 * MIB + 2048, so=1536)) == INVALID
    # in place, rows of k and v only between those of q: 1024 of q, 256 of k, 256 of v in 1536
    place = dict(fused, o=310 * MIB, so=1536)
    for name in ("k", "v"):
        for at in (0, 16, 2048 - 16, 2560 + 16, 2 * 1536 * 8, -16):
            assert call_rope(lib, batch(), cache(), **dict(place, **{name: 310 * MIB + at})) == INVALID, (name, at)
        for at in (2048, 2560, 2048 + 2 * 1536 * 8, -512, -1024):  # of the same row, of the last one, in front
            assert call_rope(lib, batch(), cache(), **dict(place, **{name: 310 * MIB + at})) == 0, (name, at)
        assert call_rope(lib, batch(), cache(), **dict(place, skv=1528)) == INVALID
    for name in ("o", "q", "k", "v"):
        assert call_rope(lib, batch(), cache(), **{name: None}) == INVALID, name
    for name in ("o", "q", "k", "v", "gq", "gk"):
        assert call_rope(lib, batch(), cache(), **{name: ROPE[name] + 8}) == INVALID, name
    for name in ("positions", "slots"):
        assert call_rope(lib, batch(**{name: None}), cache()) == INVALID, name
    for name in ("so", "sq", "skv"):
        assert call_rope(lib, batch(), cache(), **{name: ROPE[name] - 8}) == INVALID, name
        assert call_rope(lib, batch(), cache(), **{name: ROPE[name] + 4}) == INVALID, name
    for v in (0.5, 0.0, -1.0, float("nan"), float("inf")):
        assert call_rope(lib, batch(), cache(), theta=v) == INVALID, v
    for v in (-1e-6, float("nan"), float("inf")):
        assert call_rope(lib, batch(), cache(), eps=v) == INVALID, v
    for name in ("o", "q", "k", "v"):  # inside the cache
        assert call_rope(lib, batch(), cache(), **{name: 100 * MIB + 4096}) == INVALID, name
    assert call_rope(lib, None, cache()) == INVALID and call_rope(lib, batch(), None) == INVALID


def test_rope_refuses_keys_over_values(lib):
    block = 16 * 256  # halfs of a block, 2 bytes each; 50 blocks
    for at in (0, 16, 2 * block - 16, 2 * block, 50 * 2 * block - 16):
        assert call_rope(lib, batch(), cache(value=100 * MIB + at)) == INVALID, at
        assert call_rope(lib, batch(), cache(key=200 * MIB + at, value=200 * MIB)) == INVALID, at
    assert call_rope(lib, batch(), cache(value=100 * MIB + 50 * 2 * block)) == 0
    turns = dict(block_stride=2 * block)  # blocks of keys and values in turn
    for at, want in ((2 * block, 0), (2 * block - 16, INVALID), (2 * block + 16, INVALID), (6 * block, 0), (4 * block, INVALID),
                     (49 * 4 * block + 2 * block + 16, 0), (49 * 4 * block + 2 * block - 16, INVALID)):
        assert call_rope(lib, batch(), cache(value=100 * MIB + at, **turns)) == want, at
        assert call_rope(lib, batch(), cache(key=200 * MIB + at, value=200 * MIB, **turns)) == want, at
    one = cache(n_blocks=1, value=100 * MIB + 2 * block - 16, block_stride=2 * block)
    assert call_rope(lib, batch(), one) == INVALID
    assert call_rope(lib, batch(), cache(n_blocks=1, value=100 * MIB + 2 * block + 16, block_stride=2 * block)) == 0
    assert call_attention(lib, batch(), cache(value=100 * MIB)) == 0  # which only reads them


def test_cache_refusals(lib):
    for call in (call_rope, call_attention):
        for v in (0, 32, 96, 100, 256):
            assert call(lib, batch(), cache(head_size=v)) == UNSUPPORTED, v
        for v in (0, 4, 12, 2048):
            assert call(lib, batch(), cache(block_size=v)) == INVALID, v
        for v in (0, -1, 0x7FFFFFFF // 16 + 1):
            assert call(lib, batch(), cache(n_blocks=v)) == INVALID, v
        for v in (0, 3, 16, -2):
            assert call(lib, batch(), cache(n_kv_heads=v)) == INVALID, v
        for v in (16 * 256 - 8, 16 * 256 + 4, -8, 1 << 50):
            assert call(lib, batch(), cache(block_stride=v)) == INVALID, v
        assert call(lib, batch(), cache(block_stride=16 * 256 + 8)) == 0
        for name in ("key", "value"):
            assert call(lib, batch(), cache(**{name: None})) == INVALID
            assert call(lib, batch(), cache(**{name: 100 * MIB + 8})) == INVALID
        assert call(lib, batch(), cache(n_kv_heads=2), heads=2048, so=262144, sq=262144) == UNSUPPORTED


ATTENTION = dict(o=300 * MIB, q=310 * MIB, heads=8, so=1024, sq=1024, scale=0.1)


def call_attention(lib, b, c, **other):
    a = dict(ATTENTION, **other)
    return lib.attention(a["o"], a["q"], b, c, a["heads"], a["so"], a["sq"], a["scale"])


def test_attention_refusals(lib):
    assert call_attention(lib, batch(), cache()) == 0
    assert call_attention(lib, batch(slots=None, lengths=None), cache()) == 0
    assert call_attention(lib, batch(prefix_table=None, prefix_length=0), cache()) == 0
    assert call_attention(lib, batch(prefix_table=None), cache()) == INVALID
    for name in ("block_tables", "query_starts", "positions"):
        assert call_attention(lib, batch(**{name: None}), cache()) == INVALID, name
    for name, values in dict(n_requests=(0, (1 << 20) + 1), n_tokens=(0, (1 << 20) + 1), prefix_length=(-1,), table_stride=(0,),
                             max_length=(0, -1)).items():
        for v in values:
            assert call_attention(lib, batch(**{name: v}), cache()) == INVALID, (name, v)
    assert call_attention(lib, batch(max_length=0x7FFFFFFF), cache()) == 0  # no more than the tables hold
    assert call_attention(lib, batch(max_length=0x7FFFFFFF, table_stride=1 << 25), cache()) == UNSUPPORTED
    assert call_attention(lib, batch(prefix_length=(1 << 29) - 100), cache()) == UNSUPPORTED
    for name in ("o", "q"):
        assert call_attention(lib, batch(), cache(), **{name: None}) == INVALID
        assert call_attention(lib, batch(), cache(), **{name: ATTENTION[name] + 2}) == INVALID
    for name in ("so", "sq"):
        for v in (1016, 1028):
            assert call_attention(lib, batch(), cache(), **{name: v}) == INVALID
    assert call_attention(lib, batch(), cache(), o=310 * MIB + 9 * 2048 - 16) == INVALID
    assert call_attention(lib, batch(), cache(), o=310 * MIB) == INVALID
    assert call_attention(lib, batch(), cache(), o=200 * MIB + 64) == INVALID
    for v in (float("nan"), float("inf"), -float("inf")):
        assert call_attention(lib, batch(), cache(), scale=v) == INVALID


def around(rows, width, n, stride):
    """(offsets at which an array of 36 bytes touches one of n rows, offsets at which it does not)"""
    last = (n - 1) * stride
    hits = {0, 4, width - 4, -32, last, last + width - 4, stride - 32, stride, last - 32}
    misses = {-36, last + width, last + stride, last + 2 * stride}
    if stride > width + 36:
        misses |= {width, stride - 36, last - 36}
    return [rows + x for x in hits], [rows + x for x in misses]


def test_what_is_written_may_not_lie_over_what_is_read(lib):
    """9 positions, slots or entries (36 bytes), in front of, behind and between rows of outputs and blocks of the cache."""
    for stride in (1024, 1032, 1536):
        hits, misses = around(300 * MIB, 2048, 9, 2 * stride)
        for name in ("positions", "slots"):
            assert all(call_rope(lib, batch(**{name: x}), cache(), so=stride) == INVALID for x in hits), (stride, name)
            assert all(call_rope(lib, batch(**{name: x}), cache(), so=stride) == 0 for x in misses), (stride, name)
        one = dict(n_requests=8, table_stride=1, max_length=9)  # 9 starts, 8 entries
        for name in ("positions", "query_starts"):
            assert all(call_attention(lib, batch(**{name: x}, **one), cache(), so=stride) == INVALID for x in hits), (stride, name)
            assert all(call_attention(lib, batch(**{name: x}, **one), cache(), so=stride) == 0 for x in misses), (stride, name)
        for name, more in (("block_tables", dict(n_requests=9, table_stride=1)), ("block_tables", dict(n_requests=3, table_stride=3)),
                           ("prefix_table", dict(prefix_length=8 * 16 + 1))):
            assert all(call_attention(lib, batch(**{name: x}, **more), cache(), so=stride) == INVALID for x in hits), (stride, name)
            assert all(call_attention(lib, batch(**{name: x}, **more), cache(), so=stride) == 0 for x in misses), (stride, name)
        for name in ("gq", "gk"):
            assert call_rope(lib, batch(), cache(), **{name: 300 * MIB + 2032}, so=stride) == INVALID
            assert call_rope(lib, batch(), cache(), **{name: 300 * MIB - 240}, so=stride) == INVALID
            assert call_rope(lib, batch(), cache(), **{name: 300 * MIB - 256}, so=stride) == 0
    assert call_rope(lib, batch(), cache(), gq=300 * MIB + 2048, so=1536) == 0  # 256 bytes between two rows
    block = 16 * 256 * 2  # bytes
    for base, which in ((100 * MIB, "keys"), (200 * MIB, "values")):
        for stride in (block, block + 80, 3 * block):
            hits, misses = around(base, block, 50, stride)
            for name in ("positions", "slots"):
                assert all(call_rope(lib, batch(**{name: x}), cache(block_stride=stride // 2)) == INVALID for x in hits), (which, stride)
                assert all(call_rope(lib, batch(**{name: x}), cache(block_stride=stride // 2)) == 0 for x in misses), (which, stride)
            for name in ("gq", "gk"):
                assert call_rope(lib, batch(), cache(block_stride=stride // 2), **{name: base + 49 * stride + block - 16}) == INVALID
                assert call_rope(lib, batch(), cache(block_stride=stride // 2), **{name: base + 49 * stride + block}) == 0
    assert call_attention(lib, batch(prefix_table=300 * MIB, prefix_length=0), cache()) == 0  # not read


SIZES = (1, 2, 15, 16, 17, 63, 64, 65, 255, 257, 1000, 4096, 131072, 3000001)


@pytest.mark.parametrize("requests", [1, 2, 3, 7, 64, 1000])
def test_plan_covers_every_row_and_column(lib, requests):
    """Pieces of whole passes that hold all rows, not more of them than there is room for, and tiles for all columns."""
    out = (C.c_int * 8)()
    for kv_heads, group in ((1, 1), (8, 4), (40, 1), (1, 130), (2, 8)):
        for per in (1, 3, 40, 700):
            tokens = requests * per
            for prefix in (0,) + SIZES:
                for rows in SIZES:
                    b = batch(n_requests=requests, n_tokens=tokens, prefix_length=prefix)
                    lib.plan(b, kv_heads, group, rows, out)
                    kernel, tiles, splits, piece, own_tiles, own_splits, own_piece, own_prefix = out
                    what = (requests, kv_heads, group, per, prefix, rows, list(out))
                    tile = 128 if kernel >= 2 else 16
                    assert kernel != 3 or (splits == 0 and own_piece >= 256 and own_tiles * own_splits * kv_heads <= 256), what
                    assert kernel != 1 or (splits == 0 and own_splits == 1), what  # a wavefront per tile: no pieces
                    assert own_piece % 64 == 0 and own_piece > 0 and 1 <= own_splits <= 256, what
                    assert own_splits * own_piece >= own_prefix + rows > (own_splits - 1) * own_piece, what
                    assert own_tiles >= tokens * group // tile + requests, what
                    if splits:
                        assert own_prefix == 0 and prefix > 0 and piece % 64 == 0 and splits <= 256, what
                        assert splits * piece >= prefix > (splits - 1) * piece, what
                        assert (tiles - 1) * tile < tokens * group <= tiles * tile, what
                    else:
                        assert own_prefix == -(-prefix // 64) * 64 and tiles == 0, what


def test_plan_shares_a_prefix_among_narrow_requests_only(lib):
    out = (C.c_int * 8)()
    lib.plan(batch(n_requests=16, n_tokens=16, prefix_length=2048), 32, 1, 256, out)
    assert out[2] > 0 and out[7] == 0 and out[0] == 0
    lib.plan(batch(n_requests=8, n_tokens=4000, prefix_length=512), 32, 1, 1500, out)
    assert out[2] == 0 and out[7] == 512 and out[0] == 2 and out[5] == 1
    lib.plan(batch(n_requests=1, n_tokens=1, prefix_length=512), 32, 1, 300, out)  # nobody to share with
    assert out[2] == 0 and out[7] == 512 and out[0] == 0
    lib.plan(batch(n_requests=100, n_tokens=100, prefix_length=10), 32, 1, 54, out)
    assert out[0] == 1 and out[7] == 64
    lib.plan(batch(n_requests=5, n_tokens=1200, prefix_length=134), 8, 1, 609, out)  # fewer tiles than compute units
    assert out[0] == 3 and out[5] == 1
    lib.plan(batch(n_requests=5, n_tokens=1200, prefix_length=0), 8, 1, 192, out)  # and few passes
    assert out[0] == 2 and out[5] == 1


@pytest.mark.parametrize("requests", [1, 2, 7, 64, 256, 4000])
def test_plan_needs_a_bounded_scratch(lib, requests):
    """Sums, maximum and denominator of every piece of every query row: half a GiB at most, whatever the bounds of a call are."""
    out = (C.c_int * 8)()
    most = 0
    for kv_heads, group in ((1, 1), (8, 4), (32, 1), (40, 1), (8, 8)):
        for tokens in (requests, requests * 3 + 1, requests * 62, requests * 63 // group, 1 << 20):
            if requests <= tokens <= 1 << 20 and tokens * kv_heads * group < 1 << 26:
                for prefix in (0, 100, 5000, 1 << 28):
                    for rows in (1, 100, 4096, 131072, 1 << 28):
                        lib.plan(batch(n_requests=requests, n_tokens=tokens, prefix_length=prefix), kv_heads, group, rows, out)
                        slots = out[2] + out[5]
                        scratch = slots * tokens * kv_heads * group * 130 * 4 if slots > 1 else 0
                        assert scratch <= 1 << 29, (kv_heads, group, tokens, prefix, rows, list(out))
                        most = max(most, scratch)
    assert most > 0


def test_division_by_a_product(lib):
    top = (1 << 31) - 1
    lib.divide.restype = C.c_uint
    for d in list(range(1, 70)) + [127, 128, 129, 255, 641, 1023, 1024, 1040, 65535, 65537, 1 << 20, (1 << 20) + 1, (1 << 24) - 1, 1 << 24, top - 1, top]:
        near = {n for k in (1, 2, 3, 7, 1000, top // d // 2, top // d - 1, top // d) for n in (k * d - 1, k * d, k * d + 1)}
        for n in near | {0, 1, top, top - 1, 12345678}:
            if 0 <= n <= top:
                assert lib.divide(n, d) == n // d, (n, d)


def test_plan_refuses_more_workgroups_than_a_launch_holds(lib):
    assert lib.fits(batch(n_requests=100000, n_tokens=100000), 32, 1, 4000) == 0
    assert lib.fits(batch(n_requests=1 << 20, n_tokens=1 << 20), 32, 1, 4000) == UNSUPPORTED
    assert lib.fits(batch(n_requests=1, n_tokens=1 << 20), 1, 128, 4000) == UNSUPPORTED
    assert lib.fits(batch(n_requests=1, n_tokens=1 << 20), 8, 4, 1 << 20) == 0
    assert b"too many" in lib.last()


def test_entry_points_refuse_before_init():
    import sys
    code = ("import sys; sys.path.insert(0, %r)\nfrom managedllama2_amd import capi\nb, c = capi.Batch(), capi.PagedCache()\n"
            "assert capi.raw('llama2_batch_tables', b, None, None, None, 0, None, None, 16) == capi.ERR_NOT_INITIALIZED\n"
            "assert capi.raw('llama2_batch_qk_norm_rope', None, None, None, None, None, None, b, c, 1, 1, 1, 1, 0.0, 1.0) == "
            "capi.ERR_NOT_INITIALIZED\n"
            "assert capi.raw('llama2_batch_attention', None, None, b, c, 1, 1, 1, 1.0) == capi.ERR_NOT_INITIALIZED\nprint('ok')" % ROOT)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "ok" in out.stdout, out.stderr
