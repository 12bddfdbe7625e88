"""Host side of the products, norms and log probabilities of a step of several requests (csrc/batch_product_plan.hpp, plain host
code, compiled here): what the entry points refuse -- no GPU."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import test_batch_plan as tp
from managedllama2_amd import capi

ROOT, CSRC = tp.ROOT, tp.CSRC
SOURCE = tp.SOURCE.split('#include "batch_plan.hpp"')[0] + """
#include "batch_product_plan.hpp"
extern "C" {
const char* last() { return message; }
int mat_mul(const llama2_batch_matrix* m, int n, const llama2_half* x, int rows, int stride, const int* ids, const llama2_batch* b)
{
    return l2::check_batch_mat_mul(m, n, x, rows, stride, ids, b);
}
int swiglu(llama2_half* o, const llama2_half* x, const llama2_qweight* g, const llama2_qweight* u, int rows, int cols, int so, int sx,
           const llama2_adapters* ga, const llama2_adapters* ua, const int* ids, const llama2_batch* b)
{
    return l2::check_batch_swiglu(o, x, g, u, rows, cols, so, sx, ga, ua, ids, b);
}
int norm(llama2_half* o, llama2_half* ro, const llama2_half* r, const llama2_half* x, const llama2_half* g, const llama2_half* ig,
         const llama2_half* gate, const llama2_batch* b, int size, int so, int sro, int sr, int sx, float scale, float eps)
{
    return l2::check_batch_norm(o, ro, r, x, g, ig, gate, b, size, so, sro, sr, sx, scale, eps);
}
int log_probs(float* lp, float* h, int* top, float* tlp, const llama2_half* x, const int* tokens, const int* positions, int rows, int vocab,
              int stride, int n, int n_top, float temperature)
{
    return l2::check_batch_log_probs(lp, h, top, tlp, x, tokens, positions, rows, vocab, stride, n, n_top, temperature);
}
void shape(int rows, int vocab, int n_top, int cus, int* out)
{
    const l2::LogProbShape s = l2::log_prob_shape(rows, vocab, n_top, cus);
    out[0] = s.segments, out[1] = s.length, out[2] = s.pieces;
}
}
"""
NAMES = {"mat_mul": "llama2_batch_mat_mul_int4", "swiglu": "llama2_batch_mat_mul_swiglu", "norm": "llama2_batch_residual_rmsnorm",
         "log_probs": "llama2_batch_log_probs"}

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
MIB = 1 << 20
INVALID, UNSUPPORTED = capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("product_plan")
    (out / "plan.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-I",
                           os.path.join(ROOT, "include"), str(out / "plan.cpp"), "-o", str(out / "plan.so")])
    lib = C.CDLL(str(out / "plan.so"))
    for ours, name in NAMES.items():
        getattr(lib, ours).argtypes = capi._SIGNATURES[name]
    lib.last.restype = C.c_char_p
    return lib


def test_structs_are_laid_out_as_in_the_header(tmp_path):
    fields = [("llama2_adapters", f[0]) for f in capi.Adapters._fields_] + [("llama2_batch_matrix", f[0]) for f in capi.BatchMatrix._fields_]
    (tmp_path / "size.c").write_text('#include "llama2_hip.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){printf("%zu %zu", '
                                     "sizeof(llama2_adapters), sizeof(llama2_batch_matrix));"
                                     + "".join('printf(" %%zu", offsetof(%s, %s));' % f for f in fields) + "return 0;}")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "size.c"), "-o", str(tmp_path / "size")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "size")]).split()]
    types = {"llama2_adapters": capi.Adapters, "llama2_batch_matrix": capi.BatchMatrix}
    assert got == [C.sizeof(capi.Adapters), C.sizeof(capi.BatchMatrix)] + [getattr(types[t], f).offset for t, f in fields]


def adapters(at=50, **other):
    f = dict(down=at * MIB, up=(at + 10) * MIB, scales=(at + 20) * MIB, ranks=(at + 21) * MIB, n_adapters=4, max_rank=16)
    f.update(other)
    return capi.Adapters(**f)


def matrix(at=100, pool=None, **other):
    f = dict(weight=capi.QWeight(at * MIB, (at + 20) * MIB, (at + 21) * MIB), output=(at + 30) * MIB, residual=None,
             adapters=C.pointer(pool) if pool else None, cols=512, output_stride=512, residual_stride=512)
    f.update(other)
    return capi.BatchMatrix(**f)


def batch(**other):
    return tp.batch(**other)


def call_mat_mul(lib, m=None, n=None, x=7 * MIB, rows=1024, stride=1024, ids=8 * MIB, b=None):
    m = [matrix()] if m is None else m
    a = (capi.BatchMatrix * max(len(m), 1))(*m)
    return lib.mat_mul(a, len(m) if n is None else n, x, rows, stride, ids, batch() if b is None else b)


def call_swiglu(lib, o=30 * MIB, x=7 * MIB, g=(100, 120, 121), u=(200, 220, 221), rows=1024, cols=512, so=512, sx=1024, ga=None, ua=None,
                ids=8 * MIB, b=None):
    q = [capi.QWeight(*(v and v * MIB for v in t)) if t else None for t in (g, u)]
    return lib.swiglu(o, x, q[0], q[1], rows, cols, so, sx, ga, ua, ids, batch() if b is None else b)


def test_products_that_are_allowed(lib):
    assert call_mat_mul(lib) == 0, lib.last()
    assert call_mat_mul(lib, ids=None) == 0
    assert call_mat_mul(lib, [matrix(100, adapters()), matrix(200, adapters(300)), matrix(400)]) == 0, lib.last()
    assert call_mat_mul(lib, [matrix(residual=130 * MIB)]) == 0  # in place
    assert call_mat_mul(lib, [matrix(residual=140 * MIB, residual_stride=1024)]) == 0
    side = [matrix(100, output=500 * MIB, output_stride=1536), matrix(200, output=500 * MIB + 1024, output_stride=1536),
            matrix(300, output=500 * MIB + 2048, output_stride=1536)]
    assert call_mat_mul(lib, side) == 0, lib.last()
    assert call_mat_mul(lib, [matrix(100, adapters(down_stride=4 * 16 * 1024, up_stride=16 * 512 + 8))]) == 0, lib.last()
    assert call_swiglu(lib) == 0, lib.last()
    assert call_swiglu(lib, ga=adapters(), ua=adapters(300)) == 0, lib.last()
    assert call_swiglu(lib, ua=adapters(), so=520) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(m=[], n=0), INVALID), (dict(n=5), INVALID), (dict(n=-1), INVALID), (dict(x=None), INVALID), (dict(x=7 * MIB + 8), INVALID),
    (dict(rows=0), INVALID), (dict(rows=12), INVALID), (dict(rows=-8), INVALID), (dict(rows=1 << 18, stride=1 << 18), UNSUPPORTED),
    (dict(stride=1016), INVALID), (dict(stride=(1 << 24) + 8), UNSUPPORTED), (dict(stride=1028), INVALID), (dict(ids=8 * MIB + 2), INVALID),
    (dict(m=[matrix(output=None)]), INVALID), (dict(m=[matrix(output=130 * MIB + 2)]), INVALID), (dict(m=[matrix(residual=140 * MIB + 4)]), INVALID),
    (dict(m=[matrix(cols=0)]), INVALID), (dict(m=[matrix(cols=12)]), INVALID), (dict(m=[matrix(cols=1 << 21, output_stride=1 << 21)]), UNSUPPORTED),
    (dict(m=[matrix(output_stride=504)]), INVALID), (dict(m=[matrix(output_stride=516)]), INVALID),
    (dict(m=[matrix(residual=140 * MIB, residual_stride=504)]), INVALID),
    (dict(m=[matrix(weight=capi.QWeight(None, 120 * MIB, 121 * MIB))]), INVALID), (dict(m=[matrix(weight=capi.QWeight(100 * MIB, None, 121 * MIB))]), INVALID),
    (dict(m=[matrix(weight=capi.QWeight(100 * MIB + 4, 120 * MIB, 121 * MIB))]), INVALID),
    (dict(m=[matrix(weight=capi.QWeight(100 * MIB, 120 * MIB + 2, 121 * MIB))]), INVALID),
    (dict(m=[matrix(weight=capi.QWeight(100 * MIB, 120 * MIB, 121 * MIB + 1))]), INVALID),
    (dict(m=[matrix(pool=adapters())], ids=None), INVALID), (dict(m=[matrix(pool=adapters(down=None))]), INVALID),
    (dict(m=[matrix(pool=adapters(up=60 * MIB + 8))]), INVALID), (dict(m=[matrix(pool=adapters(ranks=None))]), INVALID),
    (dict(m=[matrix(pool=adapters(scales=71 * MIB + 2))]), INVALID), (dict(m=[matrix(pool=adapters(n_adapters=0))]), INVALID),
    (dict(m=[matrix(pool=adapters(max_rank=0))]), INVALID), (dict(m=[matrix(pool=adapters(max_rank=12))]), INVALID),
    (dict(m=[matrix(pool=adapters(max_rank=136))]), INVALID), (dict(m=[matrix(pool=adapters(down_stride=16 * 1024 - 8))]), INVALID),
    (dict(m=[matrix(pool=adapters(up_stride=16 * 512 + 4))]), INVALID), (dict(m=[matrix(pool=adapters(down_stride=1 << 50))]), INVALID),
    # outputs over what is read, or each other
    (dict(m=[matrix(output=7 * MIB + 16)]), INVALID), (dict(m=[matrix(output=100 * MIB)]), INVALID), (dict(m=[matrix(output=121 * MIB)]), INVALID),
    (dict(m=[matrix(output=4 * MIB)]), INVALID), (dict(m=[matrix(output=8 * MIB)]), INVALID), (dict(m=[matrix(pool=adapters(), output=50 * MIB + 4096)]), INVALID),
    (dict(m=[matrix(pool=adapters(), output=60 * MIB)]), INVALID), (dict(m=[matrix(pool=adapters(), output=71 * MIB)]), INVALID),
    (dict(m=[matrix(100), matrix(200, output=130 * MIB + 1024 * 8)]), INVALID), (dict(m=[matrix(100), matrix(200, output=100 * MIB)]), INVALID),
    (dict(m=[matrix(residual=130 * MIB, residual_stride=520)]), INVALID), (dict(m=[matrix(residual=130 * MIB + 16)]), INVALID),
    (dict(m=[matrix(100), matrix(200, residual=130 * MIB)]), INVALID),
    (dict(b=batch(n_tokens=0)), INVALID), (dict(b=batch(positions=None)), INVALID), (dict(b=batch(positions=4 * MIB + 1)), INVALID),
    (dict(b=batch(n_tokens=(1 << 20) + 1)), INVALID)])
def test_products_that_are_refused(lib, bad, code):
    assert call_mat_mul(lib, **bad) == code, lib.last()
    assert b"llama2_batch_mat_mul_int4" in lib.last()


@pytest.mark.parametrize("bad,code", [
    (dict(o=None), INVALID), (dict(o=30 * MIB + 2), INVALID), (dict(x=None), INVALID), (dict(g=None), INVALID), (dict(u=None), INVALID),
    (dict(u=(None, 220, 221)), INVALID), (dict(rows=4), INVALID), (dict(rows=32776, sx=32776), UNSUPPORTED), (dict(cols=4), INVALID), (dict(so=504), INVALID), (dict(so=516), INVALID),
    (dict(sx=1000), INVALID), (dict(ga=adapters(), ids=None), INVALID), (dict(ua=adapters(max_rank=4)), INVALID), (dict(o=7 * MIB), INVALID),
    (dict(o=200 * MIB), INVALID), (dict(o=60 * MIB, ua=adapters()), INVALID), (dict(o=4 * MIB), INVALID), (dict(b=batch(n_requests=0)), INVALID)])
def test_gated_products_that_are_refused(lib, bad, code):
    assert call_swiglu(lib, **bad) == code, lib.last()
    assert b"llama2_batch_mat_mul_swiglu" in lib.last()


NORM = dict(o=10 * MIB, ro=20 * MIB, r=30 * MIB, x=40 * MIB, g=50 * MIB, ig=51 * MIB, gate=52 * MIB, b=None, size=512, so=512, sro=512, sr=512,
            sx=512, scale=1.0, eps=1e-5)


def call_norm(lib, **other):
    a = dict(NORM, **other)
    a["b"] = a["b"] or batch()
    return lib.norm(*a.values())


def test_norms(lib):
    for good in (dict(), dict(o=40 * MIB), dict(ro=30 * MIB), dict(o=None, g=None), dict(o=None), dict(ro=None), dict(x=None, ig=None, gate=None),
                 dict(so=1024, sr=520), dict(ig=None), dict(gate=None), dict(size=1 << 16, so=1 << 16, sro=1 << 16, sr=1 << 16, sx=1 << 16)):
        assert call_norm(lib, **good) == 0, (good, lib.last())
    for bad in (dict(r=None), dict(o=None, ro=None), dict(g=None), dict(x=None), dict(x=None, ig=None), dict(o=10 * MIB + 8), dict(gate=52 * MIB + 2),
                dict(size=0), dict(size=12), dict(so=504), dict(sr=516), dict(sx=0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(eps=-1.0), dict(eps=float("nan")), dict(o=20 * MIB), dict(o=30 * MIB), dict(ro=40 * MIB), dict(ro=30 * MIB + 16),
                dict(ro=30 * MIB, sro=1024), dict(o=40 * MIB, so=520), dict(o=50 * MIB), dict(ro=52 * MIB), dict(ro=4 * MIB), dict(b=batch(positions=None)),
                dict(b=batch(n_tokens=-1))):
        assert call_norm(lib, **bad) == INVALID, (bad, lib.last())
        assert b"llama2_batch_residual_rmsnorm" in lib.last()
    big = (1 << 16) + 8
    assert call_norm(lib, size=big, so=big, sro=big, sr=big, sx=big) == UNSUPPORTED


LOG_PROBS = dict(lp=10 * MIB, h=11 * MIB, top=12 * MIB, tlp=13 * MIB, x=20 * MIB, tokens=30 * MIB, positions=31 * MIB, rows=9, vocab=32000, stride=32000,
                 n=3, n_top=5, temperature=1.0)


def test_log_probabilities(lib):
    call = lambda **o: lib.log_probs(*dict(LOG_PROBS, **o).values())  # noqa: E731
    for good in (dict(), dict(positions=None), dict(lp=None, tokens=None, n=0), dict(h=None), dict(top=None, tlp=None, n_top=0), dict(tlp=None),
                 dict(x=20 * MIB + 2), dict(vocab=1, stride=1), dict(stride=33001), dict(n=1024), dict(n_top=64)):
        assert call(**good) == 0, (good, lib.last())
    for bad in (dict(x=None), dict(x=20 * MIB + 1), dict(lp=None, h=None, top=None, tlp=None, n=0, n_top=0), dict(rows=0), dict(rows=(1 << 20) + 1),
                dict(vocab=0), dict(stride=31999), dict(n=-1), dict(n=1025), dict(n=0), dict(lp=None), dict(tokens=None), dict(n_top=65), dict(n_top=-1),
                dict(n_top=0), dict(top=None), dict(top=None, n_top=0), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(h=11 * MIB + 2), dict(tokens=30 * MIB + 1), dict(positions=31 * MIB + 3), dict(lp=11 * MIB),
                dict(top=20 * MIB + 64), dict(tlp=30 * MIB), dict(h=31 * MIB)):
        assert call(**bad) == INVALID, (bad, lib.last())
        assert b"llama2_batch_log_probs" in lib.last()
    assert call(vocab=(1 << 20) + 1, stride=(1 << 20) + 1) == UNSUPPORTED


def test_how_rows_of_logits_are_cut(lib):
    out = (C.c_int * 3)()
    for rows in (1, 2, 3, 40, 255, 256, 300, 1 << 15):
        for vocab in (1, 7, 8, 4095, 4096, 4097, 32000, 32768, 32769, 128000, 262144, (1 << 20) - 1, 1 << 20):
            for n_top in (0, 1, 5, 64):
                lib.shape(rows, vocab, n_top, 256, out)
                segments, length, pieces = out
                assert length % 8 == 0 and (segments - 1) * length < vocab <= segments * length, (rows, vocab, n_top)
                assert length <= 4096 * pieces and pieces in (1, 2, 4, 8)  # what a workgroup's registers hold
                assert segments <= 64 and segments * n_top <= 2048  # lanes, and keys in its memory
                assert segments == 1 or vocab > 4096
                assert segments * rows <= 256 or segments == -(-vocab // 32768) or length == 32768


def test_calls_before_init_are_refused():
    import sys
    code = ("import sys; sys.path.insert(0, %r)\nfrom managedllama2_amd import capi\n"
            "for n in %r:\n    assert capi.raw(n, *[a() if a is not capi.vp and not hasattr(a, 'contents') else None for a in capi._SIGNATURES[n]]) == "
            "capi.ERR_NOT_INITIALIZED, n\nprint('ok')\n" % (ROOT, sorted(NAMES.values())))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "ok" in out.stdout, out.stderr
