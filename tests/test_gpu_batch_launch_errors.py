"""An error of a launch is reported by the call that made it.  HIP keeps a thread's last error until somebody asks for it; a refused host call (a device
that does not exist) leaves one here, and no kernel is involved."""
import ctypes as C

import numpy as np
import pytest

import product_util as pu
from managedllama2_amd import capi, synth
from managedllama2_amd.device import init

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def ready():
    init(0)


def hip():
    """The HIP runtime that the library itself is linked to."""
    capi.load()
    runtime = C.CDLL(next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line))
    runtime.hipGetLastError.restype = C.c_int
    return runtime


@pytest.mark.parametrize("tokens", [1, 2, 70])
@pytest.mark.parametrize("gated", [False, True])
def test_an_error_of_a_product_is_reported_once(tokens, gated):
    p = pu.Product(synth.rng_for(1790, tokens, gated), tokens, 512, [64], gated).upload()
    p.check()
    outs, runtime = p.outputs(), hip()
    assert runtime.hipSetDevice(1 << 20) != 0
    rc, said = capi.raw(*p.args(outs)), capi.last_error()
    assert runtime.hipGetLastError() == 0, "left for another call to report"
    assert rc > 0 and ("swiglu" if gated else "int4") in said, (rc, said)
    p.check()
    assert np.isfinite(outs[0].to_host()).all()
