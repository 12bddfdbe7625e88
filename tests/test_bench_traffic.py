"""The HBM bytes that bench.py reports were counted for one state of the mat-vec kernels' source.  After a change there the counters are read again
(profiles/int4_matvec_7b_layer_set_hbm_traffic.md has the commands), else bench.py has no bytes to report -- no GPU."""
import hashlib
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def read(*path):
    return open(os.path.join(ROOT, *path), "rb").read()


def test_the_counters_were_read_for_this_source():
    bench = read("bench.py").decode()
    given = re.search(r'SWIGLU_HBM_TRAFFIC_SOURCE_SHA16 = "(\w+)"', bench).group(1)
    assert hashlib.sha256(read("managedllama2_amd", "csrc", "int4_kernels.hpp")).hexdigest()[:16] == given
    counted = int(re.search(r"SWIGLU_HBM_TRAFFIC_BYTES = (\d+)", bench).group(1))
    row = re.search(r"fused SwiGLU gate/up .*?\| ([\d.]+) \| ([\d.]+) \| (\d+) \|", read("profiles", "int4_matvec_7b_layer_set_hbm_traffic.md").decode())
    # means are given to a tenth of a KB
    assert counted == int(row.group(3)) and abs(counted - (float(row.group(1)) * 2 + float(row.group(2))) * 1024) <= (2 * 0.05 + 0.05) * 1024 + 1
