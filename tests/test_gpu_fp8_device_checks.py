"""The 8-bit operators, the routing and the experts' products in the
device-checked build (aiehlc_amd/lib_dbg), on buffers exactly as long as the header
says and on buffers declared shorter (tests/fp8_device_checks_child.py, in a process
of its own: this one holds the product build)."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_DBG = os.path.join(ROOT, "aiehlc_amd", "lib_dbg")

pytestmark = pytest.mark.gpu


@pytest.mark.skipif(not os.path.exists(os.path.join(LIB_DBG, "libmiaie.so")),
                    reason="device-checked build missing (aiehlc_amd/build.py builds it)")
def test_device_checked_fp8_and_expert_kernels():
    print("[case] device-checked 8-bit and expert kernels, child process", flush=True)
    env = dict(os.environ, MIAIE_LIB_DIR=LIB_DBG)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "fp8_device_checks_child.py")], env=env,
                       capture_output=True, text=True, timeout=110)
    sys.stderr.write(r.stderr[-4000:])
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    out = json.loads(r.stdout.strip().splitlines()[-1])
    assert len(out["cases"]) >= 100 and len(out["planted"]) == 5
