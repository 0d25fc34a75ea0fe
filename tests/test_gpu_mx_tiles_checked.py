"""Every tile of the MXFP4 products in the device-checked build
(aiehlc_amd/lib_dbg), on buffers exactly as long as the header says
(tests/mx_tiles_checks_child.py, in a process of its own: this one holds the
product build)."""
import json
import os
import subprocess
import sys

import pytest

import test_gpu_mx_tiles as tiles

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_DBG = os.path.join(ROOT, "aiehlc_amd", "lib_dbg")

pytestmark = pytest.mark.gpu


@pytest.mark.skipif(not os.path.exists(os.path.join(LIB_DBG, "libmiaie.so")),
                    reason="device-checked build missing (aiehlc_amd/build.py builds it)")
def test_every_tile_stays_in_its_buffers():
    print("[case] device-checked MXFP4 tiles, child process", flush=True)
    env = dict(os.environ, MIAIE_LIB_DIR=LIB_DBG)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "mx_tiles_checks_child.py")], env=env,
                       capture_output=True, text=True, timeout=110)
    sys.stderr.write(r.stderr[-4000:])
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    cases = json.loads(r.stdout.strip().splitlines()[-1])["cases"]
    assert {(out, str(kernel)) for kernel, (out, *_) in tiles.CASES} == {
        (out, str(tiles.planned((out, *shape)))) for out, *shape in cases}
