"""The recurrence's GPU tests on the debug build (libgdn_b200_debug.so), in a
fresh process.  Its device-side index checks (tiles against the call's rows and
channels, sequences of starts and ends, words of other chunks, rows that are
written) record device status 4 on a violation; those tests assert a clean device
status after every case.  It also holds map-only tiles back, which changes the
order in which tiles finish."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def test_recurrence_suites_pass_on_the_index_checked_build():
    sys.path.insert(0, str(ROOT / "track-c-gdn_b200"))
    try:
        import build as native_build
    finally:
        sys.path.pop(0)
    lib = native_build.build(debug=True)
    files = ["tests/test_recurrence_gpu.py", "tests/test_recurrence_modes_gpu.py"]
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", *files], cwd=ROOT,
                         env=dict(os.environ, GDN_B200_LIBRARY=str(lib)), capture_output=True, text=True, timeout=900)
    assert res.returncode == 0, res.stdout[-3000:] + res.stderr[-2000:]
