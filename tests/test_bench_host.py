"""bench.py where the reference's CPU functions were not built (no GPU)."""
from __future__ import annotations

import json
import os
import subprocess
import sys

from conftest import ROOT

CODE = """
import sys
import oracle
oracle.ref = None
sys.argv = ["bench.py", "--impl", "reference"]
import bench
assert bench.cpu_baseline(None) == {"unavailable": bench.NO_REFERENCE}
sys.exit(bench.main())
"""


def test_the_reference_arm_says_that_it_is_unavailable():
    env = dict(os.environ, PYTHONPATH=ROOT)
    res = subprocess.run([sys.executable, "-c", CODE], capture_output=True, text=True, cwd=ROOT,
                         env=env, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    line = json.loads(res.stdout)
    assert line["impl"] == "reference" and "missing" in line["unavailable"]
