"""The reference arm of the benchmark runs the reference or says that it cannot."""
import json
import os
import subprocess
import sys

from oracle import oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_reference_arm_is_the_reference_or_unavailable():
    cmd = [sys.executable, os.path.join(ROOT, "bench.py"), "--impl", "reference", "--workload", "cfg1", "--steps", "1", "--warmup", "1"]
    done = subprocess.run(cmd, capture_output=True, text=True, timeout=600, cwd=ROOT)
    assert done.returncode == 0, done.stderr[-2000:]
    line = json.loads(done.stdout.strip().splitlines()[-1])
    assert line["impl"] == "reference"
    if O.load_ref_python() is None:
        assert set(line) == {"impl", "unavailable"} and "\n" not in line["unavailable"]
    else:
        assert line["cpu_baseline"]["kind"] == "reference" and line["value"] > 0
