"""bench.py without the compiled reference: its own arm and the reference arm still end with a line."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_reference_arm_says_why_it_is_unavailable():
    import oracle
    if os.path.exists(oracle.REF_SO):
        pytest.skip("the compiled reference is here")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--impl", "reference", "--gpus", "1", "--steps", "2", "--warmup", "1"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    line = json.loads(r.stdout)
    assert line["impl"] == "reference" and "libatt1ref.so" in line["unavailable"] and "\n" not in line["unavailable"]


@pytest.mark.gpu
def test_bench_line_without_the_reference():
    """Two layers and a short context: the fields, not the figures."""
    import oracle
    if os.path.exists(oracle.REF_SO):
        pytest.skip("the compiled reference is here")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--layers", "2", "--ctx", "512", "--prompt", "8", "--steps", "4",
                        "--warmup", "3", "--no-extras"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    line = json.loads(r.stdout)
    assert line["value"] > 0 and line["e2e"]["value"] > 0 and "unavailable" in line["cpu_baseline"]
