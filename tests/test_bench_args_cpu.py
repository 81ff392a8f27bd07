"""CPU test of the benchmark's arguments: 4-bit experts are refused where no workload uses them."""
import os
import subprocess
import sys

import pytest

BENCH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bench.py")


@pytest.mark.parametrize("args", [[], ["--workload", "c3"], ["--train"], ["--impl", "reference"]])
def test_expert_bits_elsewhere(args):
    r = subprocess.run([sys.executable, BENCH, "--expert-bits", "4", *args], capture_output=True, text=True, timeout=300)
    assert r.returncode == 2 and "decoding workloads" in r.stderr and not r.stdout
