"""What the 4-bit cache's attention does once a bounded wait for a copy has run out, on the host: tests/probes/
kv4_ring_probe.cu plays the ring's loop with one copy that does not land. A kernel must not wait out the limit for
each of the copies after it, nor end with copies in flight. Built with nvcc for the host side only; no GPU."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_a_wait_that_runs_out_is_the_last_but_for_copies_in_flight(tmp_path):
    from voxgen_b200 import _build
    try:
        nvcc = _build.nvcc()
    except FileNotFoundError:
        pytest.skip("nvcc not found")
    exe = tmp_path / "kv4_ring_probe"
    subprocess.run([nvcc, "-std=c++17", "--expt-relaxed-constexpr", *_build.ARCH, "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "probes" / "kv4_ring_probe.cu"), "-o", str(exe)],
                   check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout + r.stderr
