"""Whether buffers of a call share bytes (csrc/overlap.h, which the entry points'
checks use), against a map of bytes (tests/cpp/overlap_check.cpp)."""
import os
import subprocess

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "overlap_check")


def test_blocks_and_rows():
    assert os.path.exists(BIN), "tests/cpp/overlap_check not built (run __graft_entry__.build())"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
