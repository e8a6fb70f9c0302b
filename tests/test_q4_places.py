"""The places in a packed row that the 4-bit weight products read
(csrc/q4_layout.h, which the kernels use): inside the row for every length, chunk
and lane group (tests/cpp/q4_places.cpp)."""
import os
import subprocess

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "q4_places")


def test_every_place_lies_in_its_row():
    assert os.path.exists(BIN), "tests/cpp/q4_places not built (run __graft_entry__.build())"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
