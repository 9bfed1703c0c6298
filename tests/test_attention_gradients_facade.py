"""The C++ attention module's gradients, item by item against the formulas: tests/cpp/attention_gradients_test.cpp."""
import pathlib
import subprocess

import pytest

REPO = pathlib.Path(__file__).resolve().parents[1]
BIN = REPO / "tests" / "cpp" / "bin" / "attention_gradients_test"


def test_the_comparison_tells_wrong_gradients_apart():
    subprocess.run(["make", "-s", "-C", str(REPO / "tests" / "cpp")], check=True)
    r = subprocess.run([str(BIN), "--host"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "1 cases, 0 failures" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_gradients_of_the_module():
    assert BIN.exists(), "tests/cpp/bin/attention_gradients_test is missing: run __graft_entry__.build()"
    cases = subprocess.run([str(BIN), "--list"], check=True, capture_output=True, text=True).stdout.split()
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=110)
    print(r.stdout)
    print(r.stderr)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
    assert f"{len(cases)} cases, 0 failures" in r.stdout
