"""The C++ attention module's checks, on the host: tests/cpp/attention_checks_test.cpp."""
import pathlib
import subprocess

REPO = pathlib.Path(__file__).resolve().parents[1]


def test_calls_before_create_are_refused():
    subprocess.run(["make", "-s", "-C", str(REPO / "tests" / "cpp")], check=True)
    r = subprocess.run([str(REPO / "tests" / "cpp" / "bin" / "attention_checks_test")], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
