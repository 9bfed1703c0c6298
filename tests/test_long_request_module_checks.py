"""The C++ modules' checks of the calls for long requests, on the host: tests/cpp/long_request_checks_test.cpp."""
import pathlib
import subprocess

REPO = pathlib.Path(__file__).resolve().parents[1]


def test_views_that_do_not_fit_are_refused():
    subprocess.run(["make", "-s", "-C", str(REPO / "tests" / "cpp")], check=True)
    r = subprocess.run([str(REPO / "tests" / "cpp" / "bin" / "long_request_checks_test")], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
