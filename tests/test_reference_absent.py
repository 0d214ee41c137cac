"""Tests that need the reference's own host library are skipped where neither it nor its sources are present, whether they
ask first or call it straight away; any other missing file still fails."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CASES = """
import pytest
import oracle

@pytest.fixture(autouse=True)
def absent(monkeypatch, tmp_path):
    monkeypatch.setattr(oracle, "HERE", str(tmp_path))
    monkeypatch.setattr(oracle, "REF_TREE", str(tmp_path / "none"))
    monkeypatch.setattr(oracle, "_ref", None)

def test_asks_first():
    assert not oracle.ref_available()

def test_calls_it():
    oracle.ref_twin("rmsnorm", {}, [], {})

def test_another_file():
    open("/nowhere/at/all")
"""


def test_a_call_of_the_absent_library_skips(tmp_path):
    (tmp_path / "test_cases.py").write_text(CASES)
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-rA", "-p", "tests.conftest", "-p", "no:cacheprovider",
                        "--rootdir", str(tmp_path), str(tmp_path / "test_cases.py")],
                       cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True, timeout=300)
    assert "1 failed, 1 passed, 1 skipped" in r.stdout, r.stdout + r.stderr
    assert "test_another_file" in r.stdout.split("FAILED")[-1]
