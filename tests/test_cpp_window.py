"""Windowed attention through the C++ host API: tests/cpp/test_window.cpp, built by barracuda_amd.build into
tests/cpp/bch_window_tests."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

EXE = Path(__file__).resolve().parent / "cpp" / "bch_window_tests"


def _run(mode: str) -> str:
    assert EXE.exists(), f"{EXE} not built: python -m barracuda_amd.build"
    r = subprocess.run([str(EXE), mode], capture_output=True, text=True, timeout=100)
    print(r.stdout, flush=True)
    assert r.returncode == 0 and "FAIL" not in r.stdout, r.stdout + r.stderr
    return r.stdout


def test_checks():
    assert "PASS window_checks" in _run("--cpu")


@pytest.mark.gpu
def test_result():
    assert "PASS window_result" in _run("--gpu")
