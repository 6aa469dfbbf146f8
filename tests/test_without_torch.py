"""The library, its Python binding and its tests where torch is not installed."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def without_torch(code):
    return subprocess.run([sys.executable, "-c", "import sys; sys.modules['torch'] = None; " + code], cwd=ROOT,
                          capture_output=True, text=True, timeout=120)


def test_bindings_load():
    r = without_torch("import __graft_entry__ as entry; entry.load(); import qwen_decode as qd; print(qd.lib().qd_abi_version())")
    assert r.returncode == 0, r.stderr
    assert int(r.stdout) > 0


def test_tests_are_collected():
    r = without_torch("import pytest; sys.exit(pytest.main(['tests', '--collect-only', '-q', '-p', 'no:cacheprovider']))")
    assert r.returncode == 0, r.stdout + r.stderr
    assert "test_gpu_beams.py" in r.stdout and "test_gpu_decode.py" in r.stdout
    assert "test_operators.py::" not in r.stdout and "test_gpu_operators.py::" not in r.stdout
