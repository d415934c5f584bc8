"""CPU: what `make` builds with and without torch (dry runs: nothing is compiled)."""
import os
import shutil
import stat
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stablediffusion-cpp_b200")

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make")


def dry(*args):
    r = subprocess.run(["make", "-n", "-C", PKG, *args], capture_output=True, text=True)
    return r.returncode, r.stdout + r.stderr


def interpreter(tmp_path, body):
    p = tmp_path / "python"
    p.write_text(f"#!/bin/sh\n{body}\n")
    p.chmod(p.stat().st_mode | stat.S_IXUSR)
    return f"PYTHON={p}"


@pytest.mark.parametrize("body", ["exit 1", "exit 127", f'{sys.executable} -S -c "import sys; sys.path[:] = []" >/dev/null; exit 1'])
def test_the_library_builds_where_there_is_no_torch(tmp_path, body):
    rc, text = dry("-B", interpreter(tmp_path, body))
    assert rc == 0, text
    assert "-o sdb200/libsdb200.so" in text and "serving_py.cpp" not in text


def test_an_interpreter_that_is_not_there(tmp_path):
    rc, text = dry("-B", f"PYTHON={tmp_path}/none")
    assert rc == 0 and "-o sdb200/libsdb200.so" in text and "serving_py.cpp" not in text, text


def test_the_library_alone(tmp_path):
    rc, text = dry("-B", "lib", interpreter(tmp_path, "exit 1"))
    assert rc == 0 and "-o sdb200/libsdb200.so" in text and "serving_py.cpp" not in text, text


def test_both_build_with_torch():
    rc, text = dry("-B", f"PYTHON={sys.executable}")
    assert rc == 0 and "-o sdb200/libsdb200.so" in text and "-o sdb200/_serving.so" in text, text


def test_another_torch_rebuilds_the_binding(tmp_path):
    """The binding is linked against one torch; an interpreter with another one asks for it anew."""
    subprocess.run(["make", "-C", PKG, f"PYTHON={sys.executable}", "sdb200/_serving.so"], check=True, capture_output=True)
    rc, text = dry(f"PYTHON={sys.executable}", "sdb200/_serving.so")
    assert rc == 0 and "serving_py.cpp" not in text, text
    fake = tmp_path / "site" / "torch"
    (fake / "include").mkdir(parents=True)
    (fake / "__init__.py").write_text("")
    (fake / "version.py").write_text("__version__ = '0.0.1'\n")
    rc, text = dry(interpreter(tmp_path, f'PYTHONPATH={tmp_path}/site exec {sys.executable} "$@"'), "sdb200/_serving.so")
    assert rc == 0 and f"-I{fake}/include" in text and "serving_py.cpp" in text, text
