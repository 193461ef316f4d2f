"""The build: the C library and the ctypes binding need no torch, the torch binding belongs to one Python and torch."""
import subprocess
import sys
import sysconfig
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
BLOCK = "import sys; sys.modules['torch'] = None\n"


def run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=600)


def test_library_builds_and_loads_without_torch(built_lib):
    r = run(BLOCK + "from funasrnet_b200 import build, _lib\n"
                    "print(build.build_library()); print(_lib.lib().fa_version().decode())\n"
                    "import funasrnet_b200.backend")
    assert r.returncode == 0, r.stderr
    assert r.stdout.splitlines()[0] == str(built_lib) and "sm_100a" in r.stdout
    assert "torch is not installed" in r.stderr


def test_a_library_that_is_up_to_date_imports_no_torch(built_lib):
    r = run("import sys\nfrom funasrnet_b200 import build\nbuild.build_library()\nassert 'torch' not in sys.modules")
    assert r.returncode == 0, r.stderr


def test_a_binding_that_cannot_be_compiled_leaves_the_library(built_lib, monkeypatch, capsys):
    from funasrnet_b200 import build

    def fails():
        raise RuntimeError("Python.h: no such file")

    monkeypatch.setattr(build, "build_binding", fails)
    assert build.build_library() == built_lib
    assert "Python.h" in capsys.readouterr().err


def test_the_binding_is_named_after_its_python_and_torch(built_lib):
    import torch

    from funasrnet_b200 import build

    name = build.build_binding().name
    assert sysconfig.get_config_var("SOABI") in name and str(torch.__version__) in name


def test_a_missing_binding_is_a_clear_error(built_lib):
    r = run("from pathlib import Path\nfrom funasrnet_b200 import device_ops\n"
            "device_ops.binding_path = lambda: Path('/nowhere/_torch_ops.so')\ndevice_ops._native()")
    assert r.returncode != 0 and "/nowhere/_torch_ops.so is missing" in r.stderr
