"""The compiled caller is optional: where calls.c does not compile, the build goes on
without it (sgblas_b200/build.py). No GPU needed."""
import importlib.util
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
NAME = f"_calls{sysconfig.get_config_var('EXT_SUFFIX')}"


@pytest.fixture()
def package(tmp_path):
    """A copy of what _build_calls reads, and its module."""
    shutil.copytree(ROOT / "include", tmp_path / "include")
    (tmp_path / "sgblas_b200").mkdir()
    for name in ("build.py", "calls.c"):
        shutil.copy(ROOT / "sgblas_b200" / name, tmp_path / "sgblas_b200" / name)
    spec = importlib.util.spec_from_file_location("build_of_a_copy", tmp_path / "sgblas_b200" / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def left(package):
    return sorted(p.name for p in package.PKG.iterdir() if p.name.startswith("_calls"))


def stale(package):
    """As an older source left it: no library, and a method fewer."""
    old = package.PKG / NAME
    old.write_bytes(b"old")
    os.utime(old, (0, 0))


def test_it_compiles_here(package):
    if shutil.which("gcc") is None or not pathlib.Path(sysconfig.get_paths()["include"], "Python.h").exists():
        pytest.skip("gcc and Python's headers are needed")
    stale(package)
    package._build_calls()
    assert left(package) == [NAME] and (package.PKG / NAME).read_bytes()[:4] == b"\x7fELF"


def test_a_source_that_does_not_compile(package, capsys):
    (package.PKG / "calls.c").write_text("#error an older Python\n")
    stale(package)
    package._build_calls()
    assert left(package) == [] and "ctypes" in capsys.readouterr().err


def test_no_compiler(package, capsys, monkeypatch, tmp_path):
    monkeypatch.setenv("PATH", str(tmp_path))
    monkeypatch.delenv("CC", raising=False)
    stale(package)
    package._build_calls()
    assert left(package) == [] and "no C compiler" in capsys.readouterr().err


def test_no_headers(package, capsys, monkeypatch, tmp_path):
    monkeypatch.setattr(package.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    stale(package)
    package._build_calls()
    assert left(package) == [] and "Python.h" in capsys.readouterr().err


def test_the_package_without_it():
    """Imported without the compiled caller, the same calls are refused and taken."""
    code = ("import sys; sys.modules['sgblas_b200._calls'] = None\n"
            "import sgblas_b200 as sg\n"
            "assert sg._direct is None\n"
            "with sg.Handle() as h:\n"
            "    h.rms_norm(0, 3, sg.SGBLAS_TYPE_BF16, None, 1, None, 1, None, 1e-6, y=None, ldy=1)\n"
            "    try:\n"
            "        h.sort_tokens(-1, 1, 4, None, 16, None)\n"
            "    except sg.SgblasError as e:\n"
            "        assert e.status == sg.SGBLAS_STATUS_INVALID_VALUE\n"
            "    else:\n"
            "        raise AssertionError\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)
