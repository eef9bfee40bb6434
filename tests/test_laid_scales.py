"""Where a pair's scale blocks are laid out (tests/laid_scales.cu): inside the
workspace, whatever the device's offsets hold. No GPU needed."""
import pathlib
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent


def test_blocks_stay_in_the_workspace(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not pathlib.Path(nvcc).exists():
        pytest.skip("nvcc is needed")
    exe = tmp_path / "laid_scales"
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{ROOT / 'include'}",
                    f"-I{ROOT / 'sgblas_b200' / 'csrc'}", str(ROOT / "tests" / "laid_scales.cu"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert int(run.stdout) == 6 * 5 * 6 * 4
