"""The native half of dsmoe.ops (_ops.so) is built for one PyTorch: the package imports without it, the operators say
what is missing, and make builds it anew for another PyTorch. On the CPU, with stand-ins for the compilers."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "tenstorrent-wormhole-deepseek-v41-flash_b200")

USE = """
import dsmoe, kernel, torch
from dsmoe import MoE, Expert, Int8Experts, ExpertStore, _lib
assert kernel.int8_gemm is dsmoe.int8_gemm and _lib.lib.dsmoe_version() > 0
assert not hasattr(dsmoe.ops._ops, "__wrapped__")
for call in (lambda: dsmoe.sort_tokens(torch.zeros(2, 1, dtype=torch.int64), 2), lambda: kernel.swiglu_quant(torch.zeros(2, 4))):
    try:
        call()
    except ImportError as e:
        assert "dsmoe/_ops.so" in str(e) and torch.__version__ in str(e), e
    else:
        raise AssertionError("no error")
print("fine")
"""


@pytest.mark.parametrize("module", [None, b"", b"built for something else"])
def test_package_imports_without_the_native_module(tmp_path, module):
    shutil.copytree(PKG, tmp_path / "pkg", ignore=shutil.ignore_patterns("_ops*.so", "csrc", "__pycache__"))
    if module is not None:
        (tmp_path / "pkg" / "dsmoe" / "_ops.so").write_bytes(module)
    r = subprocess.run([sys.executable, "-c", USE], cwd=tmp_path / "pkg", capture_output=True, text=True,
                       env={**os.environ, "PYTHONPATH": str(tmp_path / "pkg")})
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr


def _script(path, text):
    path.write_text("#!/bin/sh\n" + text)
    path.chmod(0o755)
    return str(path)


def test_make_follows_pytorch(tmp_path):
    """make with compilers that only touch their output and a Python that names a version of PyTorch."""
    csrc = tmp_path / "pkg" / "csrc"
    for d in (csrc, tmp_path / "pkg" / "dsmoe", tmp_path / "include"):
        d.mkdir(parents=True)
    shutil.copy(os.path.join(PKG, "csrc", "Makefile"), csrc)
    for f in (csrc / "a.cu", csrc / "pyops.cpp", tmp_path / "include" / "dsmoe.h"):
        f.write_text("")
    cc = _script(tmp_path / "cc", 'while [ $# -gt 0 ]; do if [ "$1" = -o ]; then touch "$2"; echo "$2" >> "%s/log"; fi; shift; done\n'
                 % tmp_path)
    py = _script(tmp_path / "py", 'case "$2" in *cache_tag*) [ -n "$FAKE_TORCH" ] && echo "$FAKE_TORCH" || exit 1;; *) echo /nowhere;; esac\n')

    def make(torch):
        (tmp_path / "log").write_text("")
        r = subprocess.run(["make", "-C", str(csrc), f"NVCC={cc}", f"CXX={cc}", f"PYTHON={py}", "CUDA_HOME=/nowhere"],
                           env={**os.environ, "FAKE_TORCH": torch}, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return [os.path.basename(p) for p in (tmp_path / "log").read_text().split()]

    assert make("") == ["a.o", "libdsmoe.so"]  # no PyTorch: the library alone, and no error
    assert make("2.0-cp") == ["_ops.so"]
    assert make("2.0-cp") == []
    assert make("2.1-cp") == ["_ops.so"]
    assert make("2.0-cp") == ["_ops.so"]  # and back
    assert make("") == []
