"""The torch module of the speculative-decoding calls: which library it
calls, and when it is built."""
import os
import shutil
import subprocess
import sys

import pytest

from ds_ocr_b200 import build

torch = pytest.importorskip("torch")


def test_the_module_calls_the_library_that_was_loaded(tmp_path):
    lib = shutil.copy(build.LIB, tmp_path / "libds_cuda_elsewhere.so")
    code = ("from ds_ocr_b200 import _lib, speculative\n"
            "_lib.load()\n"
            "speculative._module()\n"
            "print(sorted({l.split()[-1] for l in open('/proc/self/maps') if 'libds_cuda' in l}))\n")
    out = subprocess.run([sys.executable, "-c", code], cwd=build.ROOT, env={**os.environ, "DS_CUDA_LIB": str(lib)},
                         check=True, capture_output=True, text=True).stdout
    assert out.strip() == str([str(lib)])


def test_the_library_builds_where_the_module_does_not(monkeypatch, capsys):
    def broken(*_):
        raise subprocess.CalledProcessError(1, ["g++"])

    monkeypatch.setattr(build, "build_spec", broken)
    assert build.build() == build.LIB
    assert "_spec" in capsys.readouterr().err


def test_no_module_for_a_torch_without_cuda(monkeypatch):
    monkeypatch.setattr(torch.version, "cuda", None)
    monkeypatch.setattr(subprocess, "check_call", lambda *_: pytest.fail("built"))
    assert build.build_spec(force=True) is None


def test_an_old_module_does_not_outlive_a_failed_build(monkeypatch, tmp_path):
    def broken(*_):
        raise subprocess.CalledProcessError(1, ["g++"])

    old = tmp_path / "_spec.so"
    old.write_bytes(b"old")
    monkeypatch.setattr(build, "SPEC", str(old))
    monkeypatch.setattr(subprocess, "check_call", broken)
    with pytest.raises(subprocess.CalledProcessError):
        build.build_spec(force=True)
    assert not old.exists()
