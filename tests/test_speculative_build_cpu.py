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


def test_another_torch_or_python_rebuilds_the_module(monkeypatch):
    assert build.build_spec() == build.SPEC  # up to date now
    built = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd: built.append(cmd))
    monkeypatch.setattr(os, "remove", lambda path: None)
    assert build.build_spec() == build.SPEC and not built
    with monkeypatch.context() as m:
        m.setattr(build, "SPEC_FOR", os.devnull)  # built for something else; written to nowhere
        build.build_spec()
        assert len(built) == 1
    monkeypatch.setattr(torch, "__version__", "0.0")
    monkeypatch.setattr(build, "_write", lambda path, text: None)
    build.build_spec()
    assert len(built) == 2


def test_a_module_that_does_not_load_is_built_again(monkeypatch):
    import ds_ocr_b200
    from ds_ocr_b200 import speculative
    good, name, asked = speculative._module(), "ds_ocr_b200._spec", []
    monkeypatch.delattr(ds_ocr_b200, "_spec")
    monkeypatch.setitem(sys.modules, name, None)  # its import fails

    def rebuilt(verbose=False, force=False):
        asked.append(force)
        sys.modules[name] = good

    monkeypatch.setattr(build, "build_spec", rebuilt)
    assert speculative._module() is good and asked == [True]
