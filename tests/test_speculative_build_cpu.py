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
