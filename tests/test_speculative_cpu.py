"""Host side of the speculative-decoding operators that needs no GPU: the
ctypes descriptors match the C structs, a missing context is an error, and
the plain verification used as the GPU tests' reference keeps the target's
distribution."""
import os
import subprocess

import numpy as np

import spec_ref as R
from ds_ocr_b200 import _lib, speculative as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_descriptors_match_the_header(tmp_path):
    names = {"ds_cuda_tree_attention_t": S.TreeAttentionDesc, "ds_cuda_tree_verify_t": S.TreeVerifyDesc,
             "ds_cuda_tree_commit_t": S.TreeCommitDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ds_cuda.h"', "int main(void) {"]
    want = []
    for c, py in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(S.ctypes.sizeof(py))
        for f, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {f}));')
            want.append(getattr(py, f).offset)
    src = tmp_path / "off.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    exe = tmp_path / "off"
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want


def test_missing_context_is_an_error():
    lib = _lib.load()
    d, v, c = S.TreeAttentionDesc(), S.TreeVerifyDesc(), S.TreeCommitDesc()
    ref = S.ctypes.byref
    assert lib.ds_cuda_tree_attention_dev(None, ref(d), None) < 0
    assert lib.ds_cuda_tree_attention_workspace(None, ref(d)) == 0
    assert lib.ds_cuda_tree_verify_dev(None, ref(v), None) < 0
    assert lib.ds_cuda_tree_commit_dev(None, ref(c), None) < 0
    assert lib.ds_cuda_tree_mask_dev(None, None, None, 1, 1, None, None, None) < 0
    assert lib.ds_cuda_token_probs_dev(None, 2, None, 1, 1, 1, None, None, None) < 0
    assert lib.ds_cuda_tree_verify_greedy_dev(None, None, None, None, None, 1, 1, None, None, None, None) < 0


def test_plain_verification_keeps_the_target_distribution():
    rng = np.random.default_rng(0)
    vocab, trials = 5, 20000
    p = rng.dirichlet(np.ones(vocab)).astype(np.float32)
    for certain in (False, True):
        q = rng.dirichlet(np.ones(vocab)).astype(np.float32)
        cdf = np.cumsum(q.astype(np.float64))
        got = np.zeros(vocab)
        target, draft = np.tile(p, (3, 1)), None if certain else np.tile(q, (3, 1))
        for _ in range(trials):
            tok = np.minimum(vocab - 1, np.searchsorted(cdf, rng.random(3) * cdf[-1]))
            path, t = R.verify(tok, [-1, 0, 0], 3, target, draft, rng.random(3).astype(np.float32) * np.float32(0.9999999),
                               np.float32(rng.random()) * np.float32(0.9999999))
            got[tok[path[1]] if len(path) > 1 else t] += 1
        want = p.astype(np.float64) / p.astype(np.float64).sum() * trials
        assert ((got - want) ** 2 / want).sum() < 33  # chi-square, 4 degrees of freedom, 1e-6


def test_plain_sums_have_no_order():
    rng = np.random.default_rng(1)
    r = rng.dirichlet(np.full(4096, 0.02)).astype(np.float32)
    w = R.fixed(r)
    assert int(w.sum()) == int(w[rng.permutation(4096)].sum()) and abs(w.sum() / 2.0 ** 44 - 1) < 1e-5
    assert R.fixed(np.array([np.nan, -1, 0, 2, np.inf], np.float32)).tolist() == [0, 0, 0, 1 << 44, 1 << 44]
