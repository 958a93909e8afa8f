"""The host side of the speculative-decoding entry points, without a GPU: the
library's own objects over a CUDA runtime of counters (fake_cuda.cu)."""
import ctypes
import os
import subprocess

import pytest

from ds_ocr_b200 import build, speculative as S

HERE = os.path.dirname(os.path.abspath(__file__))


class State(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int), ("devices", ctypes.c_int), ("launches", ctypes.c_int),
                ("launch_device", ctypes.c_int), ("word", ctypes.c_uint), ("error", ctypes.c_int), ("cluster", ctypes.c_int),
                ("room", ctypes.c_int * 17)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    objs = [os.path.join(build.BUILD, f + ".cu.o") for f in ("spec_attn", "spec_verify")]
    if not all(map(os.path.exists, objs)):
        build.build()
    tmp = tmp_path_factory.mktemp("fake")
    obj, so = str(tmp / "fake.o"), str(tmp / "fake.so")
    subprocess.check_call([build._nvcc(), *build.NVCC_FLAGS, "-I", build.CSRC, "-I", os.path.join(build.ROOT, "include"),
                           "-c", os.path.join(HERE, "fake_cuda.cu"), "-o", obj])
    # (-Bsymbolic: its own runtime, whatever else the process has loaded)
    subprocess.check_call(["g++", "-shared", "-Wl,-Bsymbolic", "-Wl,-z,defs", "-o", so, obj, *objs])
    lib = ctypes.CDLL(so)
    P, I = ctypes.c_void_p, ctypes.c_int
    for name, res, args in (("fake_new", P, [I, I]), ("fake_free", None, [P]), ("fake_state", ctypes.POINTER(State), []),
                            ("fake_message", ctypes.c_char_p, [P])):
        f = getattr(lib, name)
        f.restype, f.argtypes = res, args
    from ds_ocr_b200 import _lib
    for name, (res, args) in _lib.SIGNATURES.items():
        if name.startswith(("ds_cuda_tree", "ds_cuda_token")):
            f = getattr(lib, name)
            f.restype, f.argtypes = res, args
    return lib


@pytest.fixture
def ctx(lib):
    h = lib.fake_new(1, 148)
    yield h
    lib.fake_free(h)


def attention(type=S.BF16, batch=2, n_nodes=4, n_heads=4, n_kv_heads=2, head_dim=64, kv_max=128):
    """A descriptor with addresses that nothing reads."""
    d = S.TreeAttentionDesc(type=type, batch=batch, n_nodes=n_nodes, n_heads=n_heads, n_kv_heads=n_kv_heads,
                            head_dim=head_dim, kv_max=kv_max, scale=0.125)
    for i, name in enumerate(("q", "k", "v", "tree_k", "tree_v", "lens", "mask", "out")):
        setattr(d, name, 4096 * (i + 1))
    for name, rows in (("k", kv_max), ("v", kv_max), ("tree_k", n_nodes), ("tree_v", n_nodes)):
        setattr(d, name + "_stride", (ctypes.c_int64 * 3)(n_kv_heads * rows * head_dim, rows * head_dim, head_dim))
    for name in ("q", "out"):
        setattr(d, name + "_stride", (ctypes.c_int64 * 3)(n_nodes * n_heads * head_dim, n_heads * head_dim, head_dim))
    return d


def attend(lib, ctx, d):
    d.workspace_bytes = lib.ds_cuda_tree_attention_workspace(ctx, ctypes.byref(d))
    d.workspace = 1 << 20
    return lib.ds_cuda_tree_attention_dev(ctx, ctypes.byref(d), None)


@pytest.mark.parametrize("sizes", [
    # 256 sequences with room for 65536 rows, 64 heads on 8, trees of 64: 8.4 million tiles
    dict(batch=256, n_nodes=64, n_heads=64, n_kv_heads=8, kv_max=65536),
    # one sequence of 2^28 tiles, and many of 16392 each
    dict(batch=1, n_nodes=256, n_heads=64, n_kv_heads=64, kv_max=1 << 24, type=S.F32),
    dict(batch=65535, n_nodes=1, n_heads=8, n_kv_heads=8, kv_max=131072),
])
def test_attention_takes_any_list_of_tiles_below_2_to_31(lib, ctx, sizes):
    d = attention(**sizes)
    assert attend(lib, ctx, d) == 0, lib.fake_message(ctx)
    assert d.workspace_bytes > 0 and lib.fake_state().contents.launches == 2


@pytest.mark.parametrize("sizes", [
    dict(batch=65535, n_nodes=256, n_heads=65535, n_kv_heads=65535, kv_max=1024),
    dict(batch=65535, n_nodes=1, n_heads=64, n_kv_heads=64, kv_max=131072),
    dict(batch=60000, n_nodes=256, n_heads=65000, n_kv_heads=1, kv_max=0),
])
def test_attention_refuses_more_tiles(lib, ctx, sizes):
    d = attention(**sizes)
    assert attend(lib, ctx, d) < 0 and b"tiles" in lib.fake_message(ctx)
    assert d.workspace_bytes == 0 and lib.fake_state().contents.launches == 0


@pytest.mark.parametrize("type", [S.BF16, S.F32])
def test_attention_room_stays_below_2_to_31(lib, ctx, type):
    # the kernels round lengths up to tiles in 32 bits
    d = attention(type=type, batch=1, n_nodes=1, n_heads=1, n_kv_heads=1, kv_max=2 ** 31 - 1024)
    assert attend(lib, ctx, d) == 0, lib.fake_message(ctx)
    for room in (2 ** 31 - 1023, 2 ** 31 - 1):
        d = attention(type=type, batch=1, n_nodes=1, n_heads=1, n_kv_heads=1, kv_max=room)
        assert attend(lib, ctx, d) < 0 and b"kv_max" in lib.fake_message(ctx)


def calls(lib, h):
    """name -> a call that launches."""
    a, v, c = attention(), S.TreeVerifyDesc(batch=2, n_nodes=3, vocab=100), S.TreeCommitDesc(
        n_tensors=1, layers=1, batch=2, n_nodes=3, n_kv_heads=1, head_dim=8, kv_max=9, lens=64, path=128, accepted=192, new_lens=256)
    for name in ("tokens", "parents", "target", "accept_u", "sample_u", "path", "accepted", "token"):
        setattr(v, name, 4096)
    c.cache[0] = c.tree[0] = 4096
    for t in (c.cache_stride[0], c.tree_stride[0]):
        t[:] = [256, 128, 64, 8]
    ref = ctypes.byref
    return {
        "attention": lambda: attend(lib, h, a),
        "mask": lambda: lib.ds_cuda_tree_mask_dev(h, 64, None, 2, 3, 64, None, None),
        "probs": lambda: lib.ds_cuda_token_probs_dev(h, S.F32, 4096, 2, 100, 100, None, 4096, None),
        "verify": lambda: lib.ds_cuda_tree_verify_dev(h, ref(v), None),
        "greedy": lambda: lib.ds_cuda_tree_verify_greedy_dev(h, 64, 64, None, 64, 2, 3, 64, 64, 64, None),
        "commit": lambda: lib.ds_cuda_tree_commit_dev(h, ref(c), None),
    }


@pytest.mark.parametrize("name", ["attention", "mask", "probs", "verify", "greedy", "commit"])
@pytest.mark.parametrize("current", [0, 1, 3])
def test_a_call_leaves_the_current_device(lib, ctx, name, current):
    f = lib.fake_state().contents
    call = calls(lib, ctx)[name]
    f.device = current
    assert call() == 0, lib.fake_message(ctx)
    assert f.launches >= 1 and f.launch_device == 1 and f.device == current
    f.error = 700  # a launch that fails
    assert call() < 0 and f.device == current


def test_the_check_leaves_the_current_device(lib, ctx):
    f = lib.fake_state().contents
    f.device = 3
    assert lib.ds_cuda_tree_attention_check(ctx, None) == 0 and f.device == 3


def test_every_stream_hears_of_a_wait_that_gave_up(lib, ctx):
    f = lib.fake_state().contents
    a, b = 0x1000, 0x2000
    check = lib.ds_cuda_tree_attention_check
    assert check(ctx, a) == 0 and check(ctx, b) == 0
    f.word = 3  # what a kernel on either stream, or on a third, leaves
    for s in (a, b, None):
        assert check(ctx, s) == -7 and b"wait" in lib.fake_message(ctx)
        assert check(ctx, s) == 0
    f.word += 1
    assert [check(ctx, s) for s in (b, b, a, a)] == [-7, 0, -7, 0]


@pytest.mark.parametrize("sixteen,eight,heads,cluster", [
    (14, 30, 14, 16), (14, 30, 15, 8), (14, 30, 30, 8), (14, 30, 31, 0),
    (0, 0, 1, 0),  # a share of a GPU that holds none at all
])
def test_clusters_are_as_many_as_the_gpu_holds_at_once(lib, sixteen, eight, heads, cluster):
    # (what a GPU holds is asked once a device: each case has its own)
    device = 10 + sixteen + heads
    h = lib.fake_new(device, 148)
    f = lib.fake_state().contents
    f.devices, f.room[16], f.room[8] = 64, sixteen, eight
    d = attention(type=S.F32, batch=1, n_nodes=1, n_heads=heads, n_kv_heads=heads, head_dim=128, kv_max=680)
    assert attend(lib, h, d) == 0, lib.fake_message(h)
    assert (f.cluster, f.launches, d.workspace_bytes > 0) == (cluster, 1 if cluster else 2, not cluster)
    lib.fake_free(h)


@pytest.mark.parametrize("type", [S.F32, S.BF16])
def test_room_alone_does_not_change_a_small_call(lib, type):
    # one stream of 10 heads and a tree of 16: tiles of 8 rows in 20 clusters of
    # 8 CTAs up to 8 tiles a CTA, then tiles of 16 rows in 10 clusters of 16
    h = lib.fake_new(40 + type, 148)
    f = lib.fake_state().contents
    f.devices, f.room[16], f.room[8] = 64, 14, 30
    for room, cluster in ((680, 8), (961, 8), (1024, 8), (4032, 8), (4096, 16)):
        d = attention(type=type, batch=1, n_nodes=16, n_heads=10, n_kv_heads=10, head_dim=128, kv_max=room)
        assert attend(lib, h, d) == 0 and f.cluster == cluster, room
    lib.fake_free(h)
