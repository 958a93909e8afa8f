"""The speculative-decoding operators against plain 64-bit forms: attention
of a tree over the cache (types, head layouts, lengths from nothing to many
tiles, ragged batches, strides, masks that leave rows empty, garbage in
unattended places, offsets past 32 bits, streams and graphs), probabilities,
verification (bit for bit, and its distribution), the greedy rule, commit,
and what each refuses.

Tolerances, from the formats: a float32 attention result differs from the
64-bit one by the scores' rounding, |s| 2^-23 with |s| below 40 here, i.e.
below 5e-6 relative; a 16-bit one by two roundings, of the weights and of
the result: 2 u with u = 2^-8 (bfloat16) or 2^-11 (float16). Probabilities:
|x| 2^-23 with |x| below 40, 5e-6."""
import numpy as np
import pytest
import torch

import spec_ref as R
from ds_ocr_b200 import _lib
from ds_ocr_b200.cuda import DsCudaError

pytestmark = pytest.mark.gpu
TOL = {"pair": 5e-6, "plane": 5e-6, "bf16": 2 * 2.0 ** -8, "f16": 2 * 2.0 ** -11}
I32 = dict(dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def spec(cuda_ctx):
    from ds_ocr_b200.speculative import Speculative
    return Speculative(cuda_ctx)


def rel(x, y):
    x, y = x.double(), y.double()
    n = float(y.norm())
    return float((x - y).norm()) / n if n else float((x - y).norm())


class Case:
    def __init__(self, kind, lens, counts, n, kv=2, group=1, hd=128, seed=0, layout="bhsd", masks="tree", pad=9,
                 garbage=True, device="cuda"):
        g = torch.Generator(device).manual_seed(seed)
        rng = np.random.default_rng(seed)
        b = len(lens)
        cap = max(lens) + pad
        qt = {"bf16": torch.bfloat16, "f16": torch.float16}.get(kind, torch.float32)

        def rnd(*s):
            return torch.randn(s, generator=g, device=device)

        def rows(r, used):
            x = rnd(b, kv, r, hd) if layout == "bhsd" else rnd(b, r, kv, hd).transpose(1, 2)
            if garbage:  # what is not in use holds NaN and infinities
                for i, u in enumerate(used):
                    x[i, :, u:] = float("nan")
                    x[i, :, u::2] = float("inf")
            if kind in ("pair", "plane"):
                return R.planes(x, kind == "pair")
            return x.to(qt)

        self.q = (2 * rnd(b, n, kv * group, hd)).to(qt)
        self.k, self.v = rows(cap, lens), rows(cap, lens)
        self.tk, self.tv = rows(n, counts), rows(n, counts)
        self.lens, self.counts = torch.tensor(lens, **I32), torch.tensor(counts, **I32)
        if masks == "tree":
            self.allowed = np.stack([R.ancestors(R.random_tree(rng, n, c), n, c) for c in counts])
        elif masks == "none":
            self.allowed = np.zeros((b, n, n), bool)
        else:
            self.allowed = rng.random((b, n, n)) < 0.4
        self.mask = R.words(self.allowed).to(device)
        self.scale = hd ** -0.5
        self.kind = kind

    def run(self, spec, **kw):
        return spec.tree_attention(self.q, self.k, self.v, self.tk, self.tv, self.lens, self.mask, self.counts, **kw)

    def want(self):
        return R.attention(self.q, self.k, self.v, self.tk, self.tv, self.lens, self.allowed, self.counts, self.scale)

    def check(self, spec):
        b, n, h, _ = self.q.shape
        lse = torch.full((b, n, h), 7.0, device="cuda")
        out = self.run(spec, lse=lse)
        o, l = self.want()
        assert torch.isfinite(out).all()
        assert rel(out, o) < TOL[self.kind], rel(out, o)
        empty = torch.isinf(l)
        assert torch.equal(torch.isneginf(lse), empty)
        assert not out[empty].any()
        if (~empty).any():
            assert float((lse[~empty].double() - l[~empty]).abs().max()) < 2e-5
        return out


KINDS = ["pair", "plane", "bf16", "f16"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,group", [(1, 1), (5, 1), (16, 1), (17, 3), (33, 2), (64, 1), (64, 8), (130, 1)])
def test_attention_sizes(spec, kind, hd, n, group):
    lens = [0, 1, 31, 64, 65, 300]
    counts = [n, max(1, n - 1), n, 1, n, max(1, n // 2)]
    Case(kind, lens, counts, n, 2, group, hd, seed=n + group).check(spec)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [127, 128, 129, 255, 1000, 4097])
def test_attention_lengths(spec, kind, length):
    Case(kind, [length], [11], 11, 3, 1, 128, seed=length).check(spec)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,group", [(33, 1), (25, 5), (16, 8), (43, 3), (64, 4), (37, 9), (200, 1)])
def test_attention_many_rows_long(spec, kind, hd, n, group):
    Case(kind, [5003, 0, 517], [n, max(1, n - 9), n], n, 2, group, hd, seed=hd + n).check(spec)


# Room for a long cache: calls that are brief by it take the kernel for few rows
ROOM = 20000


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("n,group", [(17, 3), (33, 2), (64, 1), (64, 8), (130, 1)])
def test_attention_many_rows_with_room(spec, kind, hd, layout, n, group):
    lens = [0, 1, 31, 64, 65, 300]
    counts = [n, max(1, n - 1), n, 1, 0, max(1, n // 2)]
    Case(kind, lens, counts, n, 2, group, hd, seed=n + group, pad=ROOM, layout=layout).check(spec)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("masks", ["none", "random"])
@pytest.mark.parametrize("n,group", [(40, 2), (70, 4)])
def test_attention_many_rows_masks(spec, kind, masks, n, group):
    Case(kind, [0, 40, 200], [n, n - 3, n], n, 2, group, 64, seed=5, masks=masks, pad=ROOM).check(spec)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_attention_many_rows_scales(spec, kind, scale):
    c = Case(kind, [150, 1], [50, 50], 50, 2, 2, 64, seed=21, pad=ROOM)
    c.scale = scale
    c.q = (c.q * (0.25 if scale == 3.0 else 1)).to(c.q.dtype)
    assert rel(c.run(spec, scale=scale), c.want()[0]) < TOL[kind]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [7, 14])
def test_attention_many_rows_nan_in_a_node(spec, kind, hd, group):
    c = Case(kind, [70, 3], [10, 10], 10, 2, group, hd, seed=9, pad=ROOM)
    c.tk[0, :, 7] = float("nan")
    c.tv[1, :, 8] = float("inf")
    c.allowed[:, :, 7:9] = False
    c.allowed[0, 7, 7] = c.allowed[1, 8, 8] = True
    c.mask = R.words(c.allowed).cuda()
    out, (o, _) = c.run(spec), c.want()
    assert torch.isnan(out[0, 7]).all() and not torch.isfinite(out[1, 8]).any()
    fine = torch.isfinite(o)
    assert torch.equal(torch.isfinite(out), fine)
    assert rel(out[fine], o[fine]) < TOL[kind]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n", [20, 140])
def test_attention_infinite_node_after_idle_sequences(spec, kind, n):
    # a sequence whose node holds an infinity (in its second or third tile of
    # 64 keys) after hundreds without a tree, of one empty tile each
    live = [i % 25 == 24 for i in range(1500)]
    c = Case(kind, [30 if x else 0 for x in live], [n if x else 0 for x in live], n, 8, 1, 64, seed=19, garbage=False)
    at = torch.tensor(live, device="cuda")
    c.tv[at, :, n - 2] = float("inf")
    c.allowed[:, :, n - 2] = False
    c.allowed[live, n - 2, n - 2] = True
    c.mask = R.words(c.allowed).cuda()
    out = c.run(spec)
    assert torch.isposinf(out[at, n - 2]).all()
    out[at, n - 2] = 0
    c.tv[at, :, n - 2] = 0  # (finite for the plain form; nobody else attends it)
    o = c.want()[0]
    o[at, n - 2] = 0
    assert rel(out, o) < TOL[kind]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("group", [8, 40])
def test_attention_many_rows_scores_far_apart(spec, kind, group):
    # the largest score of some rows arrives late and is far above the first
    c = Case(kind, [400, 333], [4, 4], 4, 2, group, 128, seed=10, pad=ROOM)
    q0 = c.q[0, 1, 0].float()
    c.k[0, 0, 390] = (q0 * 60 / q0.norm()).to(c.k.dtype)
    q1 = c.q[1, 2, group + 1].float()
    c.k[1, 1, 200] = (q1 * 30 / q1.norm()).to(c.k.dtype)
    assert rel(c.run(spec), c.want()[0]) < TOL[kind]


def test_attention_many_rows_repeatable_and_far(spec):
    # equal bits again, and rows 2^32 elements apart
    c = Case("f16", [150, 140], [33, 30], 33, 2, 4, 64, seed=13, pad=ROOM)
    want = c.check(spec)
    room = torch.empty((1 << 32) + 2 * (150 + ROOM) * 64, dtype=torch.float16, device="cuda")
    far = room.as_strided(c.k.shape, (1 << 32, (150 + ROOM) * 64, 64, 1))
    far.copy_(c.k)
    c.k = far
    for _ in range(5):
        assert torch.equal(c.run(spec), want)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("kind,n", [("pair", 7), ("pair", 20), ("f16", 12), ("bf16", 20), ("bf16", 50)])
def test_attention_scales(spec, kind, n, scale):
    # scores up to 60 with the largest scale: |s| 2^-23 stays below the bound
    c = Case(kind, [150, 1], [n, n], n, 2, 1, 64, seed=21)
    c.scale = scale
    c.q = (c.q * (0.25 if scale == 3.0 else 1)).to(c.q.dtype)
    out = c.run(spec, scale=scale)
    assert rel(out, c.want()[0]) < max(TOL[kind], 1e-5 if scale == 3.0 else 0)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_ragged_batch(spec, kind):
    lens = [0, 2000, 3, 700, 64, 0, 1, 128, 129, 513, 1500, 17]
    counts = [3, 8, 0, 1, 8, 0, 7, 8, 2, 5, 8, 4]
    Case(kind, lens, counts, 8, 5, 2, 128, seed=3, layout="bshd").check(spec)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("masks", ["none", "random"])
def test_attention_masks(spec, kind, masks):
    # no mask bit set: rows with no cache are empty, the others see the cache alone
    Case(kind, [0, 40, 200], [12, 9, 12], 12, 2, 2, 64, seed=5, masks=masks).check(spec)


def test_attention_many_sequences(spec):
    lens = [(i * 37) % 90 for i in range(300)]
    Case("bf16", lens, [1 + i % 3 for i in range(300)], 3, 2, 1, 64, seed=6).check(spec)


@pytest.mark.parametrize("kind", ["pair", "bf16"])
def test_attention_without_cache_rows(spec, kind):
    c = Case(kind, [0, 0], [6, 4], 6, 2, 1, 128, seed=8, pad=0)
    assert (c.k[0] if isinstance(c.k, tuple) else c.k).shape[2] == 0
    c.check(spec)


@pytest.mark.parametrize("group", [1, 2, 7])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_nan_in_a_node_reaches_only_its_readers(spec, kind, group):
    c = Case(kind, [70, 3], [10, 10], 10, 2, group, 128, seed=9)
    ks, vs = (c.tk, c.tv) if isinstance(c.tk, tuple) else ((c.tk,), (c.tv,))
    ks[0][0, :, 7] = float("nan")
    vs[0][1, :, 8] = float("inf")
    c.allowed[:, :, 7:9] = False
    c.allowed[0, 7, 7] = c.allowed[1, 8, 8] = True
    c.mask = R.words(c.allowed).cuda()
    out, (o, _) = c.run(spec), c.want()
    assert torch.isnan(out[0, 7]).all() and not torch.isfinite(out[1, 8]).any()
    fine = torch.isfinite(o)
    assert torch.equal(torch.isfinite(out), fine)
    assert rel(out[fine], o[fine]) < TOL[kind]


@pytest.mark.parametrize("kind", KINDS)
def test_attention_scores_far_apart(spec, kind):
    # the largest score of a row arrives late and is far above the first ones,
    # and one query's scores are minus infinity or overflow nothing
    c = Case(kind, [400, 333], [4, 4], 4, 2, 1, 128, seed=10)
    k = c.k if isinstance(c.k, tuple) else (c.k,)
    q0 = c.q[0, 1, 0].float()
    k[0][0, 0, 390] = (q0 * 60 / q0.norm()).to(k[0].dtype)
    if len(k) > 1:
        k[1][0, 0, 390] = 0
    out, (o, _) = c.run(spec), c.want()
    # scores up to 120: |s| 2^-23 allows 1.5e-5 there
    assert rel(out, o) < max(TOL[kind], 1.5e-5)


@pytest.mark.parametrize("kind,tol", [("f16", 2.0 ** -6), ("bf16", TOL["bf16"])])
@pytest.mark.parametrize("group", [4, 40])
def test_attention_small_weights_are_not_lost(spec, kind, tol, group):
    # Eight keys of weight 1 and V 0 at the start, and 2^15 of weight 2^-25.03
    # (below half of float16's smallest value) and V 1, which make all of the
    # result. Enough sequences for some to be one CTA's alone; they share one
    # cache. float16: a weight's error is 2^-32, 2^-6.97 of these, and the
    # sums' and the result's (2^-10 each) come on top.
    keys, b, hd = 1 << 15, 4 * torch.cuda.get_device_properties(0).multi_processor_count + 8, 64
    t = torch.float16 if kind == "f16" else torch.bfloat16
    k = torch.zeros(1, 1, keys, hd, dtype=t, device="cuda")
    v = torch.ones_like(k)
    k[:, :, :128:16, 0], v[:, :, :128:16] = 16, 0
    q = torch.zeros(b, 1, group, hd, dtype=t, device="cuda")
    q[..., 0] = 1
    node = torch.zeros(b, 1, 1, hd, dtype=t, device="cuda")
    out = spec.tree_attention(q, k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), node, node, torch.full((b,), keys, **I32),
                              torch.zeros(b, 1, 1, dtype=torch.long, device="cuda"), scale=25.03 * np.log(2) / 16)
    x = (keys - 8) * 2.0 ** -25.03
    assert float((out.double() * (8 + x) / x - 1).abs().max()) < tol


def test_attention_lowest_values(spec):
    # keys so large that scores reach the float32 range's end: minus infinity
    # for one query (it attends nothing), plus infinity (NaN) for another
    c = Case("bf16", [20], [2], 2, 1, 1, 64, seed=11, masks="none")
    c.k[:] = 3e38
    c.q[0, 0], c.q[0, 1] = -3e38, 3e38
    out = c.run(spec)
    assert not out[0, 0].any() and torch.isnan(out[0, 1]).all()


def test_attention_strides_and_given_out(spec):
    c = Case("bf16", [77, 130], [7, 7], 7, 3, 2, 64, seed=12, layout="bshd")
    big = torch.zeros(2, 6, 9, 80, dtype=torch.bfloat16, device="cuda")
    out = big.transpose(1, 2)[:, 1:8, :, :64]
    got = c.run(spec, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert rel(out, c.want()[0]) < TOL["bf16"]
    assert not big[:, :, :, 64:].any() and not big[:, :, 0].any() and not big[:, :, 8].any()
    qb = torch.zeros(2, 7, 6, 192, dtype=torch.bfloat16, device="cuda")
    qb[..., 64:128] = c.q
    c.q = qb[..., 64:128]
    assert torch.equal(c.run(spec), out)


def test_attention_offsets_past_32_bits(spec):
    # the second sequence's rows start 2^32 elements after the first's
    c = Case("f16", [150, 140], [5, 5], 5, 2, 1, 64, seed=13)
    room = torch.empty((1 << 32) + 2 * 160 * 64, dtype=torch.float16, device="cuda")
    far = room.as_strided((2, 2, 159, 64), (1 << 32, 160 * 64, 64, 1))
    far.copy_(c.k)
    c.k = far
    c.check(spec)
    far.copy_(c.v)
    c.k, c.v = c.v.clone(), far
    c.check(spec)
    # and a row stride that takes the last rows past 2^31 elements
    c = Case("f16", [200], [5], 5, 1, 1, 64, seed=14)
    rows = room.as_strided((1, 1, 209, 64), (0, 0, 1 << 24, 1))
    rows.copy_(c.k)
    c.k = rows
    c.check(spec)


def test_attention_of_many_sequences_with_room(spec):
    # 256 sequences, 64 heads on 8, trees of 64, room for 65536 rows (one
    # cache for all): as four calls of 64 sequences give it
    g = torch.Generator("cuda").manual_seed(23)
    b, n, kv, hd, cap = 256, 64, 8, 64, 65536

    def rnd(*s):
        return torch.randn(s, generator=g, device="cuda", dtype=torch.bfloat16)

    q, k, v, tk, tv = rnd(b, n, 64, hd), rnd(1, kv, cap, hd), rnd(1, kv, cap, hd), rnd(b, kv, n, hd), rnd(b, kv, n, hd)
    lens = torch.randint(0, 300, (b,), generator=g, device="cuda").int()
    lens[77] = cap
    mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (b, n, 1), generator=g, device="cuda")
    parts = [x.split(64) for x in (q, tk, tv, lens, mask)]
    want = torch.cat([spec.tree_attention(x, k.expand(64, -1, -1, -1), v.expand(64, -1, -1, -1), *r) for x, *r in zip(*parts)])
    got = spec.tree_attention(q, k.expand(b, -1, -1, -1), v.expand(b, -1, -1, -1), tk, tv, lens, mask)
    # (other cuts: each side within the tolerance of the exact one)
    assert torch.isfinite(got).all() and rel(got, want) < 2 * TOL["bf16"]


def test_attention_is_repeatable_on_streams_and_in_graphs(spec):
    cs = [Case("pair", [900, 40], [16, 9], 16, 4, 1, 128, seed=s) for s in (15, 16)]
    want = [c.run(spec) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.run(spec))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        assert all(torch.equal(w, x) for x in many)
    c = cs[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.run(spec)
    c.lens.copy_(torch.tensor([13, 911], **I32)[:2].clamp(max=909))
    for t in (*c.k, *c.v):
        t.nan_to_num_(0.5, 0.5, 0.5)
    g.replay()
    torch.cuda.synchronize()
    assert rel(out, c.want()[0]) < TOL["pair"]


@pytest.mark.parametrize("kind,n,group", [("pair", 16, 1), ("bf16", 12, 1), ("bf16", 20, 4), ("f16", 60, 4)])
def test_attention_with_room_on_streams_and_in_graphs(spec, kind, n, group):
    # the same for calls that cut a list of tiles and join the parts in a second
    # kernel, on mma.sync and on tcgen05; replays with other lengths, so that
    # the items are cut elsewhere
    cs = [Case(kind, [900, 40, 0], [n, n // 2, n], n, 4, group, 64, seed=s, pad=ROOM, garbage=False) for s in (25, 26)]
    want = [c.run(spec) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.run(spec))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        assert all(torch.equal(w, x) for x in many)
    c = cs[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = c.run(spec)
    for lens, counts in (([5, 2000, 64], [1, n, 0]), ([4097, 1, 127], [n, n, 3])):
        c.lens.copy_(torch.tensor(lens, **I32))
        c.counts.copy_(torch.tensor(counts, **I32))
        g.replay()
        torch.cuda.synchronize()
        assert rel(out, c.want()[0]) < TOL[kind]
    spec.check()


@pytest.mark.parametrize("kind", ["pair", "plane"])
def test_attention_of_sixteen_nodes_is_cheaper_than_twice_eight(spec, kind):
    # both read the cache once: 1.2 times the time of eight (one plane 1.6), 1.8 where the kernel spills
    times = []
    for n in (8, 16):
        c = Case(kind, [1325] * 64, [n] * 64, n, 10, 1, 128, seed=n, garbage=False)
        c.run(spec)
        e = [torch.cuda.Event(enable_timing=True) for _ in range(11)]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(5):
                c.run(spec)
        for x in e:
            g.replay()
            x.record()
        torch.cuda.synchronize()
        times.append(min(x.elapsed_time(y) for x, y in zip(e, e[1:])))
    assert times[1] < 1.75 * times[0], times


def test_attention_clamps_lengths_and_counts(spec):
    c = Case("bf16", [30, 30], [4, 4], 4, 2, 1, 64, seed=17, pad=0, garbage=False)
    want = c.run(spec)
    c.lens.fill_(1 << 30)
    c.counts.fill_(1 << 30)
    assert torch.equal(c.run(spec), want)
    c.lens.fill_(-5)
    c.counts.fill_(-5)
    assert not c.run(spec).any()


def test_attention_planes_whose_unused_strides_differ(spec):
    # one sequence, one KV head: those dimensions' strides mean nothing
    c = Case("pair", [30], [4], 4, 1, 2, 64, seed=31)
    want = c.run(spec)

    def odd(planes):
        hi, lo = planes
        return hi, lo.as_strided(lo.shape, (7, 13, *lo.stride()[2:]))

    c.k, c.v, c.tk, c.tv = map(odd, (c.k, c.v, c.tk, c.tv))
    assert torch.equal(c.run(spec), want)
    c = Case("pair", [30], [4], 4, 2, 2, 64, seed=31)
    c.k = c.k[0], c.k[1].as_strided(c.k[1].shape, (1, 64, 128, 1))  # the heads side by side
    with pytest.raises(ValueError, match="strides"):
        c.run(spec)


def test_attention_refusals(spec):
    c = Case("bf16", [30], [4], 4, 2, 2, 64, seed=18)
    ok = (c.q, c.k, c.v, c.tk, c.tv, c.lens, c.mask)

    def bad(i, t, err=ValueError):
        with pytest.raises(err):
            spec.tree_attention(*ok[:i], t, *ok[i + 1:])

    bad(0, c.q.double())
    bad(0, c.q.cpu())
    bad(0, c.q.half())                            # cache of another type than its queries'
    bad(0, c.q[:, :, :3], DsCudaError)            # 3 heads on 2 key heads
    bad(1, c.k.transpose(2, 3))
    bad(1, (c.k, c.k))                            # a second plane with 16-bit queries
    bad(2, c.v[:, :, 1:])
    bad(3, c.tk[:, :, :3])
    bad(5, c.lens.long())
    bad(6, c.mask.int())
    with pytest.raises(ValueError):
        spec.tree_attention(*ok, counts=c.lens.float())
    odd = torch.empty(1, 2, 40, 65, dtype=torch.bfloat16, device="cuda")[..., :64]
    with pytest.raises(DsCudaError, match="16 bytes"):
        spec.tree_attention(c.q, odd[:, :, :39], c.v, *ok[3:])
    wide = Case("bf16", [3], [2], 2, 1, 1, 96, seed=1)
    with pytest.raises(DsCudaError, match="head_dim"):
        wide.run(spec)
    with pytest.raises(DsCudaError, match="n_nodes"):
        Case("bf16", [3], [257], 257, 1, 1, 64, seed=1).run(spec)
    assert spec.tree_attention(*(t[:0] for t in ok)).shape == (0, 4, 4, 64)


def test_tree_mask(spec):
    rng = np.random.default_rng(1)
    for n in (1, 2, 63, 64, 65, 200, 256):
        counts = [n, max(1, n - 3), 1, 0]
        par = [R.random_tree(rng, n, c) for c in counts]
        mask, depth = spec.tree_mask(torch.tensor(par, **I32), torch.tensor(counts, **I32))
        want = np.stack([R.ancestors(p, n, c) for p, c in zip(par, counts)])
        assert torch.equal(mask.cpu(), R.words(want))
        assert np.array_equal(depth.cpu().numpy(), np.maximum(want.sum(-1) - 1, 0))
    # parents out of order, of themselves or out of range make roots
    mask, depth = spec.tree_mask(torch.tensor([[5, 1, 99, -7, 0]], **I32))
    assert mask.flatten().tolist() == [1, 2, 4, 8, 17] and depth.flatten().tolist() == [0, 0, 0, 0, 1]
    with pytest.raises(DsCudaError):
        spec.tree_mask(torch.zeros(1, 257, **I32))


# ---- probabilities ---------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 1000), (5, 4097), (2, 32001), (3, 129280), (1, 262145),
                                        (1, 600001), (300, 50)])
def test_token_probs(spec, dtype, rows, vocab):
    g = torch.Generator("cuda").manual_seed(vocab)
    x = (4 * torch.randn(rows, vocab + 3, generator=g, device="cuda")).to(dtype)[:, 1:vocab + 1]  # strided, unaligned
    t = 0.4 + torch.rand(rows, generator=g, device="cuda")
    want = torch.softmax(x.double() / t.double()[:, None], -1)
    assert rel(spec.token_probs(x, t), want) < 5e-6
    assert rel(spec.token_probs(x.contiguous()), torch.softmax(x.double(), -1)) < 5e-6


def test_token_probs_edges(spec):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(8, 5000, device="cuda")
    x[0, 17:] = -inf
    x[1] = -inf
    x[2, 100] = nan
    x[3, 4999] = inf
    x[4] = 2.5
    x[5, 7] = x[5, 4000] = 50.0
    x[6] = -3.4e38                          # the type's lowest value everywhere
    x[7, :4999] = -3.4e38
    t = torch.tensor([1, 1, 1, 1, 0, 0, 1, 1.0], device="cuda")
    p = spec.token_probs(x, t)
    assert rel(p[0], torch.softmax(x[0].double(), 0)) < 5e-6 and not p[0, 17:].any()
    assert not p[1].any()
    assert torch.isnan(p[2]).all() and torch.isnan(p[3]).all()
    assert p[4, 0] == 1 and p[4].sum() == 1
    assert p[5, 7] == 1 and p[5].sum() == 1
    assert float((p[6] * 5000 - 1).abs().max()) < 1e-5
    assert p[7, 4999] == 1 and p[7].sum() == 1
    y = torch.full((1, 3000), 1.0, device="cuda")
    for temp in (-1.0, 0.0, 1e-30):
        y[0, 1234] = 2.0
        p = spec.token_probs(y, torch.tensor([temp], device="cuda"))
        assert p[0, 1234] == 1 and p.sum() == 1, temp
    assert spec.token_probs(y[:0]).shape == (0, 3000)
    assert torch.isnan(spec.token_probs(y, torch.tensor([nan], device="cuda"))).all()


def test_token_probs_of_an_infinite_temperature(spec):
    x = torch.randn(2, 5000, device="cuda")
    x[1, ::2] = -float("inf")
    p = spec.token_probs(x, torch.full((2,), float("inf"), device="cuda"))
    assert float((p[0] * 5000 - 1).abs().max()) < 1e-5
    assert not p[1, ::2].any() and float((p[1, 1::2] * 2500 - 1).abs().max()) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [64, 70001])
def test_token_probs_of_the_largest_logits(spec, dtype, vocab):
    # logits over the type's whole range, whose differences pass it, at
    # temperatures as large: -infinity alone is excluded by an infinite one
    top, inf = torch.finfo(dtype).max, float("inf")
    x = torch.linspace(-1, 1, vocab, device="cuda").mul(top).to(dtype).repeat(4, 1)
    x[:, 5] = -inf
    x[:, 6] = top
    t = torch.tensor([inf, 3e38, 1e38, 2e37], device="cuda")
    p = spec.token_probs(x, t)
    y = x.double() / t.double()[:, None]
    y[0] = torch.where(torch.isinf(x[0]), -inf, 0.0)
    assert rel(p, torch.softmax(y, -1)) < 5e-6
    assert not p[:, 5].any()
    assert float((p[0, 6:] * (vocab - 1) - 1).abs().max()) < 5e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_probs_of_the_largest_vocabulary(spec, dtype):
    x = (2 * torch.randn(2, 917504, device="cuda")).to(dtype)
    assert rel(spec.token_probs(x), torch.softmax(x.double(), -1)) < 5e-6
    with pytest.raises(DsCudaError):
        spec.token_probs(torch.zeros(1, 917505, dtype=dtype, device="cuda"))


def test_token_probs_refusals(spec):
    x = torch.zeros(2, 8, device="cuda")
    for bad in (x.double(), x.T, x.cpu()):
        with pytest.raises(ValueError):
            spec.token_probs(bad)
    with pytest.raises(ValueError):
        spec.token_probs(x, torch.ones(3, device="cuda"))
    with pytest.raises(DsCudaError):
        spec.token_probs(torch.zeros(2, 0, device="cuda"))


# ---- verification ----------------------------------------------------------
def sampled(b, n, vocab, seed, width=3, spread=2.0, noise=1.0, certain=False):
    rng = np.random.default_rng(seed)
    f = np.float32

    def soft(x):
        e = np.exp(x - x.max(-1, keepdims=True))
        return (e / e.sum(-1, keepdims=True)).astype(f)

    x = rng.normal(0, spread, (b, n, vocab))
    target, draft = soft(x), soft(x + rng.normal(0, noise, x.shape))
    counts = [max(1, n - i % 3) for i in range(b)]
    parents = np.array([R.random_tree(rng, n, c, width) for c in counts], np.int32)
    tokens = np.zeros((b, n), np.int32)
    for i in range(b):
        for j in range(1, counts[i]):
            cdf = np.cumsum(draft[i, parents[i, j]].astype(np.float64))
            tokens[i, j] = min(vocab - 1, np.searchsorted(cdf, rng.random() * cdf[-1]))
    ua = (rng.integers(0, 1 << 24, (b, n)) / 2.0 ** 24).astype(f)
    us = (rng.integers(0, 1 << 24, b) / 2.0 ** 24).astype(f)
    return dict(tokens=tokens, parents=parents, target=target, draft=None if certain else draft, accept_u=ua,
                sample_u=us, counts=np.array(counts, np.int32))


def on_gpu(s):
    return {k: None if v is None else torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in s.items()}


def check_verify(spec, s):
    b, n = s["tokens"].shape
    path, acc, tok = (t.cpu().numpy() for t in spec.verify(**on_gpu(s)))
    for i in range(b):
        p, t = R.verify(s["tokens"][i], s["parents"][i], s["counts"][i], s["target"][i],
                        None if s["draft"] is None else s["draft"][i], s["accept_u"][i], s["sample_u"][i])
        assert path[i].tolist() == p + [-1] * (n - len(p)), i
        assert acc[i] == len(p) - 1 and tok[i] == t, i
    return path, acc, tok


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("b,n,vocab", [(1, 1, 50), (4, 2, 1), (40, 9, 33), (8, 30, 1000), (6, 17, 4099), (3, 8, 32001),
                                       (2, 12, 129280), (2, 5, 262144), (1, 256, 300), (200, 6, 12)])
def test_verify_bit_for_bit(spec, certain, b, n, vocab):
    s = sampled(b, n, vocab, b * 1000 + n, certain=certain)
    _, acc, _ = check_verify(spec, s)
    if not certain and b >= 40:
        assert acc.max() > 1 and acc.min() == 0


def test_verify_many_rejections_at_one_node(spec):
    s = sampled(4, 40, 2000, 5, spread=1.0, noise=3.0)
    s["parents"][:, 1:] = 0
    s["accept_u"][:] = 0.99999
    s["counts"][:] = 40
    check_verify(spec, s)
    s["draft"] = None
    check_verify(spec, s)


def test_verify_chains_of_one_token_after_a_rejection(spec):
    # certain drafts: at every level a child is rejected, its sibling accepted,
    # and the sibling's first child, rejected, has the sibling's own token, so
    # that the rejected tokens of a node must not be taken for those of the next
    b, vocab, levels = 256, 12, 40
    n = 1 + 2 * levels
    rng = np.random.default_rng(15)
    s = sampled(b, n, vocab, 15, certain=True)
    s["counts"][:] = n
    up = np.arange(n)
    s["parents"][:] = np.where(up == 0, -1, 2 * ((up - 1) // 2))
    s["tokens"][:, 0] = 0
    for level in range(levels):
        first, second = 1 + 2 * level, 2 + 2 * level
        s["tokens"][:, first] = s["tokens"][:, first - 1]
        s["tokens"][:, second] = (s["tokens"][:, first] + 1 + rng.integers(0, vocab - 1, b)) % vocab
        s["accept_u"][:, first], s["accept_u"][:, second] = 1 - 2.0 ** -24, 0
    want = check_verify(spec, s)
    assert (want[1] == levels).all()
    g = on_gpu(s)
    for _ in range(20):
        assert all(np.array_equal(x, y.cpu().numpy()) for x, y in zip(want, spec.verify(**g)))
    s["accept_u"][:] = (rng.integers(0, 1 << 24, (b, n)) / 2.0 ** 24).astype(np.float32) * np.float32(0.2)
    check_verify(spec, s)


def test_verify_edges(spec):
    n, vocab = 4, 700
    s = sampled(12, n, vocab, 9)
    s["counts"][:] = n
    s["parents"][:] = [-1, 0, 0, 0]
    s["tokens"][0] = [0, -1, vocab, 1 << 30]            # outside the vocabulary
    s["target"][1] = 0                                   # no mass anywhere: -1
    s["target"][2] = np.nan
    s["target"][3] = s["draft"][3]                       # the same: every draft is accepted
    s["target"][4, 0] = s["draft"][4, 0] * np.float32(0.5)  # nothing is left after a rejection
    s["accept_u"][4] = 0.75
    s["sample_u"][5], s["sample_u"][6] = 0.0, 1 - 2.0 ** -24
    s["target"][7, 0] = 0
    s["target"][7, 0, 5] = 1                             # one token has all the mass
    s["accept_u"][8] = 0
    s["target"][9, 0] = 1.0                              # not normalised: still a valid walk
    s["target"][10, 0, ::3] = np.inf
    s["target"][11, 0] = -1.0
    path, acc, tok = check_verify(spec, s)
    assert acc[0] == 0 and tok[1] == -1 and tok[2] == -1 and acc[3] >= 1 and tok[11] == -1
    for c in (0, 1, -3):
        s["counts"][:] = c
        path, acc, tok = (t.cpu().numpy() for t in spec.verify(**on_gpu(s)))
        assert (path[:, 0] == 0).all() and (path[:, 1:] == -1).all() and (acc == 0).all()


def test_verify_tokens_follow_the_target(spec):
    # whatever the drafts, the first token after the root has the target's
    # distribution: chi-square over 8 tokens below its 1e-6 quantile (7
    # degrees of freedom, 41)
    rng = np.random.default_rng(11)
    b, n, vocab = 40000, 4, 8
    p = rng.dirichlet(np.ones(vocab)).astype(np.float32)
    for certain in (False, True):
        q = rng.dirichlet(np.ones(vocab)).astype(np.float32)
        tokens = np.zeros((b, n), np.int32)
        tokens[:, 1:] = rng.choice(vocab, (b, n - 1), p=q.astype(np.float64) / q.astype(np.float64).sum())
        s = dict(tokens=tokens, parents=np.tile(np.array([-1, 0, 0, 0], np.int32), (b, 1)),
                 target=np.tile(p, (b, n, 1)), draft=None if certain else np.tile(q, (b, n, 1)),
                 accept_u=rng.random((b, n)).astype(np.float32), sample_u=rng.random(b).astype(np.float32),
                 counts=np.full(b, n, np.int32))
        s["accept_u"] = np.minimum(s["accept_u"], np.float32(1 - 2.0 ** -24))
        s["sample_u"] = np.minimum(s["sample_u"], np.float32(1 - 2.0 ** -24))
        path, acc, tok = (t.cpu().numpy() for t in spec.verify(**on_gpu(s)))
        first = np.where(acc > 0, tokens[np.arange(b), np.maximum(path[:, 1], 0)], tok)
        got = np.bincount(first, minlength=vocab)
        want = p.astype(np.float64) / p.astype(np.float64).sum() * b
        assert ((got - want) ** 2 / want).sum() < 41


def test_verify_strides(spec):
    s = sampled(3, 5, 999, 12)
    g = on_gpu(s)
    want = spec.verify(**g)
    for name in ("target", "draft"):
        room = torch.full((5, 3, 1007), float("nan"), device="cuda")
        room[:, :, 3:1002] = g[name].transpose(0, 1)
        g[name] = room[:, :, 3:1002].transpose(0, 1)
    for x, y in zip(want, spec.verify(**g)):
        assert torch.equal(x, y)


def test_verify_refusals(spec):
    g = on_gpu(sampled(2, 3, 20, 13))
    for name, t in (("tokens", g["tokens"].long()), ("parents", g["parents"][:1]), ("target", g["target"].half()),
                    ("target", g["target"][:, :, 0]), ("draft", g["draft"][:, :2]), ("accept_u", g["accept_u"].cpu()),
                    ("sample_u", g["sample_u"][:1]), ("counts", g["counts"].long())):
        with pytest.raises(ValueError):
            spec.verify(**{**g, name: t})
    with pytest.raises(DsCudaError, match="vocab"):
        spec.verify(g["tokens"][:, :1].contiguous(), g["parents"][:, :1].contiguous(),
                    torch.zeros(2, 1, (1 << 18) + 1, device="cuda"), None, g["accept_u"][:, :1].contiguous(),
                    g["sample_u"])


def test_verify_greedy(spec):
    rng = np.random.default_rng(14)
    b, n = 70, 21
    counts = rng.integers(1, n + 1, b).astype(np.int32)
    parents = np.array([R.random_tree(rng, n, c) for c in counts], np.int32)
    tokens, want = rng.integers(0, 2, (b, n)).astype(np.int32), rng.integers(0, 2, (b, n)).astype(np.int32)
    path, acc, tok = (t.cpu().numpy() for t in spec.verify_greedy(*(torch.from_numpy(x).cuda() for x in (tokens, parents, want, counts))))
    for i in range(b):
        cur, p = 0, [0]
        for c in range(1, counts[i]):
            if parents[i, c] == cur and tokens[i, c] == want[i, cur]:
                cur = c
                p.append(c)
        assert path[i].tolist() == p + [-1] * (n - len(p)) and acc[i] == len(p) - 1 and tok[i] == want[i, cur]
    with pytest.raises(ValueError):
        spec.verify_greedy(torch.zeros(2, 3, **I32), torch.zeros(2, 3, **I32), torch.zeros(2, 4, **I32))


# ---- commit ----------------------------------------------------------------
@pytest.mark.parametrize("n_tensors", [2, 4])
@pytest.mark.parametrize("hd,n", [(64, 5), (128, 33), (8, 256), (40, 1)])
def test_commit(spec, n_tensors, hd, n):
    rng = np.random.default_rng(n)
    layers, b, kv, cap = 3, 5, 2, 40
    lens = np.array([0, 10, cap - 2, cap, 7], np.int32)
    acc = np.array([min(n - 1, a) for a in (4, 0, 30, 3, 100)], np.int32)
    path = np.full((b, n), -1, np.int32)
    for i, a in enumerate(acc):
        path[i, 0] = 0
        path[i, 1:a + 1] = 1 + np.sort(rng.permutation(n - 1)[:a])
    caches = [torch.randn(layers, b, cap, kv, hd, device="cuda").bfloat16().transpose(2, 3) for _ in range(n_tensors)]
    trees = [torch.randn(layers, b, kv, n, hd, device="cuda").bfloat16() for _ in range(n_tensors)]
    want = [c.clone() for c in caches]
    new = lens.copy()
    for i in range(b):
        for j in range(acc[i] + 1):
            if lens[i] + j < cap:
                for w, t in zip(want, trees):
                    w[:, i, :, lens[i] + j] = t[:, i, :, path[i, j]]
        new[i] = min(cap, lens[i] + acc[i] + 1)
    got = spec.commit(caches, trees, *(torch.from_numpy(x).cuda() for x in (lens, path, acc)))
    assert got.cpu().numpy().tolist() == new.tolist()
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_commit_ignores_bad_indices(spec):
    c = torch.zeros(1, 2, 1, 8, 8, dtype=torch.float16, device="cuda")
    t = torch.ones(1, 2, 1, 3, 8, dtype=torch.float16, device="cuda")
    path = torch.tensor([[0, 99, 2], [-4, 1, 1 << 30]], **I32)
    new = spec.commit([c], [t], torch.tensor([2, -9], **I32), path, torch.tensor([1000, 2], **I32))
    assert new.tolist() == [5, 3]
    assert c[0, 0, 0, :, 0].tolist() == [0, 0, 1, 0, 1, 0, 0, 0] and c[0, 1, 0, :, 0].tolist() == [0, 1, 0, 0, 0, 0, 0, 0]


def test_commit_refusals(spec):
    c = torch.zeros(1, 2, 1, 8, 16, dtype=torch.float16, device="cuda")
    t = torch.ones(1, 2, 1, 3, 16, dtype=torch.float16, device="cuda")
    ok = (torch.zeros(2, **I32), torch.zeros(2, 3, **I32), torch.zeros(2, **I32))
    for args in (([], [], *ok), ([c] * 9, [t] * 9, *ok), ([c], [t, t], *ok), ([c.float()], [t.float()], *ok),
                 ([c], [t.bfloat16()], *ok), ([c], [t[:, :1]], *ok), ([c], [t], ok[0].long(), *ok[1:])):
        with pytest.raises(ValueError):
            spec.commit(*args)
    with pytest.raises(DsCudaError):
        spec.commit([c[..., 4:12]], [t[..., :8]], *ok)
    with pytest.raises(DsCudaError):
        spec.commit([c[..., :4]], [t[..., :4]], *ok)


def test_a_step_on_streams_and_in_a_graph(spec):
    # probabilities, verification and commit as one captured sequence, replayed
    # on other inputs, and on two streams at once
    rng = np.random.default_rng(27)
    b, n, vocab, cap = 5, 9, 3001, 40

    def inputs():
        s = sampled(b, n, vocab, int(rng.integers(1 << 30)), certain=True)
        s["logits"] = rng.normal(0, 2, (b * n, vocab)).astype(np.float32)
        s["lens"] = rng.integers(0, cap, b).astype(np.int32)
        del s["target"], s["draft"]
        return s

    def state():
        g = on_gpu(inputs())
        g["temperature"] = torch.full((b * n,), 0.7, device="cuda")
        g["cache"] = torch.zeros(2, b, 2, cap, 8, dtype=torch.bfloat16, device="cuda")
        g["tree"] = torch.randn(2, b, 2, n, 8, device="cuda").bfloat16()
        return g

    def step(g):
        p = spec.token_probs(g["logits"], g["temperature"]).view(b, n, vocab)
        path, acc, tok = spec.verify(g["tokens"], g["parents"], p, None, g["accept_u"], g["sample_u"], g["counts"])
        return p, path, acc, tok, spec.commit([g["cache"]], [g["tree"]], g["lens"], path, acc), g["cache"]

    def check(g, got):
        p, path, acc, tok, lens, cache = (t.float().cpu().numpy() if t.dtype == torch.bfloat16 else t.cpu().numpy() for t in got)
        h = {k: v.float().cpu().numpy() if v.dtype == torch.bfloat16 else v.cpu().numpy() for k, v in g.items()}
        want = np.zeros_like(cache)
        for i in range(b):
            w, t = R.verify(h["tokens"][i], h["parents"][i], h["counts"][i], p[i], None, h["accept_u"][i], h["sample_u"][i])
            assert path[i].tolist() == w + [-1] * (n - len(w)) and acc[i] == len(w) - 1 and tok[i] == t
            m = min(len(w), cap - h["lens"][i])
            want[:, i, :, h["lens"][i]:h["lens"][i] + m] = h["tree"][:, i][:, :, w[:m]]
            assert lens[i] == h["lens"][i] + m
        assert np.array_equal(cache, want)

    g = state()
    check(g, step(g))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(g)
    for _ in range(3):
        for k, v in state().items():
            g[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        check(g, got)
    gs, streams = [state() for _ in range(8)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i, g in enumerate(gs):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(step(g))
    torch.cuda.synchronize()
    for g, o in zip(gs, outs):
        check(g, o)


def test_sizes_past_32_bits_are_refused(spec):
    # sizes whose low 32 bits alone would be taken for small ones (views of one row)
    far = (1 << 32) + 4
    with pytest.raises(ValueError, match="rows"):
        spec.token_probs(torch.zeros(1, 1, device="cuda").expand(far, 1))
    c = Case("bf16", [3], [2], 2, 1, 1, 64, seed=1)
    k = c.k[:, :, :1].expand(-1, -1, far, -1)
    with pytest.raises(ValueError, match="kv_max"):
        spec.tree_attention(c.q, k, k, c.tk, c.tv, c.lens, c.mask)
    t, ints = torch.zeros(1, 1, 1, 1, 8, dtype=torch.float16, device="cuda"), torch.zeros(1, **I32)
    with pytest.raises(ValueError, match="kv_max"):
        spec.commit([t.expand(-1, -1, -1, far, -1)], [t], ints, ints[None], ints)


def test_c_abi_refusals(cuda_ctx):
    lib, h = _lib.load(), cuda_ctx.h
    assert lib.ds_cuda_tree_attention_dev(h, None, None) < 0
    assert lib.ds_cuda_tree_attention_workspace(h, None) == 0
    assert lib.ds_cuda_tree_verify_dev(h, None, None) < 0
    assert lib.ds_cuda_tree_commit_dev(h, None, None) < 0
    assert lib.ds_cuda_token_probs_dev(h, 9, None, 1, 1, 1, None, None, None) < 0
    assert lib.ds_cuda_tree_mask_dev(h, None, None, 1, 1, None, None, None) < 0
    assert lib.ds_cuda_tree_verify_greedy_dev(h, None, None, None, None, 1, 1, None, None, None, None) < 0
