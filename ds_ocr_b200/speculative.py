"""Speculative decoding on the GPU: several drafted tokens a step, arranged
as a tree, through the ds_cuda C ABI (the ds_cuda_tree_* entry points and
ds_cuda_token_probs_dev). The reference decodes one token a step and has no
counterpart.

A step of one decode loop, for `batch` sequences with trees of n_nodes nodes
(node 0 is the last accepted token, a node's parent has a smaller index):

    mask, depth = spec.tree_mask(parents)            # who attends whom, positions
    ...the layers: QKV of the nodes, then
    o = spec.tree_attention(q, k, v, tree_k, tree_v, lens, mask)
    ...LM head
    p = spec.token_probs(logits, temperature)
    path, accepted, token = spec.verify(tokens, parents, p, draft_p, accept_u, sample_u)
    lens = spec.commit(caches, trees, lens, path, accepted)

Tensors are torch CUDA tensors on the context's device; the work is enqueued
on torch's current stream and outputs are allocated there, so a tensor made
on another stream needs the usual event or record_stream. Nothing
synchronises and nothing is kept between calls.
"""
import ctypes
import struct

from .cuda import Context

BF16, F16, F32 = 0, 1, 2
MAX_NODES = 256

_i64, _int, _ptr = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p


class TreeAttentionDesc(ctypes.Structure):
    """ds_cuda_tree_attention_t."""
    _fields_ = [("type", _int), ("batch", _int), ("n_nodes", _int), ("n_heads", _int), ("n_kv_heads", _int),
                ("head_dim", _int), ("kv_max", _int), ("scale", ctypes.c_float), ("q", _ptr), ("q_stride", _i64 * 3),
                ("k", _ptr), ("k_lo", _ptr), ("k_stride", _i64 * 3), ("v", _ptr), ("v_lo", _ptr),
                ("v_stride", _i64 * 3), ("tree_k", _ptr), ("tree_k_lo", _ptr), ("tree_k_stride", _i64 * 3),
                ("tree_v", _ptr), ("tree_v_lo", _ptr), ("tree_v_stride", _i64 * 3), ("lens", _ptr), ("nodes", _ptr),
                ("mask", _ptr), ("out", _ptr), ("out_stride", _i64 * 3), ("lse", _ptr), ("workspace", _ptr),
                ("workspace_bytes", ctypes.c_size_t)]


class TreeVerifyDesc(ctypes.Structure):
    """ds_cuda_tree_verify_t."""
    _fields_ = [("batch", _int), ("n_nodes", _int), ("vocab", _int), ("tokens", _ptr), ("parents", _ptr),
                ("nodes", _ptr), ("target", _ptr), ("target_stride", _i64 * 2), ("draft", _ptr),
                ("draft_stride", _i64 * 2), ("accept_u", _ptr), ("sample_u", _ptr), ("path", _ptr),
                ("accepted", _ptr), ("token", _ptr)]


class TreeCommitDesc(ctypes.Structure):
    """ds_cuda_tree_commit_t."""
    _fields_ = [("n_tensors", _int), ("layers", _int), ("batch", _int), ("n_nodes", _int), ("n_kv_heads", _int),
                ("head_dim", _int), ("kv_max", _int), ("cache", _ptr * 8), ("cache_stride", _i64 * 4 * 8),
                ("tree", _ptr * 8), ("tree_stride", _i64 * 4 * 8), ("lens", _ptr), ("path", _ptr),
                ("accepted", _ptr), ("new_lens", _ptr)]


def _packer(cls):
    """A struct.Struct that packs a descriptor's fields in order (a tenth of
    the time of setting them one by one)."""
    code = {_int: "i", ctypes.c_float: "f", _ptr: "P", _i64: "q", ctypes.c_size_t: "N"}

    def one(t):
        n = 1
        while issubclass(t, ctypes.Array):
            n, t = n * t._length_, t._type_
        return f"{n}{code[t]}"

    s = struct.Struct("@" + "".join(one(t) for _, t in cls._fields_))
    assert s.size == ctypes.sizeof(cls)
    return s.pack


_pack_attention, _pack_verify, _pack_commit = (_packer(c) for c in (TreeAttentionDesc, TreeVerifyDesc, TreeCommitDesc))


class Speculative:
    """The speculative-decoding operators of one context."""

    def __init__(self, ctx=None):
        import torch
        self.torch = torch
        self.ctx = ctx or Context(0)
        self.lib = self.ctx.lib
        self.device = torch.device("cuda", self.ctx.device)
        self._index = self.ctx.device
        self._types = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
        self._workspace = {}  # bytes by sizes
        # the handle alone, without the Stream object (2 us) around it
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda i: torch.cuda.current_stream(i).cuda_stream)

    def _stream(self):
        # torch's default stream is the legacy stream (handle 0), which the C
        # ABI would take for the context's own: cudaStreamLegacy is handle 1
        return self._raw_stream(self._index) or 1

    def _refuse(self, name, t, shape, dtype, why):
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self._index:
            why = f"expected {dtype} {tuple(shape)} on {self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}"
        raise ValueError(f"{name}: {why}")

    def _want(self, name, t, shape, dtype):
        """The address of a contiguous tensor that has to be as given."""
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self._index or not t.is_contiguous():
            self._refuse(name, t, shape, dtype, "must be contiguous")
        return t.data_ptr()

    def _strided(self, name, t, shape, dtype):
        """Address and strides but the last, which is 1."""
        st = t.stride()
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self._index or (st[-1] != 1 and shape[-1] > 1):
            self._refuse(name, t, shape, dtype, "the last dimension must be contiguous")
        return t.data_ptr(), *st[:-1]

    def _rows(self, name, planes, shape, dtype, pair):
        """Address, lo address, strides of a K or V tensor: one tensor, or
        with F32 queries its BF16 plane and optional lo plane."""
        if isinstance(planes, self.torch.Tensor):
            planes = (planes,)
        t, n = planes[0], len(planes)
        st = t.stride()
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self._index or st[-1] != 1:
            self._refuse(name, t, shape, dtype, "the last dimension must be contiguous")
        if n == 1:
            return t.data_ptr(), 0, *st[:3]
        if n != 2 or not pair:
            raise ValueError(f"{name}: {n} planes" + (" (at most 2)" if pair else
                                                     " (a second plane goes with float32 queries)"))
        lo = planes[1]
        if lo.dtype is not dtype or lo.shape != shape or lo.get_device() != self._index or lo.stride() != st:
            self._refuse(name + " lo plane", lo, shape, dtype, "the planes must have the same strides")
        return t.data_ptr(), lo.data_ptr(), *st[:3]

    def tree_mask(self, parents, counts=None):
        """Mask words [batch x n_nodes x ceil(n_nodes / 64)] (int64 bits) and
        depths [batch x n_nodes] of trees given by parents (int32)."""
        torch = self.torch
        b, n = parents.shape
        pp = self._want("parents", parents, (b, n), torch.int32)
        cp = None if counts is None else self._want("counts", counts, (b,), torch.int32)
        mask = torch.empty((b, n, (n + 63) // 64), dtype=torch.int64, device=self.device)
        depth = torch.empty((b, n), dtype=torch.int32, device=self.device)
        self.ctx.check(self.lib.ds_cuda_tree_mask_dev(self.ctx.h, pp, cp, b, n, mask.data_ptr(), depth.data_ptr(),
                                                      self._stream()), "tree_mask")
        return mask, depth

    def tree_attention(self, q, k, v, tree_k, tree_v, lens, mask, counts=None, scale=None, out=None, lse=None):
        """Attention of q [batch x n_nodes x n_heads x head_dim] over the
        cached rows k, v [batch x n_kv_heads x kv_max x head_dim] below lens
        [batch] (int32) and the tree's own tree_k, tree_v [batch x n_kv_heads
        x n_nodes x head_dim] where the mask words [batch x n_nodes x words]
        (int64) allow it. bfloat16 and float16 throughout, or float32 q with
        each of k, v, tree_k, tree_v a bfloat16 plane or a (plane, lo plane)
        pair (the decoder's cache form). counts [batch]: nodes in use (the
        other rows are zeros); scale: default head_dim ** -0.5; lse: optional
        [batch x n_nodes x n_heads] float32 output. Returns out."""
        torch = self.torch
        b, n, heads, hd = q.shape
        qt = q.dtype
        ty = self._types.get(qt)
        if ty is None:
            raise ValueError(f"q: unsupported dtype {qt}")
        pair = ty == F32
        kt = torch.bfloat16 if pair else qt
        k0 = k if isinstance(k, torch.Tensor) else k[0]
        if k0.dim() != 4:
            raise ValueError("k: expected [batch x n_kv_heads x kv_max x head_dim]")
        _, kv, cap, _ = k0.shape
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        cache, tree, i32 = (b, kv, cap, hd), (b, kv, n, hd), torch.int32
        head = (ty, b, n, heads, kv, hd, cap)
        fields = (*head, hd ** -0.5 if scale is None else scale,
                  *self._strided("q", q, (b, n, heads, hd), qt),
                  *self._rows("k", k, cache, kt, pair), *self._rows("v", v, cache, kt, pair),
                  *self._rows("tree_k", tree_k, tree, kt, pair), *self._rows("tree_v", tree_v, tree, kt, pair),
                  self._want("lens", lens, (b,), i32), 0 if counts is None else self._want("counts", counts, (b,), i32),
                  self._want("mask", mask, (b, n, (n + 63) // 64), torch.int64),
                  *self._strided("out", out, (b, n, heads, hd), qt),
                  0 if lse is None else self._want("lse", lse, (b, n, heads), torch.float32))
        key = (head, pair and any(fields[13:29:5]))  # a lo plane's presence
        need = self._workspace.get(key)
        if need is None:
            need = self._workspace[key] = self.lib.ds_cuda_tree_attention_workspace(self.ctx.h,
                                                                                    _pack_attention(*fields, 0, 0))
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self.ctx.check(self.lib.ds_cuda_tree_attention_dev(
            self.ctx.h, _pack_attention(*fields, ws.data_ptr() if need else 0, need), self._stream()), "tree_attention")
        return out

    def token_probs(self, logits, temperature=None, out=None):
        """softmax(logits / temperature) of each row: logits [rows x vocab]
        float32, bfloat16 or float16 (rows may be strided), temperature
        [rows] float32 or None; <= 0 is 1 at the row's argmax. float32."""
        torch = self.torch
        rows, vocab = logits.shape
        ty = self._types.get(logits.dtype)
        if ty is None:
            raise ValueError(f"logits: unsupported dtype {logits.dtype}")
        lp, st = self._strided("logits", logits, (rows, vocab), logits.dtype)
        tp = None if temperature is None else self._want("temperature", temperature, (rows,), torch.float32)
        if out is None:
            out = torch.empty((rows, vocab), dtype=torch.float32, device=self.device)
        self.ctx.check(self.lib.ds_cuda_token_probs_dev(self.ctx.h, ty, lp, rows, vocab, st, tp,
                                                        self._want("out", out, (rows, vocab), torch.float32),
                                                        self._stream()), "token_probs")
        return out

    def verify(self, tokens, parents, target, draft, accept_u, sample_u, counts=None):
        """Speculative sampling over each sequence's tree: tokens, parents
        [batch x n_nodes] int32; target [batch x n_nodes x vocab] float32,
        the target's probabilities after each node; draft the same, row p
        what p's children were drawn from (None: drafts are certain);
        accept_u [batch x n_nodes] and sample_u [batch] uniforms in [0, 1).
        Returns path [batch x n_nodes] (accepted node indices, then -1),
        accepted [batch] and the next token [batch], all int32."""
        torch = self.torch
        b, n = tokens.shape
        if target.dim() != 3:
            raise ValueError("target: expected [batch x n_nodes x vocab]")
        vocab = target.shape[2]
        i32, f32, shape = torch.int32, torch.float32, (b, n, vocab)
        res = self._results(tokens)
        d = _pack_verify(b, n, vocab, self._want("tokens", tokens, (b, n), i32),
                         self._want("parents", parents, (b, n), i32),
                         0 if counts is None else self._want("counts", counts, (b,), i32),
                         *self._strided("target", target, shape, f32),
                         *((0, 0, 0) if draft is None else self._strided("draft", draft, shape, f32)),
                         self._want("accept_u", accept_u, (b, n), f32), self._want("sample_u", sample_u, (b,), f32),
                         *(t.data_ptr() for t in res))
        self.ctx.check(self.lib.ds_cuda_tree_verify_dev(self.ctx.h, d, self._stream()), "tree_verify")
        return res

    def _results(self, tokens):
        accepted, token = tokens.new_empty((2, tokens.shape[0]))
        return self.torch.empty_like(tokens), accepted, token

    def verify_greedy(self, tokens, parents, target_tokens, counts=None):
        """The greedy rule on the target's argmax tokens [batch x n_nodes]
        int32: a child is accepted if its token is its parent's target token.
        Returns path, accepted and token as verify."""
        torch = self.torch
        b, n = tokens.shape
        tp = self._want("tokens", tokens, (b, n), torch.int32)
        pp = self._want("parents", parents, (b, n), torch.int32)
        wp = self._want("target_tokens", target_tokens, (b, n), torch.int32)
        cp = None if counts is None else self._want("counts", counts, (b,), torch.int32)
        res = self._results(tokens)
        self.ctx.check(self.lib.ds_cuda_tree_verify_greedy_dev(self.ctx.h, tp, pp, cp, wp, b, n,
                                                               *(t.data_ptr() for t in res), self._stream()),
                       "tree_verify_greedy")
        return res

    def commit(self, caches, trees, lens, path, accepted):
        """Copies the accepted nodes' rows into the caches, in place: for
        each pair of caches [layers x batch x n_kv_heads x kv_max x head_dim]
        and trees [layers x batch x n_kv_heads x n_nodes x head_dim] (at most
        8 pairs of 16-bit tensors, K and V or their planes) row path[b, j] of
        the tree to row lens[b] + j of the cache, j = 0 .. accepted[b].
        Returns the new lengths."""
        torch = self.torch
        b, n = path.shape
        if not 1 <= len(caches) == len(trees) <= 8:
            raise ValueError(f"commit: {len(caches)} caches and {len(trees)} trees (1 to 8 pairs)")
        first = caches[0]
        if first.dim() != 5 or first.element_size() != 2:
            raise ValueError("caches: expected 16-bit [layers x batch x n_kv_heads x kv_max x head_dim]")
        layers, _, kv, cap, hd = first.shape
        m, shape, rows, dt = len(caches), (layers, b, kv, cap, hd), (layers, b, kv, n, hd), first.dtype
        i32 = torch.int32
        cp, cs, tp, ts = [0] * 8, [0] * 32, [0] * 8, [0] * 32
        for i in range(m):
            cp[i], *cs[4 * i:4 * i + 4] = self._strided("cache", caches[i], shape, dt)
            tp[i], *ts[4 * i:4 * i + 4] = self._strided("tree", trees[i], rows, dt)
        new = torch.empty_like(lens)
        d = _pack_commit(m, layers, b, n, kv, hd, cap, *cp, *cs, *tp, *ts, self._want("lens", lens, (b,), i32),
                         self._want("path", path, (b, n), i32), self._want("accepted", accepted, (b,), i32),
                         new.data_ptr())
        self.ctx.check(self.lib.ds_cuda_tree_commit_dev(self.ctx.h, d, self._stream()), "tree_commit")
        return new
