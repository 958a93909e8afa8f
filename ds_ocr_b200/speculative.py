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


class Speculative:
    """The speculative-decoding operators of one context."""

    def __init__(self, ctx=None):
        import torch
        self.torch = torch
        self.ctx = ctx or Context(0)
        self.lib = self.ctx.lib
        self.device = torch.device("cuda", self.ctx.device)
        self._types = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}

    def _stream(self):
        # torch's default stream is the legacy stream (handle 0), which the C
        # ABI would take for the context's own: cudaStreamLegacy is handle 1
        return self.torch.cuda.current_stream(self.device).cuda_stream or 1

    def _want(self, name, t, shape, dtype, contiguous=True):
        if t.device != self.device or t.dtype != dtype or t.shape != shape:
            raise ValueError(f"{name}: expected {dtype} {tuple(shape)} on {self.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        if contiguous and not t.is_contiguous():
            raise ValueError(f"{name}: must be contiguous")
        return t.data_ptr()

    def _rows(self, name, planes, shape, dtype, pair):
        """(address, lo address, strides) of a K or V tensor: one tensor, or
        with F32 queries its BF16 plane and optional lo plane."""
        if isinstance(planes, self.torch.Tensor):
            planes = (planes,)
        if not 1 <= len(planes) <= (2 if pair else 1):
            raise ValueError(f"{name}: {len(planes)} planes" + (" (at most 2)" if pair else
                                                               " (a second plane goes with float32 queries)"))
        a = planes[0]
        p = self._want(name, a, shape, dtype, False)
        st = a.stride()
        if st[-1] != 1:
            raise ValueError(f"{name}: the head dimension must be contiguous")
        if len(planes) == 1:
            return p, None, st
        lo = planes[1]
        if lo.stride() != st:
            raise ValueError(f"{name}: the planes must have the same strides")
        return p, self._want(name + " lo plane", lo, shape, dtype, False), st

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
        ty = self._types.get(q.dtype)
        if ty is None:
            raise ValueError(f"q: unsupported dtype {q.dtype}")
        kt = torch.bfloat16 if ty == F32 else q.dtype
        k0 = k if isinstance(k, torch.Tensor) else k[0]
        if k0.dim() != 4:
            raise ValueError("k: expected [batch x n_kv_heads x kv_max x head_dim]")
        kv, cap = k0.shape[1], k0.shape[2]
        qp = self._want("q", q, (b, n, heads, hd), q.dtype, False)
        qs = q.stride()
        if qs[3] != 1:
            raise ValueError("q: the head dimension must be contiguous")
        if out is None:
            out = torch.empty((b, n, heads, hd), dtype=q.dtype, device=self.device)
        op = self._want("out", out, (b, n, heads, hd), q.dtype, False)
        os = out.stride()
        if os[3] != 1:
            raise ValueError("out: the head dimension must be contiguous")
        d = TreeAttentionDesc()
        d.type, d.batch, d.n_nodes, d.n_heads, d.n_kv_heads, d.head_dim, d.kv_max = ty, b, n, heads, kv, hd, cap
        d.scale = hd ** -0.5 if scale is None else scale
        d.q, d.q_stride = qp, qs[:3]
        d.out, d.out_stride = op, os[:3]
        d.k, d.k_lo, st = self._rows("k", k, (b, kv, cap, hd), kt, ty == F32)
        d.k_stride = st[:3]
        d.v, d.v_lo, st = self._rows("v", v, (b, kv, cap, hd), kt, ty == F32)
        d.v_stride = st[:3]
        d.tree_k, d.tree_k_lo, st = self._rows("tree_k", tree_k, (b, kv, n, hd), kt, ty == F32)
        d.tree_k_stride = st[:3]
        d.tree_v, d.tree_v_lo, st = self._rows("tree_v", tree_v, (b, kv, n, hd), kt, ty == F32)
        d.tree_v_stride = st[:3]
        d.lens = self._want("lens", lens, (b,), torch.int32)
        d.mask = self._want("mask", mask, (b, n, (n + 63) // 64), torch.int64)
        d.nodes = None if counts is None else self._want("counts", counts, (b,), torch.int32)
        d.lse = None if lse is None else self._want("lse", lse, (b, n, heads), torch.float32)
        need = self.lib.ds_cuda_tree_attention_workspace(self.ctx.h, ctypes.byref(d))
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            d.workspace, d.workspace_bytes = ws.data_ptr(), need
        self.ctx.check(self.lib.ds_cuda_tree_attention_dev(self.ctx.h, ctypes.byref(d), self._stream()),
                       "tree_attention")
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
        lp = self._want("logits", logits, (rows, vocab), logits.dtype, False)
        if vocab > 1 and logits.stride(1) != 1:
            raise ValueError("logits: the vocabulary must be contiguous")
        tp = None if temperature is None else self._want("temperature", temperature, (rows,), torch.float32)
        if out is None:
            out = torch.empty((rows, vocab), dtype=torch.float32, device=self.device)
        self.ctx.check(self.lib.ds_cuda_token_probs_dev(self.ctx.h, ty, lp, rows, vocab, logits.stride(0), tp,
                                                        self._want("out", out, (rows, vocab), torch.float32),
                                                        self._stream()), "token_probs")
        return out

    def _probs(self, name, p, b, n, vocab):
        a = self._want(name, p, (b, n, vocab), self.torch.float32, False)
        if vocab > 1 and p.stride(2) != 1:
            raise ValueError(f"{name}: the vocabulary must be contiguous")
        return a, p.stride()[:2]

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
        d = TreeVerifyDesc()
        d.batch, d.n_nodes, d.vocab = b, n, vocab
        d.tokens = self._want("tokens", tokens, (b, n), torch.int32)
        d.parents = self._want("parents", parents, (b, n), torch.int32)
        d.nodes = None if counts is None else self._want("counts", counts, (b,), torch.int32)
        d.target, d.target_stride = self._probs("target", target, b, n, vocab)
        if draft is not None:
            d.draft, d.draft_stride = self._probs("draft", draft, b, n, vocab)
        d.accept_u = self._want("accept_u", accept_u, (b, n), torch.float32)
        d.sample_u = self._want("sample_u", sample_u, (b,), torch.float32)
        res = self._results(b, n)
        d.path, d.accepted, d.token = (t.data_ptr() for t in res)
        self.ctx.check(self.lib.ds_cuda_tree_verify_dev(self.ctx.h, ctypes.byref(d), self._stream()), "tree_verify")
        return res

    def _results(self, b, n):
        torch = self.torch
        r = torch.empty(b * (n + 2), dtype=torch.int32, device=self.device)
        return r[:b * n].view(b, n), r[b * n:b * n + b], r[b * n + b:]

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
        res = self._results(b, n)
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
        d = TreeCommitDesc()
        d.n_tensors, d.layers, d.batch, d.n_nodes, d.n_kv_heads, d.head_dim, d.kv_max = (len(caches), layers, b, n, kv,
                                                                                         hd, cap)
        for i, (c, t) in enumerate(zip(caches, trees)):
            d.cache[i] = self._want("cache", c, (layers, b, kv, cap, hd), first.dtype, False)
            d.tree[i] = self._want("tree", t, (layers, b, kv, n, hd), first.dtype, False)
            cs, ts = c.stride(), t.stride()
            if cs[4] != 1 or ts[4] != 1:
                raise ValueError("commit: the head dimension must be contiguous")
            d.cache_stride[i][:] = cs[:4]
            d.tree_stride[i][:] = ts[:4]
        d.lens = self._want("lens", lens, (b,), torch.int32)
        d.path = self._want("path", path, (b, n), torch.int32)
        d.accepted = self._want("accepted", accepted, (b,), torch.int32)
        new = torch.empty(b, dtype=torch.int32, device=self.device)
        d.new_lens = new.data_ptr()
        self.ctx.check(self.lib.ds_cuda_tree_commit_dev(self.ctx.h, ctypes.byref(d), self._stream()), "tree_commit")
        return new
