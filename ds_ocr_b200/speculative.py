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

from ._lib import SIGNATURES, DsCudaError, load
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
    """The speculative-decoding operators of one context. The tensors are
    checked and the descriptors filled in native code (ds_ocr_b200._spec): a
    wrong tensor raises ValueError, a refused call DsCudaError."""

    def __init__(self, ctx=None):
        import torch
        self.ctx = ctx or Context(0)
        self.device = torch.device("cuda", self.ctx.device)
        self._spec = _module()
        self._index = self.ctx.device

    def tree_mask(self, parents, counts=None):
        """Mask words [batch x n_nodes x ceil(n_nodes / 64)] (int64 bits) and
        depths [batch x n_nodes] of trees given by parents (int32)."""
        return self._spec.tree_mask(self.ctx.h, self._index, parents, counts)

    def tree_attention(self, q, k, v, tree_k, tree_v, lens, mask, counts=None, scale=None, out=None, lse=None):
        """Attention of q [batch x n_nodes x n_heads x head_dim] over the
        cached rows k, v [batch x n_kv_heads x kv_max x head_dim] below lens
        [batch] (int32) and the tree's own tree_k, tree_v [batch x n_kv_heads
        x n_nodes x head_dim] where the mask words [batch x n_nodes x words]
        (int64) allow it. bfloat16 and float16 throughout (weights rounded
        to that type for the product with v, sums in float32), or float32 q
        with each of k, v, tree_k, tree_v a bfloat16 plane or a (plane, lo
        plane) pair (the decoder's cache form). counts [batch]: nodes in use (the
        other rows are zeros); scale: default head_dim ** -0.5; lse: optional
        [batch x n_nodes x n_heads] float32 output. Returns out."""
        return self._spec.tree_attention(self.ctx.h, self._index, q, k, v, tree_k, tree_v, lens, mask, counts, scale, out, lse)

    def check(self):
        """Synchronise the current stream and raise if a tree attention
        kernel's bounded wait gave up since this stream's last check."""
        import torch
        st = torch.cuda.current_stream(self.device).cuda_stream or 1  # cudaStreamLegacy
        self.ctx.check(self.ctx.lib.ds_cuda_tree_attention_check(self.ctx.h, st), "tree_attention")

    def token_probs(self, logits, temperature=None, out=None):
        """softmax(logits / temperature) of each row: logits [rows x vocab]
        float32, bfloat16 or float16 (rows may be strided), temperature
        [rows] float32 or None; <= 0 is 1 at the row's argmax. float32."""
        return self._spec.token_probs(self.ctx.h, self._index, logits, temperature, out)

    def verify(self, tokens, parents, target, draft, accept_u, sample_u, counts=None):
        """Speculative sampling over each sequence's tree: tokens, parents
        [batch x n_nodes] int32; target [batch x n_nodes x vocab] float32,
        the target's probabilities after each node; draft the same, row p
        what p's children were drawn from (None: drafts are certain);
        accept_u [batch x n_nodes] and sample_u [batch] uniforms in [0, 1).
        Returns path [batch x n_nodes] (accepted node indices, then -1),
        accepted [batch] and the next token [batch], all int32."""
        return self._spec.verify(self.ctx.h, self._index, tokens, parents, target, draft, accept_u, sample_u, counts)

    def verify_greedy(self, tokens, parents, target_tokens, counts=None):
        """The greedy rule on the target's argmax tokens [batch x n_nodes]
        int32: a child is accepted if its token is its parent's target token.
        Returns path, accepted and token as verify."""
        return self._spec.verify_greedy(self.ctx.h, self._index, tokens, parents, target_tokens, counts)

    def commit(self, caches, trees, lens, path, accepted):
        """Copies the accepted nodes' rows into the caches, in place: for
        each pair of caches [layers x batch x n_kv_heads x kv_max x head_dim]
        and trees [layers x batch x n_kv_heads x n_nodes x head_dim] (at most
        8 pairs of 16-bit tensors, K and V or their planes) row path[b, j] of
        the tree to row lens[b] + j of the cache, j = 0 .. accepted[b].
        Returns the new lengths."""
        return self._spec.commit(self.ctx.h, self._index, caches, trees, lens, path, accepted)


def _module():
    """ds_ocr_b200._spec, built first if only the sources are present or it was
    built for another torch, on the entry points of the library that the
    contexts come from."""
    import importlib
    import torch  # noqa: F401  (its libraries have to be loaded)
    from . import build
    if build.spec_is_for_another():
        build.build_spec()
        importlib.invalidate_caches()
    try:
        from . import _spec
    except ImportError:
        build.build_spec(force=True)
        importlib.invalidate_caches()
        from . import _spec
    lib = load()
    _spec.bind({name: ctypes.cast(getattr(lib, name), _ptr).value for name in SIGNATURES})
    _spec.set_error(DsCudaError)
    return _spec
