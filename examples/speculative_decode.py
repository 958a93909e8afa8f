"""Speculative decoding of the DeepSeek3B-MoE decoder with n-gram drafts.

Each stream's draft is a tree of continuations that followed the last token
earlier in its own history. One step runs the whole tree through the decoder
(QKV, tree attention over the cache, the MoE block), turns the logits into
probabilities, verifies the drafts and commits the accepted rows, so a step
yields one token and as many more as were drafted right. At temperature 0 the
tokens are those that single-token trees give; above, they are distributed as
those trees' samples. (Decoder's own step takes the reference's approximate
exponential in its attention and dense layer, where the softmax here is exact:
logits differ by about a hundredth, near ties the token may.)

    python examples/speculative_decode.py [--layers 3] [--vocab 8192] [--tokens 64] [--temperature 0]

The prompt goes through Decoder.prefill, whose K and V rows become the cache.
The weights are synthetic (seeded).
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ds_ocr_b200 import synth  # noqa: E402
from ds_ocr_b200.cuda import Context  # noqa: E402
from ds_ocr_b200.decoder import Decoder  # noqa: E402
from ds_ocr_b200.prefill import Prefill  # noqa: E402
from ds_ocr_b200.speculative import Speculative  # noqa: E402

HEAD_SLICE = 64000  # LM-head rows a product call takes (at most 128000)


DRAFT_DEPTH = 6


def ngram_tree(history, n_nodes, branches=4, depth=DRAFT_DEPTH):
    """(tokens, parents) of a tree whose root is history[-1]: up to `branches`
    continuations of the places where it stood before, those that share the
    longest context first; the most recent first among equals."""
    root = history[-1]

    def shared(i):
        n = 0
        while n < 3 and i - n >= 0 and history[i - n] == history[-1 - n]:
            n += 1
        return n

    places = [i for i in range(len(history) - 1) if history[i] == root]
    places.sort(key=lambda i: (-shared(i), -i))
    tokens, parents, child = [root], [-1], {}
    for i in places[:branches]:
        cur = 0
        for t in history[i + 1:i + 1 + depth]:
            if (cur, t) not in child:
                if len(tokens) == n_nodes:
                    break
                child[cur, t] = len(tokens)
                tokens.append(t)
                parents.append(cur)
            cur = child[cur, t]
    return tokens, parents


def planes(x):
    """The cache form of F32 values: two BF16 planes, value = hi + lo."""
    hi = x.bfloat16()
    return hi, (x - hi.float()).bfloat16()


class SpeculativeDecoder:
    """n_streams streams, trees of n_nodes nodes (n_streams * n_nodes <= 64,
    the rows of one product call)."""

    def __init__(self, model, n_streams, n_nodes, ctx=None, kv_max=1024):
        assert n_streams * n_nodes <= 64
        self.ctx = ctx or Context(0)
        self.model, self.d = model, model.d
        self.B, self.N, self.kv_max = n_streams, n_nodes, kv_max
        d, self.device = self.d, torch.device("cuda", self.ctx.device)
        self.spec, self.moe = Speculative(self.ctx), Prefill(self.d, self.ctx)
        for lw in model.layers:
            for w in (lw.wq, lw.wk, lw.wv, lw.wo, lw.dense_gate, lw.dense_up, lw.dense_down):
                if w is not None:
                    self.ctx.register(w)
        self.ctx.register(model.lm_head)
        self.norms = [[torch.from_numpy(w).to(self.device) for w in (lw.input_norm, lw.post_norm)] for lw in model.layers]
        self.final_norm = torch.from_numpy(model.final_norm).to(self.device)
        self.embedding = torch.from_numpy(model.lm_head.view(np.int16)).to(self.device).view(torch.bfloat16)
        # K, V as (plane, lo plane): caches and the trees' own rows
        self.caches = [torch.zeros(d.n_layers, self.B, d.n_heads, kv_max, d.head_dim, dtype=torch.bfloat16,
                                   device=self.device) for _ in range(4)]
        self.trees = [torch.zeros(d.n_layers, self.B, d.n_heads, self.N, d.head_dim, dtype=torch.bfloat16,
                                  device=self.device) for _ in range(4)]
        self.lens = torch.zeros(self.B, dtype=torch.int32, device=self.device)
        half = torch.arange(0, d.head_dim, 2, device=self.device, dtype=torch.float32) / d.head_dim
        angle = torch.arange(kv_max + n_nodes, device=self.device)[:, None] * (1.0 / synth.ROPE_THETA ** half)
        self.cos, self.sin = angle.cos(), angle.sin()

    def prefill(self, stream, tokens):
        """Runs the prompt but its last token (which becomes the first
        tree's root) and takes over its K and V rows."""
        n = len(tokens) - 1
        self.lens[stream] = n
        if n == 0:
            return
        dec = Decoder(self.model, self.ctx, kv_max=self.kv_max)
        try:
            dec.prefill(np.stack([self.model.embed(t) for t in tokens[:-1]]))
            for l in range(self.d.n_layers):
                for i, rows in enumerate(dec.kv(l, 0, n)):
                    x = torch.from_numpy(rows).to(self.device).view(n, self.d.n_heads, self.d.head_dim).transpose(0, 1)
                    for c, p in zip(self.caches[2 * i:2 * i + 2], planes(x)):
                        c[l, stream, :, :n] = p
        finally:
            dec.close()

    def _matmul(self, x, w, resid=None, rows=None, start=0):
        """x W^T (+ resid) with W a registered weight, or `rows` of its rows."""
        n, K = x.shape
        rows = rows or w.shape[0]
        y = torch.empty(n, rows, device=self.device)
        st = torch.cuda.current_stream(self.device).cuda_stream or 1
        self.ctx.check(self.ctx.lib.ds_cuda_skinny_matmul_dev(
            self.ctx.h, x.data_ptr(), n, K, self.ctx.device_ptr(w) + 2 * start * K, rows,
            None if resid is None else resid.data_ptr(), y.data_ptr(), st), "skinny_matmul")
        return y

    def _norm(self, x, w):
        return (x * w) * torch.rsqrt(x.square().mean(-1, keepdim=True) + synth.RMS_EPS)

    def _rope(self, x, pos):
        c, s = self.cos[pos][:, :, None], self.sin[pos][:, :, None]
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    def logits(self, tokens, parents, counts):
        """The decoder over the trees: [n_streams x n_nodes x vocab]."""
        d, shape = self.d, (self.B, self.N, self.d.n_heads, self.d.head_dim)
        mask, depth = self.spec.tree_mask(parents, counts)
        pos = self.lens[:, None] + depth
        x = self.embedding[tokens.view(-1)].float()
        st = torch.cuda.current_stream(self.device).cuda_stream or 1
        for l, lw in enumerate(self.model.layers):
            xn = self._norm(x, self.norms[l][0])
            q = self._rope(self._matmul(xn, lw.wq).view(shape), pos)
            k = self._rope(self._matmul(xn, lw.wk).view(shape), pos)
            v = self._matmul(xn, lw.wv).view(shape)
            for t, p in zip(self.trees, (*planes(k), *planes(v))):
                t[l] = p.transpose(1, 2)
            kc, kl, vc, vl = (c[l] for c in self.caches)
            tk, tkl, tv, tvl = (t[l] for t in self.trees)
            o = self.spec.tree_attention(q, (kc, kl), (vc, vl), (tk, tkl), (tv, tvl), self.lens, mask, counts)
            x = self._matmul(o.view(len(x), -1), lw.wo, resid=x)
            if lw.dense:
                xn = self._norm(x, self.norms[l][1])
                h = torch.nn.functional.silu(self._matmul(xn, lw.dense_gate)) * self._matmul(xn, lw.dense_up)
                x = self._matmul(h, lw.dense_down, resid=x)
            else:
                self.moe.moe_layer_dev(lw, x.data_ptr(), len(x), stream=st)
        x = self._norm(x, self.final_norm)
        return torch.cat([self._matmul(x, self.model.lm_head, rows=min(HEAD_SLICE, d.vocab - s), start=s)
                          for s in range(0, d.vocab, HEAD_SLICE)], -1).view(self.B, self.N, d.vocab)

    def step(self, trees, temperature=0.0, generator=None):
        """One step of every stream on its (tokens, parents); returns each
        stream's new tokens."""
        tokens = torch.zeros(self.B, self.N, dtype=torch.int32)
        parents = torch.full((self.B, self.N), -1, dtype=torch.int32)
        for b, (t, p) in enumerate(trees):
            tokens[b, :len(t)] = torch.tensor(t, dtype=torch.int32)
            parents[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        counts = torch.tensor([len(t) for t, _ in trees], dtype=torch.int32, device=self.device)
        tokens, parents = tokens.to(self.device), parents.to(self.device)
        logits = self.logits(tokens, parents, counts)
        temp = torch.full((self.B * self.N,), temperature, device=self.device)
        p = self.spec.token_probs(logits.view(self.B * self.N, -1), temp).view_as(logits)
        u = torch.rand(self.B, self.N + 1, device=self.device, generator=generator)
        path, accepted, token = self.spec.verify(tokens, parents, p, None, u[:, :-1].contiguous(),
                                                 u[:, -1].contiguous(), counts)
        self.lens = self.spec.commit(self.caches, self.trees, self.lens, path, accepted)
        drafted = tokens.gather(1, path.clamp(min=0).long())
        out = torch.cat((accepted[:, None], token[:, None], drafted), 1).tolist()  # the step's one read
        return [row[3:3 + row[0]] + [row[1]] for row in out]

    def generate(self, prompts, n_tokens, temperature=0.0, generator=None):
        """n_tokens tokens after each prompt, and the number of steps. A
        stream that is done before the others goes on without drafts."""
        assert max(map(len, prompts)) + 2 * n_tokens + DRAFT_DEPTH <= self.kv_max
        histories = [list(p) for p in prompts]
        for b, p in enumerate(prompts):
            self.prefill(b, p)
        steps = 0
        while any(len(h) - len(p) < n_tokens for h, p in zip(histories, prompts)):
            new = self.step([ngram_tree(h, self.N if len(h) - len(p) < n_tokens else 1)
                             for h, p in zip(histories, prompts)], temperature, generator)
            for h, t in zip(histories, new):
                h.extend(t)
            steps += 1
        self.spec.check()
        self.moe.check()
        return [h[len(p):len(p) + n_tokens] for h, p in zip(histories, prompts)], steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=3)
    ap.add_argument("--vocab", type=int, default=8192)
    ap.add_argument("--streams", type=int, default=4)
    ap.add_argument("--nodes", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=48)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    model = synth.Model(n_layers=a.layers, vocab=a.vocab)
    dec = SpeculativeDecoder(model, a.streams, a.nodes, kv_max=a.prompt + 2 * a.tokens + DRAFT_DEPTH)
    prompts = [[(b * 977 + i * 37 + 11) % a.vocab for i in range(a.prompt)] for b in range(a.streams)]
    out, steps = dec.generate(prompts, a.tokens, a.temperature)
    for b, t in enumerate(out):
        print(f"stream {b}: {t[:16]} ...")
    print(f"{a.tokens} tokens a stream in {steps} steps")


if __name__ == "__main__":
    main()
