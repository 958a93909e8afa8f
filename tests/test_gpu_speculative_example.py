"""examples/speculative_decode.py: the operators of a speculative step
together, on a decoder with synthetic weights, against one token at a time
in F64 from the same prompt rows (the MoE block through Prefill, which has
its own tests). The tokens are greedy up to the rounding of the logits: each
token's logit, given the same history, is within 2e-3 of the largest one's
magnitude (1e-3 relative on either side, the bound of the prefill's and the
decode step's own tests)."""
import numpy as np
import pytest

from ds_ocr_b200 import synth
from ds_ocr_b200.decoder import Decoder
from ds_ocr_b200.prefill import Prefill
from test_speculative_example_cpu import example  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    return synth.Model(n_layers=2, vocab=2048)


class Plain:
    """The decoder, a token at a time."""

    def __init__(self, model, ctx, prompt):
        import torch
        self.m, self.d, self.torch = model, model.d, torch
        self.moe = Prefill(model.d, ctx)
        self.w = {}
        n = len(prompt) - 1
        dec = Decoder(model, ctx, kv_max=128)
        try:
            if n:
                dec.prefill(np.stack([model.embed(t) for t in prompt[:-1]]))
            self.kv = [[list(self.to(r).view(n, self.d.n_heads, -1)) if n else [] for r in dec.kv(l, 0, n)]
                       if n else [[], []] for l in range(self.d.n_layers)]
        finally:
            dec.close()

    def to(self, a):
        return self.torch.from_numpy(a).double()

    def mul(self, x, w):
        if id(w) not in self.w:
            self.w[id(w)] = self.to(synth.bf16_to_f32(w))
        return self.w[id(w)] @ x

    def norm(self, x, w):
        return x * self.to(w) * (x.square().mean() + synth.RMS_EPS).rsqrt()

    def rope(self, x, pos):
        torch, hd = self.torch, self.d.head_dim
        angle = pos / synth.ROPE_THETA ** (torch.arange(0, hd, 2).double() / hd)
        a, b = x.chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)

    def step(self, token):
        torch, d = self.torch, self.d
        x = self.to(self.m.embed(token))
        for lw, (ks, vs) in zip(self.m.layers, self.kv):
            xn, pos = self.norm(x, lw.input_norm), len(ks)
            q, k, v = (self.mul(xn, w).view(d.n_heads, d.head_dim) for w in (lw.wq, lw.wk, lw.wv))
            ks.append(self.rope(k, pos))
            vs.append(v)
            s = torch.einsum("hd,thd->ht", self.rope(q, pos), torch.stack(ks)) * d.head_dim ** -0.5
            x = x + self.mul(torch.einsum("ht,thd->hd", s.softmax(-1), torch.stack(vs)).reshape(-1), lw.wo)
            if lw.dense:
                xn = self.norm(x, lw.post_norm)
                h = torch.nn.functional.silu(self.mul(xn, lw.dense_gate)) * self.mul(xn, lw.dense_up)
                x = x + self.mul(h, lw.dense_down)
            else:
                row = x.float().numpy()[None].copy()
                self.moe.moe_layer(lw, row)
                x = self.to(row[0])
        return self.mul(self.norm(x, self.m.final_norm), self.m.lm_head)


def prompts(kind, vocab):
    if kind == "repeating":
        return [[(7 * b + i % 5) % vocab for i in range(23)] for b in range(3)]
    return [[(977 * b + 37 * i + 11) % vocab for i in range(n)] for b, n in enumerate((1, 2, 40))]


@pytest.mark.parametrize("kind,nodes", [("repeating", 16), ("repeating", 5), ("distinct", 16), ("distinct", 1)])
def test_tokens_are_the_greedy_ones(cuda_ctx, model, example, kind, nodes):  # noqa: F811
    ps, n = prompts(kind, model.d.vocab), 24
    spec = example.SpeculativeDecoder(model, len(ps), nodes, cuda_ctx, kv_max=128)
    out, steps = spec.generate(ps, n)
    assert steps <= n and (nodes > 1 or steps == n)
    for p, tokens in zip(ps, out):
        assert len(tokens) == n
        plain, last = Plain(model, cuda_ctx, p), p[-1]
        for t in tokens:
            logits = plain.step(last)
            assert logits[t] >= logits.max() - 2e-3 * logits.abs().max()
            last = t


def test_sampling_uses_its_generator(cuda_ctx, model, example):  # noqa: F811
    import torch
    ps = prompts("repeating", model.d.vocab)
    runs = []
    for seed in (1, 1, 2):
        spec = example.SpeculativeDecoder(model, len(ps), 16, cuda_ctx, kv_max=128)
        g = torch.Generator(device="cuda").manual_seed(seed)
        runs.append(spec.generate(ps, 20, 1.0, g)[0])
    assert runs[0] == runs[1] != runs[2]
    assert all(0 <= t < model.d.vocab for r in runs for s in r for t in s)
