"""Plain 64-bit forms of the speculative-decoding operators, for tests: the
attention of one tree over its cache in torch float64, the verification walk
in numpy float32 operations and Python integers, one element at a time."""
import math

import numpy as np
import torch


def planes(x, pair):
    """A float32 tensor as the planes of the decoder's cache."""
    hi = x.bfloat16()
    return (hi, (x - hi.float()).bfloat16()) if pair else (hi,)


def whole(t):
    t = (t,) if isinstance(t, torch.Tensor) else t
    return sum(p.double() for p in t)


def attention(q, k, v, tree_k, tree_v, lens, allowed, counts, scale):
    """allowed [batch][node][node] truth values. Only what a row attends is
    touched, so garbage elsewhere cannot reach it. Returns out and lse."""
    b, n, heads, hd = q.shape
    k, v, tree_k, tree_v = whole(k), whole(v), whole(tree_k), whole(tree_v)
    g = heads // k.shape[1]
    out = torch.zeros(b, n, heads, hd, dtype=torch.float64, device=q.device)
    lse = torch.full((b, n, heads), -math.inf, dtype=torch.float64, device=q.device)
    for i in range(b):
        m = int(lens[i])
        for r in range(int(counts[i])):
            see = [j for j in range(int(counts[i])) if allowed[i][r][j]]
            if m + len(see) == 0:
                continue
            kk = torch.cat([k[i, :, :m], tree_k[i][:, see]], 1).repeat_interleave(g, 0)
            vv = torch.cat([v[i, :, :m], tree_v[i][:, see]], 1).repeat_interleave(g, 0)
            s = (kk @ q[i, r].double()[:, :, None])[:, :, 0] * scale
            lse[i, r] = torch.logsumexp(s, 1)
            out[i, r] = (torch.softmax(s, 1)[:, None] @ vv)[:, 0]
    return out, lse


def words(allowed):
    """Mask words of [batch][node][node] truth values."""
    a = np.asarray(allowed)
    b, n, _ = a.shape
    w = (n + 63) // 64
    out = np.zeros((b, n, w), np.uint64)
    for j in range(n):
        out[:, :, j >> 6] |= a[:, :, j].astype(np.uint64) << np.uint64(j & 63)
    return torch.from_numpy(out.view(np.int64))


def random_tree(rng, n, count, width=4):
    par = [-1] * n
    for i in range(1, count):
        par[i] = int(rng.integers(max(0, i - width), i))
    return par


def ancestors(par, n, count):
    a = np.zeros((n, n), bool)
    for i in range(count):
        j = i
        while j >= 0:
            a[i, j] = True
            j = par[j]
    return a


def fixed(r):
    """Probabilities (float32) as whole multiples of 2**-44."""
    r = np.where(r > 0, np.minimum(r, np.float32(1)), np.float32(0)).astype(np.float32)
    return (r.astype(np.float64) * 2.0 ** 44).astype(np.int64)  # both steps exact but for the truncation


def verify(tokens, parents, count, target, draft, accept_u, sample_u):
    """One sequence: target, draft [n x vocab] float32 (draft may be None).
    Returns (path, token)."""
    f = np.float32
    vocab = target.shape[1]
    cur, path, mass, r = 0, [0], f(1), target[0].copy()
    for c in range(1, count):
        if parents[c] != cur:
            continue
        x = int(tokens[c])
        if draft is None:
            d = np.zeros(vocab, f)
            if 0 <= x < vocab:
                d[x] = 1
        else:
            d = draft[cur]
        if 0 <= x < vocab and f(accept_u[c]) * f(d[x] * mass) < r[x]:
            cur, mass, r = c, f(1), target[c].copy()
            path.append(c)
            continue
        with np.errstate(invalid="ignore"):
            # certain drafts touch the drafted token alone
            at = slice(None) if draft is not None else slice(x, x + 1) if 0 <= x < vocab else slice(0, 0)
            diff = (r[at] - (mass * d[at]).astype(f)).astype(f)
            r[at] = np.where(diff > 0, diff, f(0))  # fmaxf(NaN, 0) is 0
        mass = fixed(r).sum().astype(f) * f(2.0 ** -44)
    w = fixed(r)
    if w.sum() == 0:
        w = fixed(target[cur])
    total = int(w.sum())
    if total == 0:
        return path, -1
    u = int(f(sample_u) * f(2.0 ** 24))
    lim = (total >> 24) * u + (((total & 0xFFFFFF) * u) >> 24)
    return path, int(np.searchsorted(np.cumsum(w), lim, side="right"))
