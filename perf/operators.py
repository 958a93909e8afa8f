"""What the speculative-decoding operators are measured on.

Four operators a decode loop with drafted tokens runs in turn:
  attention  the tree of drafted tokens over the KV cache,
  probs      the target's logits to probabilities at each row's temperature,
  verify     drafted tokens accepted or rejected from given uniforms, and the next token drawn,
  commit     the accepted tokens' K and V rows into the cache.
`listed()` has the cases, `run()` one pass of one operator: with `own` false in plain torch operations in 32 bits,
with `own` true through ds_ocr_b200.speculative.
"""
import functools
import math

import torch

own = False

DEV = "cuda"
FIX = 44  # probabilities are summed as whole multiples of 2**-44, so that no order of summation changes a token


def listed():
    return [
        # one token of one stream after the benchmark's 662-token prompt, on the decoder's two-plane cache: latency
        dict(name="attn_decode_1", op="attention", type="pair", batch=1, nodes=1, heads=10, kv_heads=10, dim=128, keys=662, layout="bhsd"),
        # one stream, a tree of 16 drafted tokens
        dict(name="attn_tree16_1", op="attention", type="pair", batch=1, nodes=16, heads=10, kv_heads=10, dim=128, keys=662, layout="bhsd"),
        # the multi-stream decoder's 64 streams, a tree of 8 each, prompts of many lengths
        dict(name="attn_tree8_64", op="attention", type="pair", batch=64, nodes=8, heads=10, kv_heads=10, dim=128, keys=1325, layout="bhsd"),
        # shared key heads, a tree of 31, documents of up to 8191 tokens, a token's heads side by side in the cache
        dict(name="attn_tree31_gqa_8", op="attention", type="bf16", batch=8, nodes=31, heads=32, kv_heads=8, dim=128, keys=8191, layout="bshd"),
        # one very long context, a wide tree, few key heads
        dict(name="attn_tree64_long_1", op="attention", type="f16", batch=1, nodes=64, heads=16, kv_heads=2, dim=64, keys=131071, layout="bhsd"),
        # one stream's tree of 9 on the decoder's vocabulary
        dict(name="probs_9", op="probs", type="f32", rows=9, vocab=129280),
        # 64 streams with a tree of 8, 16-bit logits, an odd vocabulary
        dict(name="probs_512", op="probs", type="bf16", rows=512, vocab=50257),
        # a chain of 7 drafted tokens of one stream: latency
        dict(name="verify_chain_1", op="verify", batch=1, nodes=8, width=1, vocab=129280),
        # 16 streams, trees of 31 with up to 3 children a node
        dict(name="verify_tree_16", op="verify", batch=16, nodes=31, width=3, vocab=129280),
        # 64 streams, trees of 16 with up to 2 children a node, an odd vocabulary
        dict(name="verify_tree_64", op="verify", batch=64, nodes=16, width=2, vocab=32001),
        # the decoder's 12 layers, one stream, a tree of 16, two planes
        dict(name="commit_1", op="commit", type="pair", layers=12, batch=1, nodes=16, kv_heads=10, dim=128, keys=703),
        # 12 layers, 16 streams, trees of 64 of which up to 40 are accepted
        dict(name="commit_16", op="commit", type="bf16", layers=12, batch=16, nodes=64, kv_heads=10, dim=128, keys=768),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "probs", "verify", "commit"])
    while True:
        if op == "attention":
            kv = rng.choice([1, 2, 3, 4, 8, 10, 16])
            c = dict(op=op, type=rng.choice(["pair", "bf16", "f16"]), batch=_log(rng, 1, 64), nodes=_log(rng, 1, 64),
                     heads=kv * rng.choice([1, 1, 2, 4, 8]), kv_heads=kv, dim=rng.choice([64, 128, 128]),
                     keys=_log(rng, 1, 131071), layout=rng.choice(["bhsd", "bshd"]))
            score = c["batch"] * c["heads"] * c["nodes"] * c["keys"]
            if score > 1 << 27:
                continue
        elif op == "probs":
            c = dict(op=op, type=rng.choice(["f32", "bf16", "f16"]), rows=_log(rng, 1, 1024), vocab=_log(rng, 500, 160000))
        elif op == "verify":
            c = dict(op=op, batch=_log(rng, 1, 64), nodes=_log(rng, 2, 48), width=rng.choice([1, 2, 3, 4]), vocab=_log(rng, 500, 160000))
            if c["batch"] * c["nodes"] * c["vocab"] > 16 * 31 * 129280:
                continue
        else:
            c = dict(op=op, type=rng.choice(["pair", "bf16", "f16"]), layers=_log(rng, 1, 16), batch=_log(rng, 1, 32), nodes=_log(rng, 1, 64),
                     kv_heads=rng.choice([1, 2, 4, 8, 10]), dim=rng.choice([64, 128]), keys=_log(rng, 64, 2048))
            if c["layers"] * c["batch"] * c["kv_heads"] * c["dim"] * c["keys"] > 12 * 16 * 10 * 128 * 768:
                continue
        most = [work(x) for x in listed() if x["op"] == op]
        w = work(c)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            return c


# ---- what follows from a case alone -------------------------------------------------------------------------------
def _lens(c):
    """Cached tokens of each sequence: the longest first, then spread down to a quarter of it."""
    n, b = c["keys"], c["batch"]
    return [n - (3 * n * ((i * 7) % b)) // (4 * b) for i in range(b)]


def _counts(c):
    """Nodes in use of each tree: all, or up to a third fewer."""
    return [max(1, c["nodes"] - (i % 3) * (c["nodes"] // 6)) for i in range(c["batch"])]


def _accepted(c):
    """commit: drafted tokens accepted of each tree."""
    return [(c["nodes"] - 1) * (1 + (i * 5) % 8) // 12 for i in range(c["batch"])]


def _kv_bytes(c):
    return {"pair": 4, "bf16": 2, "f16": 2}[c["type"]]


def work(case):
    c = case
    if c["op"] == "attention":
        lens, counts, d = _lens(c), _counts(c), c["dim"]
        rows = sum(n + t for n, t in zip(lens, counts)) * c["kv_heads"] * d
        out = 2 * sum(counts) * c["heads"] * d * (4 if c["type"] == "pair" else 2)
        return {"bytes": 2 * rows * _kv_bytes(c) + out, "flops": 4 * d * c["heads"] * sum(t * (n + 1) for n, t in zip(lens, counts))}
    if c["op"] == "probs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * (4 + (4 if c["type"] == "f32" else 2)), "flops": 4 * n}
    if c["op"] == "verify":
        # the walk ends at one node: its row of the target's and of the draft's probabilities
        n = c["batch"] * c["vocab"]
        return {"bytes": 8 * n, "flops": 6 * n}
    moved = sum(a + 1 for a in _accepted(c)) * c["layers"] * c["kv_heads"] * c["dim"] * 2 * _kv_bytes(c)
    return {"bytes": 2 * moved, "flops": 0}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _trees(c, g, width=4):
    """Parents [batch, nodes] (-1 for a root and for unused nodes): a node's parent is an earlier one with fewer than `width` children."""
    import random
    r = random.Random(int(torch.randint(1 << 30, (1,), generator=g, device=DEV)))
    rows = []
    for n in _counts(c):
        par, kids = [-1], [0] * c["nodes"]
        for i in range(1, n):
            free = [j for j in range(i) if kids[j] < width]
            p = r.choice(free[-max(2, width + 1):])
            kids[p] += 1
            par.append(p)
        rows.append(par + [-1] * (c["nodes"] - n))
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def _ancestors(parents, counts):
    """[batch, nodes, nodes]: node j is node i or above it."""
    b, n = parents.shape
    at = torch.arange(n, device=DEV)
    a = (parents.long()[:, :, None] == at) | torch.eye(n, dtype=torch.bool, device=DEV)
    a = a.float()
    for _ in range(max(1, n.bit_length())):
        a = ((a @ a) > 0).float()
    return (a > 0) & (at[None, :, None] < counts[:, None, None])


def _words(mask):
    """[..., n] truth values as [..., ceil(n / 64)] 64-bit words, the lowest bit first."""
    n = mask.shape[-1]
    w = -(-n // 64)
    m = torch.nn.functional.pad(mask, (0, 64 * w - n)).unflatten(-1, (w, 64)).long()
    return (m << torch.arange(64, device=DEV)).sum(-1)


def _planes(x):
    hi = x.bfloat16()
    return hi, (x - hi.float()).bfloat16()


def _rows(shape, kind, g):
    """K or V rows in a cache's form: a list of planes."""
    if kind == "pair":
        return list(_planes(torch.randn(shape, generator=g, device=DEV)))
    return [torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16 if kind == "bf16" else torch.float16)]


def prepare(case, seed):
    c = case
    g = torch.Generator(DEV).manual_seed(seed)
    s = {"case": c}
    ints = dict(dtype=torch.int32, device=DEV)
    if c["op"] == "probs":
        x = 3 * torch.randn(c["rows"], c["vocab"], generator=g, device=DEV)
        s["logits"] = x.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[c["type"]])
        s["temperature"] = 0.5 + torch.rand(c["rows"], generator=g, device=DEV)
        return s
    s["counts"] = torch.tensor(_counts(c), **ints)
    if c["op"] == "attention":
        b, n, h, d = c["batch"], c["nodes"], c["kv_heads"], c["dim"]
        cap = -(-(c["keys"] + n) // 8) * 8
        f = torch.float32 if c["type"] == "pair" else torch.bfloat16 if c["type"] == "bf16" else torch.float16
        s["q"] = (1.5 * torch.randn(b, n, c["heads"], d, generator=g, device=DEV)).to(f)
        for x in "kv":
            shape = (b, h, cap, d) if c["layout"] == "bhsd" else (b, cap, h, d)
            s[x] = [t if c["layout"] == "bhsd" else t.transpose(1, 2) for t in _rows(shape, c["type"], g)]
            s["tree_" + x] = _rows((b, h, n, d), c["type"], g)
        s["lens"] = torch.tensor(_lens(c), **ints)
        s["parents"] = _trees(c, g)
        s["mask"] = _words(_ancestors(s["parents"], s["counts"]))
    elif c["op"] == "verify":
        b, n, v = c["batch"], c["nodes"], c["vocab"]
        x = 3 * torch.randn(b, n, v, generator=g, device=DEV)
        s["target"] = torch.softmax(x, -1)
        x += 0.7 * torch.randn(b, n, v, generator=g, device=DEV)
        s["draft"] = torch.softmax(x, -1)
        del x
        s["parents"] = _trees(c, g, c["width"])
        s["ancestors"] = _ancestors(s["parents"], s["counts"])
        pick = torch.multinomial(s["draft"].flatten(0, 1), c["nodes"], replacement=True, generator=g).view(b, n, n)
        at = s["parents"].long().clamp(min=0)
        s["tokens"] = pick.gather(1, at[:, :, None].expand(-1, -1, n)).diagonal(dim1=1, dim2=2).int().contiguous()
        s["accept_u"] = torch.rand(b, n, generator=g, device=DEV)
        s["sample_u"] = torch.rand(b, generator=g, device=DEV)
    else:
        l, b, n, h, d = c["layers"], c["batch"], c["nodes"], c["kv_heads"], c["dim"]
        cap = c["keys"] + n
        s["cache"] = _rows((l, b, h, cap, d), c["type"], g) + _rows((l, b, h, cap, d), c["type"], g)
        s["tree"] = _rows((l, b, h, n, d), c["type"], g) + _rows((l, b, h, n, d), c["type"], g)
        s["lens"] = torch.tensor([c["keys"] - (37 * i) % (c["keys"] // 2) for i in range(b)], **ints)
        acc = _accepted(c)
        s["accepted"] = torch.tensor(acc, **ints)
        path = torch.full((b, n), -1, **ints)
        for i, a in enumerate(acc):
            path[i, 0] = 0
            if a:
                path[i, 1:a + 1] = (torch.randperm(n - 1, generator=g, device=DEV)[:a].sort().values + 1).int()
        s["path"] = path
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------
@functools.lru_cache(None)
def _framework():
    from ds_ocr_b200.speculative import Speculative
    return Speculative()


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        f = _framework()
        if op == "attention":
            return f.tree_attention(s["q"], s["k"], s["v"], s["tree_k"], s["tree_v"], s["lens"], s["mask"], s["counts"])
        if op == "probs":
            return f.token_probs(s["logits"], s["temperature"])
        if op == "verify":
            return f.verify(s["tokens"], s["parents"], s["target"], s["draft"], s["accept_u"], s["sample_u"], s["counts"])
        lens = f.commit(s["cache"], s["tree"], s["lens"], s["path"], s["accepted"])
        return s["cache"], lens
    return {"attention": _attention, "probs": _probs, "verify": _verify, "commit": _commit}[op](s)


def _whole(planes, dtype=torch.float32):
    return planes[0].to(dtype) if len(planes) == 1 else planes[0].to(dtype) + planes[1].to(dtype)


def _allowed(s, keys):
    """[batch, nodes, keys + nodes]: which cached rows and which nodes of its tree a node attends."""
    n = s["q"].shape[1]
    at = torch.arange(n, device=DEV)
    used = (at < s["counts"][:, None])[:, :, None]
    old = torch.arange(keys, device=DEV) < s["lens"][:, None, None]
    new = (s["mask"][:, :, at // 64] >> (at % 64)) & 1 > 0
    return torch.cat([old & used, new & used & (at < s["counts"][:, None, None])], -1)


def _attention(s, dtype=torch.float32):
    q = s["q"].to(dtype)
    b, n, heads, d = q.shape
    k = torch.cat([_whole(s["k"], dtype), _whole(s["tree_k"], dtype)], 2)
    v = torch.cat([_whole(s["v"], dtype), _whole(s["tree_v"], dtype)], 2)
    h = k.shape[1]
    ok = _allowed(s, s["k"][0].shape[2])[:, None, :, None, :]
    q = q.view(b, n, h, heads // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    x = (q @ k.transpose(2, 3)).view(b, h, n, heads // h, -1) * d ** -0.5
    x = torch.where(ok, x, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(dtype).min)
    p = torch.exp(x - m)
    z = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).view(b, h, n, heads // h, d) / torch.where(z > 0, z, 1)
    return o.permute(0, 2, 1, 3, 4).reshape(b, n, heads, d).to(s["q"].dtype if dtype == torch.float32 else dtype)


def _probs(s):
    x = s["logits"].float() / s["temperature"][:, None]
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _fixed(p):
    return (p.clamp(0, 1) * 2.0 ** FIX).long()


def _verify(s):
    tokens, parents, target, draft = s["tokens"].long(), s["parents"].long(), s["target"], s["draft"]
    b, n, v = target.shape
    at = torch.arange(n, device=DEV)
    real = (at > 0) & (at < s["counts"][:, None])
    same = (parents[:, :, None] == parents[:, None, :]) & real[:, None, :] & real[:, :, None] & (at[None, :] < at[:, None])
    rank = same.sum(-1)
    child = torch.full((b, n, s["case"]["width"] + 1), -1, device=DEV)
    child[torch.arange(b, device=DEV)[:, None].expand(b, n)[real], parents[real], rank[real]] = at.expand(b, n)[real]
    # each node's children in turn: taken with probability r(x) / (mass * d(x)), else r <- max(r - mass * d, 0)
    r, mass, taken = target, torch.ones(b, n, device=DEV), torch.full((b, n), -1, device=DEV)
    for k in range(s["case"]["width"]):
        c = child[:, :, k]
        there, c = (c >= 0) & (taken < 0), c.clamp(min=0)
        x = tokens.gather(1, c)[:, :, None]
        ok = s["accept_u"].gather(1, c) * (draft.gather(2, x)[:, :, 0] * mass) < r.gather(2, x)[:, :, 0]
        taken = torch.where(there & ok, c, taken)
        out = there & ~ok
        r = torch.where(out[:, :, None], (r - mass[:, :, None] * draft).clamp(min=0), r)
        mass = torch.where(out, _fixed(r).sum(-1).float() * 2.0 ** -FIX, mass)
    # a node is on the path if it and all above it were taken; the path's indices ascend
    got = (taken.gather(1, parents.clamp(min=0)) == at) | (at == 0)
    on = ~(s["ancestors"] & ~got[:, None, :]).any(-1) & (at < s["counts"][:, None])
    path = torch.where(on, at, n).sort(-1).values
    accepted = on.sum(-1) - 1
    last = torch.where(on, at, 0).amax(-1)[:, None, None].expand(b, 1, v)
    w = _fixed(r.gather(1, last)[:, 0])
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, _fixed(target.gather(1, last)[:, 0]))
    cum = w.cumsum(-1)
    total, u = cum[:, -1], (s["sample_u"] * 2.0 ** 24).long()
    t = (total >> 24) * u + (((total & 0xffffff) * u) >> 24)
    token = torch.where(total > 0, (cum <= t[:, None]).sum(-1), -1)
    return torch.where(path < n, path, -1).int(), accepted.int(), token.int()


def _commit(s):
    cache, tree, lens = s["cache"], s["tree"], s["lens"].long()
    b, n = s["path"].shape
    j = torch.arange(n, device=DEV)
    use = j <= s["accepted"][:, None]
    at = torch.arange(b, device=DEV)[:, None].expand(b, n)[use]
    to, src = (lens[:, None] + j)[use], s["path"].long()[use]

    def put(c, t):
        c[:, at, :, to] = t[:, at, :, src]
        return c
    return list(map(put, cache, tree)), (lens + s["accepted"] + 1).int()


# ---- the definition in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "probs":
        x = s["logits"].double() / s["temperature"].double()[:, None]
        return torch.softmax(x, -1)
    if op == "attention":
        return _exact_attention(s)
    if op == "verify":
        return _exact_verify(s)
    return None  # rows are copied, none is computed


def _exact_attention(s):
    q = s["q"].double()
    b, n, heads, d = q.shape
    h = s["k"][0].shape[1]
    out = torch.zeros_like(q)
    for i in range(b):
        m, t = int(s["lens"][i]), int(s["counts"][i])
        see = torch.ones(t, m + t, dtype=torch.bool, device=DEV)
        par = s["parents"][i].tolist()
        for r in range(t):
            up, at = set(), r
            while at >= 0:
                up.add(at)
                at = par[at]
            see[r, m:] = torch.tensor([j in up for j in range(t)], device=DEV)
        for j in range(heads):
            g = j // (heads // h)
            k = torch.cat([_whole([p[i, g, :m] for p in s["k"]], torch.float64), _whole([p[i, g, :t] for p in s["tree_k"]], torch.float64)])
            v = torch.cat([_whole([p[i, g, :m] for p in s["v"]], torch.float64), _whole([p[i, g, :t] for p in s["tree_v"]], torch.float64)])
            x = (q[i, :t, j] @ k.T / math.sqrt(d)).masked_fill(~see, -math.inf)
            out[i, :t, j] = torch.softmax(x, -1) @ v
    return out


def _exact_verify(s):
    b, n, v = s["target"].shape
    path, took, token = [], [], []
    for i in range(b):
        par, tok, u = s["parents"][i].tolist(), s["tokens"][i].tolist(), s["accept_u"][i].tolist()
        at, way, r = 0, [0], s["target"][i, 0].double()
        for c in range(1, int(s["counts"][i])):
            if par[c] != at:
                continue
            d = s["draft"][i, at].double()
            if u[c] * float(d[tok[c]]) < float(r[tok[c]]):
                at = c
                way.append(c)
                r = s["target"][i, c].double()
            else:
                r = (r - d).clamp(min=0)
                r = r / r.sum()
        cum = r.cumsum(0)
        token.append(min(v - 1, int((cum <= float(s["sample_u"][i]) * float(cum[-1])).sum())))
        path.append(way + [-1] * (n - len(way)))
        took.append(len(way) - 1)
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (path, took, token))
