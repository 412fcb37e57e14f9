"""Speculative decoding with a tree of drafted tokens: what one step of it asks of the GPU.

Three operators are run here, each in a plain form of elementary torch operations and, where
``own`` is true, as a user's program calls the framework:

* ``tree_attention``: T drafted tokens of every sequence, the nodes of a tree, attend over the
  sequence's paged history and over their own ancestors (and themselves) in the tree. Node i of
  sequence b sits in cache slot kv_lens[b] - T + i; parents[b, i] < i is its parent, -1 none.
* ``verify_drafts``: speculative sampling over that tree from given uniform numbers (or greedily):
  which nodes are kept, and the token that follows them.
* ``keep_path``: the kept nodes' K and V rows move, in every layer's pool, to the slots right behind
  the history, and the sequences' new lengths come back.
"""

import math
import sys
from functools import lru_cache
from pathlib import Path

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@lru_cache(maxsize=None)
def _framework():
    root = str(Path(__file__).resolve().parent.parent / "custom-inference-engine_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from kernels import draft_tree

    return draft_tree


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one request with a handful of drafts over a short prompt: a call whose latency counts
        dict(name="tree attention, one short", op="attention", b=1, t=6, hq=32, hkv=8, d=64, lo=300, hi=300, bs=16, type="bf16"),
        # one user, a wide tree over a long conversation: few sequences, many rows
        dict(name="tree attention, one wide", op="attention", b=1, t=64, hq=32, hkv=8, d=128, lo=8192, hi=8192, bs=16, type="bf16"),
        # a ragged serving batch of a 64-wide model with odd trees
        dict(name="tree attention, odd batch", op="attention", b=12, t=27, hq=32, hkv=8, d=64, lo=256, hi=8192, bs=16, type="fp16"),
        # heads without sharing, pages of 24 tokens that end inside every tile
        dict(name="tree attention, odd pages", op="attention", b=5, t=13, hq=16, hkv=16, d=128, lo=100, hi=4001, bs=24, type="bf16"),
        # the serving batch of the verify benchmark with trees of 16: the cache's bytes count
        dict(name="tree attention, long batch", op="attention", b=32, t=16, hq=32, hkv=8, d=128, lo=1024, hi=32768, bs=16, type="bf16"),
        # four drafted tokens of one request, a small vocabulary: latency
        dict(name="verify, one chain", op="verify", b=1, t=5, branch=1, v=32000, drafts="sampled", type="fp32"),
        # a serving batch's chains of four, sampled from the draft model's probabilities
        dict(name="verify, chains", op="verify", b=32, t=5, branch=1, v=128256, drafts="sampled", type="fp32"),
        # trees of the draft model's best tokens (no draft probabilities), rows of odd length
        dict(name="verify, best-token trees", op="verify", b=16, t=27, branch=3, v=50257, drafts="chosen", type="fp32"),
        # trees verified greedily from 16-bit logits
        dict(name="verify, greedy trees", op="verify", b=8, t=21, branch=4, v=128256, drafts="greedy", type="bf16"),
        # one request's kept path in the sixteen layers of a small model
        dict(name="keep path, one", op="keep", b=1, t=8, n=4, layers=16, hkv=8, d=64, lo=200, hi=200, bs=16, type="bf16"),
        # a serving batch's kept paths
        dict(name="keep path, batch", op="keep", b=64, t=32, n=6, layers=16, hkv=8, d=128, lo=64, hi=500, bs=16, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "verify", "verify", "keep"])
    if op == "attention":
        g = rng.choice([1, 2, 4, 8])
        hkv = rng.choice([1, 2, 4, 8, 16])
        c = dict(op=op, b=_log(rng, 1, 32), t=_log(rng, 1, 100), hq=g * hkv, hkv=hkv, d=rng.choice([32, 64, 64, 128, 128, 256]),
                 lo=0, hi=_log(rng, 130, 32768), bs=rng.choice([8, 16, 16, 16, 20, 32, 64]), type=rng.choice(["bf16", "bf16", "fp16"]))
        while c["b"] * c["hi"] * c["hkv"] * c["d"] > 32 * 16384 * 1024 or c["b"] * c["hq"] * c["t"] * c["hi"] > 32 * 32 * 16 * 16384:
            c["b"], c["hi"] = max(1, c["b"] * 3 // 4), max(130, c["hi"] * 3 // 4)
            c["t"] = max(1, c["t"] * 7 // 8)
        c["lo"] = rng.randint(c["t"], c["hi"])
        return c
    if op == "verify":
        branch = rng.choice([1, 1, 2, 3, 5])
        c = dict(op=op, b=_log(rng, 1, 64), t=rng.randint(2, 9) if branch == 1 else _log(rng, 4, 64), branch=branch,
                 v=rng.choice([_log(rng, 500, 130000), 32000, 50257, 128256]), drafts=rng.choice(["sampled", "sampled", "chosen", "greedy"]),
                 type=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
        while c["b"] * c["t"] * c["v"] > 32 * 5 * 128256:
            c["b"], c["t"] = max(1, c["b"] * 3 // 4), max(2, c["t"] * 7 // 8)
        return c
    t = _log(rng, 2, 64)
    return dict(op=op, b=_log(rng, 1, 64), t=t, n=rng.randint(1, min(t, 9)), layers=rng.randint(1, 24), hkv=rng.choice([1, 2, 4, 8]),
                d=rng.choice([32, 64, 128]), lo=t, hi=t + _log(rng, 1, 400), bs=rng.choice([8, 16, 16, 24, 32]), type=rng.choice(["bf16", "fp16"]))


# ------------------------------------------------------------------ inputs
def _lens(case):
    """Lengths spread evenly from lo to hi: the same for every seed but for their order."""
    b, lo, hi = case["b"], case["lo"], case["hi"]
    return np.array([max(case["t"], hi if b == 1 else lo + (hi - lo) * i // (b - 1)) for i in range(b)], dtype=np.int64)


def _kept(case):
    """Nodes kept by each sequence of a keep case."""
    return np.array([1 + (case["n"] - 1 + i) % case["n"] for i in range(case["b"])], dtype=np.int64)


def _pages(lens, bs, rs):
    """A random page of a pool of just enough pages for each block of each sequence; unused entries are 0."""
    need = -(-lens // bs)
    ids = rs.permutation(int(need.sum())).astype(np.int32)
    table = np.zeros((len(lens), int(need.max())), dtype=np.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = ids[at:at + k]
        at += k
    return table, at


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = _TYPES[case["type"]]

    def cuda(x, dtype):
        return torch.from_numpy(np.ascontiguousarray(x)).to(device="cuda", dtype=dtype)

    def randn(*shape, dtype=kind):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    b, t = case["b"], case["t"]
    if case["op"] == "verify":
        v, branch = case["v"], case["branch"]
        parents = np.array([-1] + [(i - 1) // branch for i in range(1, t)])
        if case["drafts"] != "sampled":  # each request has a tree of its own
            parents = np.stack([parents] + [np.array([-1] + [int(rs.randint(max(0, i - branch), i)) for i in range(1, t)]) for _ in range(b - 1)])
        rows = torch.from_numpy(np.broadcast_to(parents, (b, t)).clip(0)).cuda()
        # a few likely tokens and a long tail; the draft model differs from the target by noise
        target = 2.5 * randn(b, t, v, dtype=torch.float32)
        draft = target + 0.7 * randn(b, t, v, dtype=torch.float32)
        if case["drafts"] == "sampled":
            scores = draft - torch.log(-torch.log(torch.rand(b, t, v, generator=gen, device="cuda").clamp_(1e-12, 1 - 1e-7)))
            tokens = scores.argmax(-1) if branch == 1 else None
            if tokens is None:  # siblings are independent draws from their parent's row
                tokens = torch.stack([(draft[torch.arange(b), rows[:, i]] - torch.log(-torch.log(
                    torch.rand(b, v, generator=gen, device="cuda").clamp_(1e-12, 1 - 1e-7)))).argmax(-1) for i in range(t)], 1)
            else:
                tokens = torch.cat([tokens[:, :1], tokens[:, :-1]], 1)
        else:  # the i-th child of a node is the draft model's i-th best token there
            best = draft.topk(min(v, max(8, t)), -1).indices
            p = np.broadcast_to(parents, (b, t))
            nth = np.array([[int((row[:i] == row[i]).sum()) for i in range(t)] for row in p])
            tokens = best[torch.arange(b, device="cuda")[:, None], rows, cuda(nth, torch.int64)]
        s = dict(tokens=tokens.to(torch.int32), parents=cuda(parents, torch.int32))
        if case["drafts"] == "greedy":
            return dict(case=case, **s, target=target.to(kind), uniforms=None, draft=None)
        uniforms = torch.rand(b, t, generator=gen, device="cuda")
        q = torch.softmax(draft, -1).to(kind) if case["drafts"] == "sampled" else None
        return dict(case=case, **s, target=torch.softmax(target, -1).to(kind), uniforms=uniforms, draft=q)
    lens = rs.permutation(_lens(case))
    table, blocks = _pages(lens, case["bs"], rs)
    s = dict(case=case, tables=cuda(table, torch.int32), lens=cuda(lens, torch.int32))
    shape = (blocks, case["bs"], case["hkv"], case["d"])
    if case["op"] == "attention":
        parents = np.array([[-1] + [int(rs.randint(0, i)) for i in range(1, t)] for _ in range(b)])
        # the model's q as its projection leaves it: (B, T, Hq, D) seen as (B, Hq, T, D)
        return dict(**s, parents=cuda(parents, torch.int32), q=randn(b, t, case["hq"], case["d"]).transpose(1, 2), k=randn(*shape), v=randn(*shape))
    n = rs.permutation(_kept(case))
    path = np.full((b, t), -1)
    for i in range(b):
        path[i, 0] = 0
        path[i, 1:n[i]] = np.sort(rs.permutation(t - 1)[:n[i] - 1]) + 1
    pools = [randn(*shape) for _ in range(2 * case["layers"])]
    return dict(**s, pools=pools, path=cuda(path, torch.int32), n=cuda(n, torch.int32))


# ------------------------------------------------------------------ the calls, and their plain forms
def run(state):
    op = state["case"]["op"]
    if own:
        f = _framework()
        if op == "attention":
            return f.tree_attention(state["q"], state["k"], state["v"], state["tables"], state["lens"], state["parents"])
        if op == "verify":
            return tuple(f.verify_drafts(state["tokens"], state["parents"], state["target"], state["uniforms"], state["draft"]))
        return state["pools"], f.keep_path(state["pools"], state["tables"], state["lens"], state["path"], state["n"])
    return {"attention": _attention, "verify": _verify, "keep": _keep}[op](state)


def _slots(state, pos):
    """Pool rows of the positions pos (B, N) of each sequence."""
    bs = state["case"]["bs"]
    block = state["tables"].long().gather(1, (pos // bs).clamp(0, state["tables"].shape[1] - 1))
    return block * bs + pos % bs


def _attention(s):
    c = s["case"]
    b, t, g = c["b"], c["t"], c["hq"] // c["hkv"]
    n = s["tables"].shape[1] * c["bs"]
    pos = torch.arange(n, device="cuda").expand(b, n)
    at = _slots(s, pos)
    k = s["k"].view(-1, c["hkv"], c["d"])[at].permute(0, 2, 3, 1).float()
    v = s["v"].view(-1, c["hkv"], c["d"])[at].permute(0, 2, 1, 3).float()
    # reach[i, j]: j is i or an ancestor of i
    reach = torch.eye(t, device="cuda").expand(b, t, t) + (s["parents"][:, :, None] == torch.arange(t, device="cuda")).float()
    for _ in range(t.bit_length()):
        reach = (reach @ reach > 0).float()
    node = pos - (s["lens"].long()[:, None] - t)  # (B, N): < 0 is history, >= T is past the end
    seen = (node < 0)[:, None, :] | ((node < t)[:, None, :] & (reach.gather(2, node.clamp(0, t - 1)[:, None, :].expand(b, t, n)) > 0) & (node >= 0)[:, None, :])
    q = s["q"].float().reshape(b, c["hkv"], g * t, c["d"])
    x = (q @ k) / math.sqrt(c["d"])
    x = x.view(b, c["hkv"], g, t, n).masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    return (x.view(b, c["hkv"], g * t, n) @ v).view(b, c["hq"], t, c["d"]).to(s["q"].dtype)


def _verify(s):
    c = s["case"]
    b, t, v = c["b"], c["t"], c["v"]
    tokens, parents = s["tokens"].long(), s["parents"].long().expand(b, t)
    rows = torch.arange(b, device="cuda")
    cur = torch.zeros(b, dtype=torch.long, device="cuda")
    path, out = torch.full_like(tokens, -1), torch.full_like(tokens, -1)
    path[:, 0] = 0
    n = torch.ones_like(cur)
    if s["uniforms"] is None:
        top = s["target"] == s["target"].amax(-1, keepdim=True)
        best = torch.where(top, torch.arange(v, device="cuda"), v).amin(-1)
    else:
        u = s["uniforms"].double()
        p = s["target"].double()
        r = torch.where(p[:, 0] > 0, p[:, 0], 0.0)  # what is left of the current node's row
        mass = torch.ones(b, dtype=torch.double, device="cuda")
    # A child's index is above its parent's, so one ascending pass over the nodes is the whole walk.
    for i in range(1, t):
        tested, x = parents[:, i] == cur, tokens[:, i]
        if s["uniforms"] is None:
            kept = tested & (best[rows, cur] == x)
        else:
            q = s["draft"][rows, cur].double() if s["draft"] is not None else torch.zeros_like(r).scatter_(1, x[:, None], 1.0)
            kept = tested & (u[:, i] * q[rows, x] * mass < r[rows, x])
            lost = tested & ~kept
            if s["draft"] is not None:
                rest = r - mass[:, None] * q
                rest = torch.where(rest > 0, rest, 0.0)
                less = rest.sum(-1)
            else:
                rest = r * (1.0 - q)
                less = mass - r[rows, x]
            r = torch.where(lost[:, None], rest, r)
            mass = torch.where(lost, less, mass)
            nxt = p[:, i]
            r = torch.where(kept[:, None], torch.where(nxt > 0, nxt, 0.0), r)
            mass = torch.where(kept, 1.0, mass)
        cur = torch.where(kept, i, cur)
        out[rows, n - 1] = torch.where(kept, x, out[rows, n - 1])
        path[rows, n.clamp(max=t - 1)] = torch.where(kept, i, path[rows, n.clamp(max=t - 1)])
        n = n + kept
    if s["uniforms"] is None:
        last = best[rows, cur]
    else:
        whole = torch.where(p[rows, cur] > 0, p[rows, cur], 0.0)
        r = torch.where(r.sum(-1, keepdim=True) > 0, r, whole)
        cum = r.cumsum(-1)
        want = u[:, :1].clamp(max=1.0 - 2.0 ** -24) * cum[:, -1:]
        last = (cum <= want).sum(-1).clamp(max=v - 1)
    out[rows, n - 1] = last
    return out.to(s["tokens"].dtype), path.to(torch.int32), n.to(torch.int32)


def _keep(s):
    t = s["case"]["t"]
    base = s["lens"].long()[:, None] - t
    i = torch.arange(t, device="cuda")[None]
    live = i < s["n"][:, None]
    to = _slots(s, base + i)
    source = torch.where(live, _slots(s, base + s["path"].long().clamp(min=0)), to)
    for pool in s["pools"]:
        flat = pool.view(-1, *pool.shape[2:])
        flat[to] = flat[source]
    return s["pools"], (base[:, 0] + s["n"]).to(torch.int32)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b, t, e = case["b"], case["t"], 4 if case["type"] == "fp32" else 2
    if case["op"] == "attention":
        keys = int(_lens(case).sum())
        kv = 2 * keys * case["hkv"] * case["d"] * e
        return {"bytes": kv + 2 * b * t * case["hq"] * case["d"] * e + 4 * (keys // case["bs"] + b * t + b), "flops": 4 * keys * case["hq"] * t * case["d"]}
    if case["op"] == "verify":
        # one row of the target to draw the last token from (greedy: one for each node on a path of
        # about two), one of the draft's where a draft was refused, the nodes' own entries
        lines = {"sampled": 2, "chosen": 1, "greedy": 2}[case["drafts"]]
        return {"bytes": b * lines * case["v"] * e + b * t * (4 * 5 + 2 * e), "flops": b * lines * case["v"] * 2}
    moved = int((_kept(case) - 1).sum())
    return {"bytes": 2 * moved * 2 * case["layers"] * case["hkv"] * case["d"] * e + b * t * 4 * 2 + b * 12, "flops": 0}


# ------------------------------------------------------------------ 64 bits, written apart from the plain forms
def exact(case, seed):
    s = prepare(case, seed)
    t = case["t"]
    if case["op"] == "attention":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        g = case["hq"] // case["hkv"]
        parents, lens, tables = s["parents"].cpu().numpy(), s["lens"].cpu().numpy(), s["tables"].long()
        for b in range(case["b"]):
            n = int(lens[b])
            seen = torch.ones(t, n, dtype=torch.bool)
            seen[:, n - t:] = False
            for i in range(t):
                j = i
                while j >= 0:
                    seen[i, n - t + j] = True
                    j = int(parents[b, j])
            seen = seen.cuda()
            pages = tables[b, : -(-n // case["bs"])]
            k = s["k"][pages].flatten(0, 1)[:n].double()
            v = s["v"][pages].flatten(0, 1)[:n].double()
            for h in range(case["hq"]):
                x = s["q"][b, h].double() @ k[:, h // g].T * case["d"] ** -0.5
                x = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                out[b, h] = x @ v[:, h // g]
        return out
    if case["op"] == "verify":
        parents = np.broadcast_to(s["parents"].cpu().numpy(), (case["b"], t))
        tokens = s["tokens"].cpu().numpy()
        out, path, count = np.full((case["b"], t), -1), np.full((case["b"], t), -1), np.zeros(case["b"], int)
        for b in range(case["b"]):
            row = lambda m, i: m[b, i].double().cpu().numpy()  # noqa: E731,B023
            u = None if s["uniforms"] is None else s["uniforms"][b].double().cpu().numpy()
            walk, node = [0], 0
            while node is not None:
                here, node = node, None
                p = row(s["target"], here)
                if u is None:
                    last = int(p.argmax())
                    node = next((c for c in range(here + 1, t) if parents[b, c] == here and tokens[b, c] == last), None)
                else:
                    left, mass = np.maximum(p, 0), 1.0
                    q = None if s["draft"] is None else row(s["draft"], here)
                    for c in range(here + 1, t):
                        if parents[b, c] != here:
                            continue
                        x = int(tokens[b, c])
                        if u[c] * (1.0 if q is None else q[x]) * mass < left[x]:
                            node = c
                            break
                        if q is None:
                            mass, left[x] = mass - left[x], 0.0
                        else:
                            left = np.maximum(left - mass * q, 0)
                            mass = left.sum()
                    if node is None:
                        left = left if left.sum() > 0 else np.maximum(p, 0)
                        cum = left.cumsum()
                        last = min(int(np.searchsorted(cum, min(u[0], 1 - 2.0 ** -24) * cum[-1], side="right")), len(cum) - 1)
                if node is not None:
                    walk.append(node)
            count[b] = len(walk)
            path[b, :len(walk)] = walk
            out[b, :len(walk)] = [int(tokens[b, c]) for c in walk[1:]] + [last]
        return torch.from_numpy(out).to(torch.int32), torch.from_numpy(path).to(torch.int32), torch.from_numpy(count).to(torch.int32)
    lens, n, path, tables = (s[k].cpu().numpy() for k in ("lens", "n", "path", "tables"))
    place = lambda b, p: (int(tables[b, p // case["bs"]]), int(p % case["bs"]))  # noqa: E731
    moves = [(place(b, lens[b] - t + path[b, i]), place(b, lens[b] - t + i)) for b in range(case["b"]) for i in range(1, n[b])]
    pools = []
    for pool in s["pools"]:
        new = pool.clone()
        if moves:
            (sb, so), (db, do) = (torch.tensor(m).T.cuda() for m in zip(*moves))
            new[db, do] = pool[sb, so]
        pools.append(new)
    return pools, torch.from_numpy(lens - t + n).to(torch.int32)
