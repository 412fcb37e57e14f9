"""Plain 64-bit restatements of the tree-of-drafts operators, and the error bounds that
the tests hold the kernels to."""

from __future__ import annotations

import math

import numpy as np
import torch


def half_step(dtype) -> float:
    """A rounding to ``dtype`` is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def ancestors(parents) -> torch.Tensor:
    """(T, T) bool: [i, j] is True when j is node i or one of its ancestors."""
    T = len(parents)
    seen = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        j = i
        while j >= 0:
            seen[i, j] = True
            j = int(parents[j])
    return seen


def depths(parents) -> list[int]:
    return [int(r.sum()) - 1 for r in ancestors(parents)]


def rotate(x, cos, sin, pos):
    """Half-split rotation of x (..., T, D) at positions pos (T,), in 64 bits."""
    h = x.shape[-1] // 2
    c, s = cos.double()[pos], sin.double()[pos]
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def tree_attention_ref(q, k_pool, v_pool, tables, lens, parents, scale=None, rope=None):
    """(out, bound), both float64 (B, Hq, T, D).

    ``bound`` counts the kernel's roundings, h = half a step of q's type:
      * the output's own:                    h |o|
      * P, rounded once per key for bf16:    h A,  A = sum_j p_j |v_j|
        (fp16 P is held as two halves:       2^-21 A covers both)
      * a score off by e makes p_j / sum p off by up to 2 e relative:  2 e A, with
        e = fp32 sum of D products and the scaling, (D + 4) 2^-24 of sum |q k| scale,
        2^-21 for the exponential (its own error and its argument's), and, when q is
        rotated, the rotated q's rounding, h of sum |q k| scale
      * partitions: log-sum-exps and their weights, fp32, 2^-18 A
    """
    B, Hq, T, D = q.shape
    nb, bs, Hkv, _ = k_pool.shape
    h = half_step(q.dtype)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    par = parents.cpu()
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        tree = par if par.ndim == 1 else par[b]
        anc = ancestors(tree).to(q.device)
        seen = torch.ones(T, n, dtype=torch.bool, device=q.device)
        lo = max(0, n - T)
        seen[:, lo:] = anc[:, T - (n - lo):]
        pages = tables[b, : -(-n // bs)].long()
        k = k_pool[pages].flatten(0, 1)[:n].double()
        v = v_pool[pages].flatten(0, 1)[:n].double()
        x = q[b].double()
        if rope is not None:
            pos = torch.tensor([n - T + d for d in depths(tree)], device=q.device)
            x = rotate(x, *rope, pos.clamp(0, rope[0].shape[0] - 1))
        for hd in range(Hq):
            kh, vh = k[:, hd // (Hq // Hkv)], v[:, hd // (Hq // Hkv)]
            s = (x[hd] @ kh.T) * scale
            s = torch.where(seen, s, -math.inf)
            p = torch.softmax(s, -1)
            p = torch.where(seen, p, 0.0)
            # 0 x NaN of a masked row must not count: rows that no node may see here
            some = seen.any(0)
            vals = torch.where(some[:, None], vh, 0.0)
            o = torch.zeros(T, D, dtype=torch.float64, device=q.device)
            a = torch.zeros_like(o)
            clean = torch.isfinite(vals).all(-1)
            o += p[:, clean] @ vals[clean]
            a += p[:, clean] @ vals[clean].abs()
            for j in torch.nonzero(~clean).flatten().tolist():
                hit = seen[:, j]
                o[hit] += p[hit, j, None] * vals[j]
                a[hit] += p[hit, j, None] * vals[j].abs()
            mag = torch.where(seen, (x[hd].abs() @ torch.nan_to_num(kh, 0, 0, 0).abs().T) * abs(scale), 0.0).amax(-1, keepdim=True)
            e = mag * ((D + 4) * 2.0 ** -24 + (h if rope is not None else 0.0)) + 2.0 ** -21
            o[~seen.any(-1)] = math.nan
            out[b, hd] = o
            bound[b, hd] = h * o.abs() + a * ((h if q.dtype == torch.bfloat16 else 2.0 ** -21) + 2 * e + 2.0 ** -18)
    return out, bound


def assert_within(got, ref, bound, what=""):
    got = got.double()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places ({int(torch.isnan(got).sum())} for {int(nan.sum())})"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities differ"
    ok = ~nan & ~inf
    over = (got - ref).abs()[ok] - bound[ok] - 1e-30
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} beyond the bound, by up to {float(over.max()):.3e}"


def verify_ref(tokens, parents, target, uniforms=None, draft=None):
    """(tokens, path, n) as lists, straight from the definition, numpy float64."""
    tokens = tokens.cpu().numpy()
    B, T = tokens.shape
    par = np.broadcast_to(parents.cpu().numpy(), (B, T))
    p_all = target.double().cpu().numpy()
    q_all = None if draft is None else draft.double().cpu().numpy()
    u_all = None if uniforms is None else uniforms.double().cpu().numpy()
    V = p_all.shape[2]
    outs, paths, ns = [], [], []
    pos = lambda a: np.where(a > 0, a, 0.0)  # noqa: E731  NaN counts as nothing
    for b in range(B):
        path, cur = [0], 0
        while True:
            p = p_all[b, cur]
            kids = [c for c in range(cur + 1, T) if par[b, c] == cur]
            if q_all is not None and cur >= q_all.shape[1]:
                kids = []
            kept, last = None, None
            if u_all is None:
                last = int(np.argmax(p))
                kept = next((c for c in kids if tokens[b, c] == last), None)
            else:
                r, m = pos(p), 1.0
                for c in kids:
                    x = int(tokens[b, c])
                    inside = 0 <= x < V
                    qx = (1.0 if inside else 0.0) if q_all is None else (q_all[b, cur, x] if inside else 0.0)
                    rx = r[x] if inside else 0.0
                    if u_all[b, c] * (1.0 if q_all is None else qx) * m < rx:
                        kept = c
                        break
                    if q_all is None:
                        m -= rx
                        if inside:
                            r = r.copy()
                            r[x] = 0.0
                    else:
                        r = pos(r - m * q_all[b, cur])
                        m = r.sum()
                if kept is None:
                    if not r.sum() > 0:
                        r = pos(p)
                    cum = np.cumsum(r)
                    if not cum[-1] > 0 or np.isinf(cum[-1]):
                        last = -1
                    else:
                        last = int((cum <= min(u_all[b, 0], 1 - 2.0 ** -24) * cum[-1]).sum())
                        last = min(last, int(np.nonzero(r)[0][-1]))
            if kept is None:
                break
            path.append(kept)
            cur = kept
        n = len(path)
        outs.append([int(tokens[b, c]) for c in path[1:]] + [last] + [-1] * (T - n))
        paths.append(path + [-1] * (T - n))
        ns.append(n)
    return outs, paths, ns
