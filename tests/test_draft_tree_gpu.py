"""The tree-of-drafts operators (kernels.draft_tree) on the GPU against 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.tree_ref import (ancestors, assert_within, depths, rotate, tree_attention_ref,
                            verify_ref)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_status(cuda):
    from kernels import _lib

    _lib.device_status()
    yield
    assert _lib.device_status() == 0, "a kernel raised a status bit that the test did not expect"


def tree(kind, T, rs):
    if kind == "chain":
        return [i - 1 for i in range(T)]
    if kind == "star":
        return [-1] + [0] * (T - 1)
    if kind == "roots":
        return [-1] * T
    if kind == "binary":
        return [-1] + [(i - 1) // 2 for i in range(1, T)]
    return [-1] + [int(rs.randint(0, i)) for i in range(1, T)]


def setup(B, T, Hq, Hkv, D, bs, dtype, lens, kind="random", seed=0, extra=3):
    """A pool with more pages than needed; the rows that no sequence holds are NaN."""
    rs = np.random.RandomState(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens = [int(x) for x in lens]
    need = [-(-n // bs) for n in lens]
    total = sum(need) + extra
    ids = rs.permutation(total)
    table = np.full((B, max(need + [1])), 0, dtype=np.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    k, v = rnd(total, bs, Hkv, D), rnd(total, bs, Hkv, D)
    used = torch.zeros(total * bs, dtype=torch.bool)
    for b in range(B):
        for t in range(lens[b]):
            used[int(table[b, t // bs]) * bs + t % bs] = True
    for pool in (k, v):
        pool.view(total * bs, Hkv, D)[~used.cuda()] = float("nan")
    parents = torch.tensor([tree(kind, T, rs) for _ in range(B)], dtype=torch.int32, device="cuda")
    return dict(q=rnd(B, Hq, T, D), k=k, v=v, tables=torch.from_numpy(table).cuda(),
                lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), parents=parents)


def rope_tables(D, n=4096):
    f = 10000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
    a = torch.arange(n, device="cuda").double()[:, None] * f
    return a.cos().float(), a.sin().float()


def run(s, **kw):
    from kernels.draft_tree import tree_attention

    return tree_attention(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"], **kw)


def check(s, what="", **kw):
    out = run(s, **kw)
    ref_kw = {k: v for k, v in kw.items() if k in ("scale", "rope")}
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"], **ref_kw)
    assert_within(out, ref, bound, what)
    return out


ATTN = [
    # B, T, Hq, Hkv, D, bs, dtype, lens, tree
    (1, 1, 4, 1, 64, 16, BF16, [1], "chain"),
    (1, 1, 32, 8, 128, 16, FP16, [777], "chain"),
    (2, 2, 4, 4, 64, 16, BF16, [2, 3], "star"),
    (3, 7, 6, 2, 64, 16, BF16, [7, 8, 500], "random"),
    (3, 5, 32, 8, 128, 16, BF16, [300, 5, 1023], "binary"),
    (2, 13, 9, 3, 128, 24, FP16, [130, 1500], "random"),
    (2, 16, 8, 1, 64, 32, FP16, [47, 2049], "random"),
    (1, 17, 16, 4, 128, 16, BF16, [4000], "random"),
    (4, 33, 8, 2, 128, 16, BF16, [33, 64, 128, 129], "random"),
    (2, 31, 4, 4, 16, 8, BF16, [90, 300], "random"),
    (2, 40, 8, 4, 32, 16, FP16, [41, 555], "binary"),
    (2, 12, 4, 2, 256, 16, BF16, [100, 700], "random"),
    (2, 64, 32, 8, 128, 16, BF16, [64, 1111], "random"),
    (1, 64, 8, 1, 64, 16, FP16, [700], "random"),
    (2, 100, 8, 2, 128, 16, FP16, [100, 611], "random"),
    (1, 130, 4, 2, 64, 64, BF16, [3001], "chain"),
    (1, 257, 2, 1, 128, 16, BF16, [300], "random"),
    (1, 300, 2, 2, 64, 4, BF16, [1300], "random"),
    (1, 1024, 2, 1, 64, 16, BF16, [1030], "random"),
    (1, 1024, 1, 1, 32, 16, FP16, [1024], "chain"),
    (2, 9, 4, 2, 64, 5, BF16, [23, 61], "roots"),
    (3, 6, 5, 1, 128, 16, BF16, [2500, 6, 33], "star"),
    (3, 18, 8, 2, 128, 20, FP16, [18, 700, 1999], "random"),
    (2, 40, 8, 4, 64, 12, BF16, [1234, 2500], "binary"),
    (2, 7, 4, 4, 128, 1, BF16, [90, 400], "random"),
]


@pytest.mark.parametrize("B,T,Hq,Hkv,D,bs,dtype,lens,kind", ATTN)
def test_tree_attention(B, T, Hq, Hkv, D, bs, dtype, lens, kind):
    check(setup(B, T, Hq, Hkv, D, bs, dtype, lens, kind, seed=T + D))


@pytest.mark.parametrize("split", [16, 48, 256])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,bs,dtype,lens,kind", [ATTN[4], ATTN[5], ATTN[12], ATTN[10], ATTN[14], ATTN[22]])
def test_tree_attention_partitions(B, T, Hq, Hkv, D, bs, dtype, lens, kind, split):
    check(setup(B, T, Hq, Hkv, D, bs, dtype, lens, kind, seed=3), split_tokens=split)


@pytest.mark.parametrize("B,T,Hq,Hkv,D,bs,dtype,lens,kind", [ATTN[3], ATTN[4], ATTN[11], ATTN[12], ATTN[15]])
def test_tree_attention_rope(B, T, Hq, Hkv, D, bs, dtype, lens, kind):
    check(setup(B, T, Hq, Hkv, D, bs, dtype, lens, kind, seed=4), rope=rope_tables(D), scale=0.11)


def test_tree_attention_shared_tree():
    s = setup(3, 11, 8, 2, 64, 16, BF16, [11, 200, 90], seed=5)
    s["parents"] = s["parents"][0].clone()
    check(s)


@pytest.mark.parametrize("D,T,Hq,bs", [(128, 32, 32, 16), (64, 12, 32, 16), (64, 48, 32, 24), (128, 40, 64, 16), (128, 20, 32, 20), (64, 6, 32, 10)])
def test_tree_attention_many_units(D, T, Hq, bs):
    """More work than fits on the GPU at once, in ragged sequences: every pipeline wait ends (the
    status word stays clear) and repeated calls agree bit for bit."""
    rs = np.random.RandomState(D + T)
    s = setup(32, T, Hq, 8, D, bs, BF16, [int(x) for x in rs.randint(T, 6000, 32)], seed=21)
    out = run(s)
    for _ in range(10):
        assert torch.equal(run(s), out)
    pick = [0, 13, 31]
    ref, bound = tree_attention_ref(s["q"][pick], s["k"], s["v"], s["tables"][pick], s["lens"][pick], s["parents"][pick])
    assert_within(out[pick], ref, bound)


@pytest.mark.parametrize("B,T,Hq,Hkv,D,bs,lens", [
    (700, 3, 4, 2, 64, 16, lambda rs: [int(x) * int(y) for x, y in zip(rs.randint(3, 90, 700), rs.rand(700) > 0.3)]),  # many, a third idle
    (300, 4, 4, 4, 128, 8, lambda rs: [2500] + [int(x) for x in rs.randint(0, 60, 298)] + [1900]),                     # two long among short
    (3, 40, 320, 40, 64, 16, lambda rs: [700, 41, 40]),                                                               # more head groups than CTAs for one part each
    (1, 50, 256, 1, 128, 16, lambda rs: [1500]),                                                                      # a hundred row groups
])
def test_tree_attention_batches(B, T, Hq, Hkv, D, bs, lens):
    rs = np.random.RandomState(B)
    s = setup(B, T, Hq, Hkv, D, bs, BF16, lens(rs), "random", seed=B)
    out = run(s)
    pick = sorted(set([0, B - 1] + [int(x) for x in rs.randint(0, B, 40)]))
    ref, bound = tree_attention_ref(s["q"][pick], s["k"], s["v"], s["tables"][pick], s["lens"][pick], s["parents"][pick])
    assert_within(out[pick], ref, bound)
    idle = [b for b in range(B) if int(s["lens"][b]) == 0]
    assert not idle or float(out[idle].abs().max()) == 0.0


def test_tree_attention_length_beyond_the_table(cuda):
    """A length that the table cannot hold is reported and cut to what it holds."""
    from kernels import _lib

    for D, T in ((128, 6), (32, 6)):
        s = setup(2, T, 8, 2, D, 16, BF16, [128, 100], seed=23)
        s["k"].nan_to_num_(0)
        s["v"].nan_to_num_(0)
        want = run(s)
        s["lens"][0] = 5000
        out = run(s)
        assert _lib.device_status() == _lib.CIE_DEV_BAD_BLOCK_ID
        assert torch.equal(out, want)


def test_pools_beyond_32_bits():
    """Pages behind the first 4 GB of a pool: attention, append and the kept path."""
    from kernels.draft_tree import keep_path
    from kernels.flash_attention import rope_append

    D, Hkv, T, nb = 128, 8, 7, 140_000                       # 4.6 GB a pool
    s = setup(2, T, 16, Hkv, D, 16, BF16, [300, 90], seed=24)
    big = dict(s, k=torch.empty(nb, 16, Hkv, D, dtype=BF16, device="cuda"), v=torch.empty(nb, 16, Hkv, D, dtype=BF16, device="cuda"))
    n = s["k"].shape[0]
    big["k"][nb - n:], big["v"][nb - n:] = s["k"], s["v"]
    big["tables"] = s["tables"] + (nb - n)
    assert torch.equal(run(big), run(s))
    kn, vn = torch.randn(2, T, Hkv, D, device="cuda").to(BF16), torch.randn(2, T, Hkv, D, device="cuda").to(BF16)
    path = torch.tensor([[0, 2, 5, -1, -1, -1, -1], [0, 1, 3, 6, -1, -1, -1]], dtype=torch.int32, device="cuda")
    kept = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    for x in (s, big):
        rope_append(kn, vn, x["k"], x["v"], x["tables"], x["lens"] - T, rope=rope_tables(D), parents=x["parents"])
        keep_path([x["k"], x["v"]], x["tables"], x["lens"], path, kept)
    for name in "kv":
        assert torch.equal(big[name][nb - n:].view(torch.int16), s[name].view(torch.int16))


@pytest.mark.parametrize("D,Hq,Hkv,T", [(64, 8, 2, 6), (128, 8, 2, 40), (32, 4, 4, 6)])
def test_tree_attention_idle_and_short_sequences(D, Hq, Hkv, T):
    """A sequence of length 0 gives zeros; one shorter than the tree has no slots for its first nodes."""
    s = setup(4, T, Hq, Hkv, D, 16, BF16, [0, T - 2, 1, T + 100], "random", seed=6)
    out = check(s)
    assert float(out[0].abs().max()) == 0.0
    assert bool(torch.isnan(out[1, :, :2]).all())


@pytest.mark.parametrize("D,dtype,T,bad", [(64, BF16, 9, "nan"), (128, FP16, 9, "inf"), (128, BF16, 50, "nan"), (64, FP16, 70, "inf"), (32, BF16, 20, "nan"), (256, FP16, 5, "nan")])
def test_tree_attention_bad_values_stay_where_they_are_seen(D, dtype, T, bad):
    s = setup(2, T, 8, 2, D, 16, dtype, [T + 40, T + 333], "random", seed=7)
    x = float(bad)
    for b in range(2):
        base = int(s["lens"][b]) - T
        for node, pool in ((T - 1, "v"), (T // 2, "v"), (T - 2, "k")):
            t = base + node
            s[pool][int(s["tables"][b, t // 16]), t % 16] = x
        t = base + T // 3
        s["v"][int(s["tables"][b, t // 16]), t % 16, :, 3] = -x
    got = run(s, split_tokens=64)
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"])
    clean = torch.isfinite(ref).all(-1)
    assert bool(clean.any()) and not bool(clean.all())
    assert_within(got[clean], ref[clean], bound[clean])
    # what sees a NaN or an infinity is no finite number either
    assert not bool((torch.isfinite(got.double()) & torch.isnan(ref)).any())


def test_tree_attention_strides_and_out():
    s = setup(2, 10, 8, 2, 64, 16, BF16, [80, 300], seed=8)
    want = run(s)
    qt = s["q"].transpose(1, 2).contiguous().transpose(1, 2)             # (B, T, H, D) storage
    assert torch.equal(run({**s, "q": qt}), want)
    odd = torch.empty(s["q"].numel() + 3, dtype=BF16, device="cuda")[3:].view_as(s["q"])
    odd.copy_(s["q"])
    assert torch.equal(run({**s, "q": odd}), want)                       # an unaligned base
    wide = torch.full((2, 8, 10, 192), 7.0, dtype=BF16, device="cuda")
    out = run(s, out=wide[..., 64:128])
    assert torch.equal(out, want) and float(wide[..., :64].min()) == 7.0 == float(wide[..., 128:].max())
    lone = torch.zeros(2, 8, 10, 67, dtype=BF16, device="cuda")[..., 1:65]  # rows at odd offsets
    assert torch.equal(run(s, out=lone), want)
    tables = torch.stack([s["tables"], s["tables"]], -1)[..., 0]
    parents = torch.stack([s["parents"], s["parents"]], -1)[..., 0]
    assert torch.equal(run({**s, "tables": tables, "parents": parents}), want)
    both = torch.cat([s["parents"], s["parents"].flip(0)], 1)[:, :10]
    assert torch.equal(run({**s, "parents": both}), want)
    assert run({**s, "q": s["q"][:, :, :0], "parents": s["parents"][:, :0]}).shape == (2, 8, 0, 64)


@pytest.mark.parametrize("D,T", [(128, 5), (64, 5), (128, 40)])
def test_tree_attention_chain_is_paged_attention(D, T):
    from kernels.flash_attention import paged_attention

    s = setup(3, T, 16, 4, D, 16, BF16, [T, 200, 1000], "chain", seed=9)
    rope = rope_tables(D)
    a = run(s, rope=rope).double()
    b = paged_attention(s["q"], s["k"].nan_to_num(0), s["v"].nan_to_num(0), s["tables"], s["lens"], True, rope=rope).double()
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"], rope=rope)
    assert float(((a - b).abs() - 2 * bound).max()) <= 0


def test_tree_attention_bad_parents_are_roots(cuda):
    from kernels import _lib

    s = setup(1, 6, 4, 2, 64, 16, BF16, [50], seed=10)
    s["parents"] = torch.tensor([[-1, 0, 5, 2, -7, 4]], dtype=torch.int32, device="cuda")
    out = run(s)
    assert _lib.device_status() == _lib.CIE_DEV_BAD_TREE
    s["parents"] = torch.tensor([[-1, 0, -1, 2, -1, 4]], dtype=torch.int32, device="cuda")
    assert torch.equal(out, run(s))


@pytest.mark.parametrize("D,T,bs", [(64, 6, 16), (128, 40, 16), (64, 6, 12), (128, 6, 24), (32, 6, 12)])
def test_tree_attention_bad_block_id(cuda, D, T, bs):
    from kernels import _lib

    s = setup(2, T, 4, 2, D, bs, BF16, [300, 400], seed=11)
    want = run(s)
    s["tables"][0, 3] = s["k"].shape[0] + 5
    s["tables"][0, 7] = -3
    out = run(s)
    assert _lib.device_status() & _lib.CIE_DEV_BAD_BLOCK_ID
    assert torch.equal(out[1], want[1])
    assert bool(torch.isfinite(out[0]).all())


@pytest.mark.parametrize("D,T,Hq", [(64, 6, 8), (128, 48, 16)])
def test_tree_attention_graph_and_streams(D, T, Hq):
    """Captured once, replayed over other lengths, trees and values; two graphs of one workspace pool."""
    s = setup(2, T, Hq, 2, D, 16, BF16, [900, 1200], seed=12)
    t = setup(2, T, Hq, 2, D, 16, BF16, [T + 1, 1201], seed=13)
    t["tables"] = torch.nn.functional.pad(t["tables"], (0, s["tables"].shape[1] - t["tables"].shape[1]))if t["tables"].shape[1] < s["tables"].shape[1] else t["tables"]
    want_s, want_t = run(s), run(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run(s), want_s)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = run(s)
    with torch.cuda.graph(g2, pool=g1.pool()):
        o2 = run(t)
    for _ in range(2):
        g1.replay()
        assert torch.equal(o1, want_s)
        g2.replay()
        assert torch.equal(o2, want_t)
    s["q"].copy_(s["q"].flip(2))
    s["lens"].copy_(torch.tensor([700, 1000], dtype=torch.int32))
    s["parents"][0] = torch.arange(-1, T - 1, dtype=torch.int32)
    s["k"].nan_to_num_(0)
    s["v"].nan_to_num_(0)
    g1.replay()
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"])
    assert_within(o1, ref, bound)


@pytest.mark.parametrize("D,bs,T", [(128, 16, 8), (64, 20, 30), (32, 16, 8)])
def test_tree_attention_wait_that_runs_out(cuda, D, bs, T):
    """With a wait limit of 0 the kernels give up at the first wait that is not over at once, say so in
    the status word and leave the context usable. (At d = 32 the tiles, out of L2, may all be there in
    time: then no wait ran out, and the output is the right one.)"""
    from kernels import _lib

    rs = np.random.RandomState(22)
    s = setup(16, T, 16, 4, D, bs, BF16, [int(x) for x in rs.randint(3000, 6000, 16)], seed=22)
    want = run(s)
    torch.cuda.synchronize()
    old = _lib.set_wait_limit(0)
    try:
        out = run(s)
        torch.cuda.synchronize()
    finally:
        _lib.set_wait_limit(old)
    status = _lib.device_status()
    assert status == _lib.CIE_DEV_TIMEOUT or (D == 32 and status == 0 and torch.equal(out, want))
    for _ in range(3):
        assert torch.equal(run(s), want)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("D,Hkv,dtype", [(64, 2, BF16), (128, 8, FP16), (16, 1, BF16)])
def test_rope_append_of_a_tree(D, Hkv, dtype):
    from kernels.flash_attention import apply_rotary, rope_append

    T, bs = 9, 16
    s = setup(2, T, Hkv, Hkv, D, bs, dtype, [30, T], seed=14)
    cos, sin = rope_tables(D)
    start = s["lens"] - T
    kn, vn = torch.randn(2, T, Hkv, D, device="cuda").to(dtype), torch.randn(2, T, Hkv, D, device="cuda").to(dtype)
    k0, v0 = s["k"].clone(), s["v"].clone()
    rope_append(kn, vn, s["k"], s["v"], s["tables"], start, rope=(cos, sin), parents=s["parents"])
    for b in range(2):
        dep = depths(s["parents"][b].cpu())
        for i in range(T):
            t = int(start[b]) + i
            at = (int(s["tables"][b, t // bs]), t % bs)
            rot = apply_rotary(kn[b, i][None, :, None], cos, sin, int(start[b]) + dep[i])[0, :, 0]
            assert torch.equal(s["k"][at], rot) and torch.equal(s["v"][at], vn[b, i])
            exact = rotate(kn[b, i][:, None].double(), cos, sin, torch.tensor([int(start[b]) + dep[i]], device="cuda"))[:, 0]
            assert float(((s["k"][at].double() - exact).abs() - torch.finfo(dtype).eps / 2 * exact.abs() - 1e-6).max()) <= 0
            k0[at], v0[at] = s["k"][at], vn[b, i]
    assert torch.equal(s["k"].view(torch.int16), k0.view(torch.int16)) and torch.equal(s["v"].view(torch.int16), v0.view(torch.int16))


# ------------------------------------------------------------------ verify
def probs(B, T, V, seed, dtype=FP32, sharp=2.0, mix=0.7):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    a = sharp * torch.randn(B, T, V, generator=gen, device="cuda")
    d = a + mix * torch.randn(B, T, V, generator=gen, device="cuda")
    u = torch.rand(B, T, generator=gen, device="cuda")
    return torch.softmax(a, -1).to(dtype), torch.softmax(d, -1).to(dtype), u


def drafted(q, parents, seed):
    """Children drawn from their parents' rows of q (nodes of parent -1: any token)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, T, V = q.shape
    par = parents.expand(B, T).long().clamp(0)
    rows = q.float().gather(1, par[:, :, None].expand(B, T, V)).clamp_min(1e-30)
    g = -torch.log(-torch.log(torch.rand(B, T, V, generator=gen, device="cuda").clamp(1e-9, 1 - 1e-7)))
    return (rows.log() + g).argmax(-1)


def check_verify(tokens, parents, target, uniforms=None, draft=None):
    from kernels.draft_tree import verify_drafts

    got = verify_drafts(tokens, parents, target, uniforms, draft)
    want = verify_ref(tokens, parents, target, uniforms, draft)
    assert got.tokens.dtype == tokens.dtype and got.path.dtype == got.n.dtype == torch.int32
    for g, w in zip(got, want):
        assert g.tolist() == w
    return got


VERIFY = [(1, 2, 1, "chain"), (3, 1, 7, "chain"), (4, 5, 2, "chain"), (8, 5, 31, "chain"), (5, 9, 1023, "random"), (4, 6, 1024, "star"),
          (3, 12, 1025, "binary"), (4, 5, 33000, "chain"), (3, 30, 9001, "random"), (2, 7, 50257, "star"), (2, 40, 128256, "random"), (40, 4, 300, "chain"),
          (2, 100, 500, "binary"), (1, 1024, 64, "random"), (2, 70, 70, "star")]


@pytest.mark.parametrize("B,T,V,kind", VERIFY)
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("mode", ["sampled", "chosen", "greedy"])
def test_verify(B, T, V, kind, dtype, mode):
    rs = np.random.RandomState(T)
    parents = torch.tensor([tree(kind, T, rs) for _ in range(B)], dtype=torch.int32, device="cuda")
    for seed in range(3):
        p, q, u = probs(B, T, V, seed, dtype, sharp=(0.5, 2.0, 5.0)[seed])
        tokens = drafted(q, parents, seed)
        if seed == 1:
            tokens = tokens.to(torch.int32)
        if mode == "sampled":
            check_verify(tokens, parents, p, u, q)
        elif mode == "chosen":
            check_verify(tokens, parents, p, u)
        else:
            check_verify(tokens, parents, (p.float() + 1e-30).log().to(dtype))


def test_verify_chain_with_its_own_rows_and_shared_tree():
    """A chain of T - 1 drafts passes T - 1 draft rows; a node beyond them has no children."""
    parents = torch.tensor([-1, 0, 1, 2, 3], dtype=torch.int32, device="cuda")
    p, q, u = probs(6, 5, 777, 1, mix=0.2)
    tokens = drafted(q, parents, 2)
    a = check_verify(tokens, parents, p, u, q[:, :4].contiguous())
    b = check_verify(tokens, parents, p, u, q)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    check_verify(tokens, parents, p, u, q[:, :2].contiguous())


def test_verify_strides():
    parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
    p, q, u = probs(3, 4, 2048, 3)
    tokens = drafted(q, parents, 4)
    want = check_verify(tokens, parents, p, u, q)
    wide = torch.zeros(3, 4, 2049 + 6, device="cuda")
    for off in (0, 1, 4):
        wide[..., off:off + 2048] = p
        got = check_verify(tokens, parents, wide[..., off:off + 2048], u, q)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    got = check_verify(tokens.t().contiguous().t(), parents, p.transpose(1, 2).contiguous().transpose(1, 2), u.t().contiguous().t(), q.transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("V", [16, 4000])
def test_verify_borders(V):
    """u at 0 and just below 1, drafts equal to the target, one-point rows, repeated siblings."""
    parents = torch.tensor([-1, 0, 0, 0, 1, 1], dtype=torch.int32, device="cuda")
    p, q, u = probs(4, 6, V, 5)
    tokens = drafted(q, parents, 6)
    for x in (0.0, 1 - 2.0 ** -24, 0.5):
        check_verify(tokens, parents, p, torch.full_like(u, x), q)
        check_verify(tokens, parents, p, torch.full_like(u, x))
        check_verify(tokens, parents, p, torch.full_like(u, x), p)          # draft == target: all kept
    got = check_verify(tokens, parents, p, u, p)
    assert got.n.tolist() == [3] * 4
    same = tokens.clone()
    same[:, 2:4] = same[:, 1:2]                                             # the same token three times
    for x in (u, torch.full_like(u, 1 - 2.0 ** -24)):
        check_verify(same, parents, p, x)
        check_verify(same, parents, p, x, q)
    point = torch.zeros_like(p)
    point[..., V - 1] = 1.0
    check_verify(tokens, parents, point, u, q)
    check_verify(tokens, parents, point, u)
    check_verify(torch.full_like(tokens, V - 1), parents, point, u, point)
    # a refused draft that leaves no mass: the whole row is drawn from
    none = torch.zeros_like(p)
    none[..., 0] = 0.25
    check_verify(torch.zeros_like(tokens), parents, none, torch.full_like(u, 0.9), point.flip(-1))
    check_verify(torch.zeros_like(tokens), parents, none, torch.full_like(u, 0.9))


def test_verify_bad_rows_and_tokens(cuda):
    from kernels import _lib
    from kernels.draft_tree import verify_drafts

    parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
    p, q, u = probs(3, 4, 3000, 7)
    tokens = drafted(q, parents, 8)
    p[0] = 0.0
    p[1] = float("nan")
    p[1, :, 5] = 0.3                                # NaN is nothing: one token is left
    p[2, :, 7] = float("inf")
    tokens[1] = 9
    got = verify_drafts(tokens, parents, p, u)
    assert _lib.device_status() == _lib.CIE_DEV_BAD_PROBS
    want = verify_ref(tokens, parents, p, u)
    assert [g.tolist() for g in got] == list(want)
    assert got.tokens[0, 0].item() == -1 and got.tokens[1, 0].item() == 5
    p, q, u = probs(2, 4, 3000, 9)
    for bad in (-1, 3000, 2 ** 40):
        t = drafted(q, parents, 10)
        t[0, 1], t[0, 2], t[1, 0] = bad, bad, bad   # the root's own token is not looked at
        for kw in (dict(uniforms=u, draft_probs=q), dict(uniforms=u), dict()):
            got = verify_drafts(t, parents, p, **kw)
            assert _lib.device_status() == _lib.CIE_DEV_BAD_TREE
            assert [g.tolist() for g in got] == list(verify_ref(t, parents, p, kw.get("uniforms"), kw.get("draft_probs")))
            assert got.n[0].item() == 1


def test_verify_padded_trees():
    """Nodes without a parent fill a batch's smaller trees; their tokens may be anything."""
    parents = torch.tensor([[-1, 0, 0, 1], [-1, 0, -1, -1], [-1, -1, -1, -1]], dtype=torch.int32, device="cuda")
    p, q, u = probs(3, 4, 900, 16)
    tokens = drafted(q, parents, 17)
    tokens[1, 2:], tokens[2] = -1, -1
    for kw in (dict(uniforms=u, draft=q), dict(uniforms=u), dict()):
        got = check_verify(tokens, parents, p, **kw)
        assert got.n[2].item() == 1 and got.n[1].item() <= 2


def test_verify_greedy_ties_and_nan():
    parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
    for V in (9, 5000):
        x = torch.zeros(4, 4, V, device="cuda")
        x[0] = -float("inf")                       # all equal: the lowest index
        x[1, :, V - 1] = x[1, :, V - 3] = 2.0
        x[2, :, 4], x[2, :, 6] = float("nan"), 9.0  # NaN counts as the largest, as in torch.argmax
        x[3, :, 3], x[3, :, 1] = -0.0, 0.0
        tokens = torch.tensor([[0, 1, 0, 5], [0, V - 1, V - 3, 1], [0, 6, 4, 0], [0, 0, 0, 0]], device="cuda")
        check_verify(tokens, parents, x)
        check_verify(tokens, parents, x.to(BF16))


def test_verify_keeps_the_target_distribution():
    """The first new token is distributed as the target's row, whatever the draft was."""
    from kernels.draft_tree import verify_drafts

    B, V = 200_000, 7
    gen = torch.Generator(device="cuda").manual_seed(11)
    p = torch.softmax(torch.randn(1, 4, V, generator=gen, device="cuda"), -1).expand(B, 4, V).contiguous()
    q = torch.softmax(torch.randn(1, 4, V, generator=gen, device="cuda"), -1).expand(B, 4, V).contiguous()
    u = torch.rand(B, 4, generator=gen, device="cuda")
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    drawn = torch.multinomial(q[0, 0], 3 * B, replacement=True, generator=gen).view(B, 3)
    tokens = torch.cat([torch.zeros_like(drawn[:, :1]), drawn], 1)
    first = verify_drafts(tokens, parents, p, u, q).tokens[:, 0]
    got = torch.bincount(first, minlength=V).double() / B
    row = p[0, 0].double()
    sigma = (row * (1 - row) / B).sqrt()           # six of them: one in 5e8 by chance
    assert float(((got - row).abs() - 6 * sigma).max()) <= 0


def test_verify_graph():
    from kernels.draft_tree import verify_drafts

    parents = torch.tensor([-1, 0, 0, 1, 1, 2], dtype=torch.int32, device="cuda")
    p, q, u = probs(5, 6, 40000, 12)
    tokens = drafted(q, parents, 13)
    verify_drafts(tokens, parents, p, u, q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = verify_drafts(tokens, parents, p, u, q)
    for seed in (14, 15):
        p2, q2, u2 = probs(5, 6, 40000, seed)
        for a, b in ((p, p2), (q, q2), (u, u2), (tokens, drafted(q2, parents, seed))):
            a.copy_(b)
        g.replay()
        assert [x.tolist() for x in got] == list(verify_ref(tokens, parents, p, u, q))


# ------------------------------------------------------------------ kept path
def keep_ref(pools, tables, lens, path, n, T, bs):
    out = [p.clone() for p in pools]
    new = []
    for b in range(len(lens)):
        base = int(lens[b]) - T
        new.append(max(0, base + int(n[b])))
        for i in range(1, int(n[b])):
            s, d = base + int(path[b][i]), base + i
            for o, p in zip(out, pools):
                o[int(tables[b, d // bs]), d % bs] = p[int(tables[b, s // bs]), s % bs]
    return out, new


@pytest.mark.parametrize("B,T,Hkv,D,bs,dtype,n_pools", [(1, 1, 1, 16, 16, BF16, 2), (3, 8, 8, 64, 16, BF16, 4), (2, 33, 3, 128, 24, FP16, 6), (4, 64, 2, 32, 5, BF16, 3),
                                                        (1, 1024, 1, 16, 16, FP16, 1), (2, 6, 8, 128, 16, BF16, 300), (40, 16, 8, 128, 16, BF16, 40)])
def test_keep_path(B, T, Hkv, D, bs, dtype, n_pools):
    from kernels.draft_tree import keep_path

    rs = np.random.RandomState(T)
    s = setup(B, T, Hkv, Hkv, D, bs, dtype, [T + int(rs.randint(0, 60)) for _ in range(B)], seed=T)
    gen = torch.Generator(device="cuda").manual_seed(1)
    pools = [torch.randn(s["k"].shape, generator=gen, device="cuda").to(dtype) for _ in range(n_pools)]
    n = [int(rs.randint(1, T + 1)) if b else T for b in range(B)]
    path = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        pick = np.sort(rs.permutation(T - 1)[:n[b] - 1]) + 1 if b else np.arange(1, T)  # b = 0: all kept, nothing moves
        path[b, :n[b]] = torch.from_numpy(np.concatenate([[0], pick]).astype(np.int32))
    if B > 1 and T > 2:                                     # a shift by one: every source is a destination too
        n[1] = T - 1
        path[1, :T - 1] = torch.tensor([0] + list(range(2, T)), dtype=torch.int32)
    want, lens = keep_ref(pools, s["tables"].cpu(), s["lens"].tolist(), path, n, T, bs)
    got = keep_path(pools, s["tables"], s["lens"], path.cuda(), torch.tensor(n, dtype=torch.int32, device="cuda"))
    assert got.tolist() == lens
    for a, w in zip(pools, want):
        assert torch.equal(a, w)


def test_keep_path_idle_and_bad_entries(cuda):
    from kernels import _lib
    from kernels.draft_tree import keep_path

    s = setup(3, 5, 2, 2, 64, 16, BF16, [0, 40, 20], seed=20)
    pools = [torch.randn(s["k"].shape, device="cuda").to(BF16)]
    path = torch.tensor([[0, -1, -1, -1, -1], [0, 2, 1, 9, 4], [0, 3, 4, -1, -1]], dtype=torch.int32, device="cuda")
    n = torch.tensor([1, 5, 3], dtype=torch.int32, device="cuda")
    before = pools[0].clone()
    got = keep_path(pools, s["tables"], s["lens"], path, n)
    assert _lib.device_status() == _lib.CIE_DEV_BAD_TREE
    assert got.tolist() == [0, 40, 18]
    good = torch.tensor([[0, -1, -1, -1, -1], [0, 2, 2, 3, 4], [0, 3, 4, -1, -1]], dtype=torch.int32)
    want, _ = keep_ref([before], s["tables"].cpu(), [5, 40, 20], good, [1, 5, 3], 5, 16)
    assert torch.equal(pools[0], want[0])
    keep_path(pools, s["tables"], s["lens"], path, torch.tensor([1, -4, 6], dtype=torch.int32, device="cuda"))
    assert _lib.device_status() == _lib.CIE_DEV_BAD_TREE
    tables = s["tables"].clone()
    tables[1, 2] = 1 << 20
    now = pools[0].clone()
    keep_path(pools, tables, s["lens"], good.cuda(), torch.tensor([1, 2, 1], dtype=torch.int32, device="cuda"))
    assert _lib.device_status() == _lib.CIE_DEV_BAD_BLOCK_ID
    assert torch.equal(now, pools[0])


# ------------------------------------------------------------------ together
def _model(layers, hq, hkv, d, vocab, seed):
    """A small attention-only model in 64 bits and its weights in bf16."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dim = hq * d
    r = lambda *s: (torch.randn(*s, generator=gen, device="cuda") * s[0] ** -0.5).to(BF16)  # noqa: E731
    return dict(embed=(torch.randn(vocab, dim, generator=gen, device="cuda")).to(BF16), head=r(dim, vocab),
                layers=[dict(q=r(dim, hq * d), k=r(dim, hkv * d), v=r(dim, hkv * d), o=r(dim, dim)) for _ in range(layers)])


def _forward(m, cache, step, tokens, hq, hkv, d, rope):
    from engine.attention import attention_forward_batch

    B, T = tokens.shape
    x = m["embed"][tokens]
    for i, w in enumerate(m["layers"]):
        heads = lambda n, h: (x @ w[n]).view(B, T, h, d).transpose(1, 2)  # noqa: E731,B023
        a = attention_forward_batch(heads("q", hq), heads("k", hkv), heads("v", hkv), cache, i, step, rope=rope)
        x = x + a.transpose(1, 2).reshape(B, T, hq * d) @ w["o"]
    return x.float() @ m["head"].float()


@pytest.mark.parametrize("hq,hkv,d,bs", [(8, 2, 64, 16), (4, 4, 32, 8)])
def test_tree_steps_decode_like_chains(hq, hkv, d, bs):
    """Greedy decoding by trees of drafts, one of whose paths is right: the cache after every
    step holds the rows that plain decoding of the same tokens appends, and the tokens are its tokens."""
    from engine.attention import attention_forward_batch, begin_step, end_tree_step
    from engine.cache import KVCacheConfig, PagedKVCache
    from kernels.draft_tree import verify_drafts

    layers, vocab, B = 3, 97, 3
    m = _model(layers, hq, hkv, d, vocab, 1)
    rope = rope_tables(d)
    mk = lambda: PagedKVCache(KVCacheConfig(num_layers=layers, num_kv_heads=hkv, head_dim=d, num_blocks=80, block_size=bs))  # noqa: E731
    plain, treed = mk(), mk()
    pt, tt = [plain.new_sequence() for _ in range(B)], [treed.new_sequence() for _ in range(B)]
    rs = np.random.RandomState(3)
    prompt = torch.from_numpy(rs.randint(0, vocab, (B, 9))).cuda()
    first = []
    for cache, tables in ((plain, pt), (treed, tt)):
        first.append(_forward(m, cache, begin_step(cache, tables, 9), prompt, hq, hkv, d, rope)[:, -1].argmax(-1))
    assert torch.equal(*first)
    # plain greedy decoding
    want, last = [[] for _ in range(B)], first[0]
    for _ in range(14):
        for b in range(B):
            want[b].append(int(last[b]))
        last = _forward(m, plain, begin_step(plain, pt, 1), last[:, None], hq, hkv, d, rope)[:, -1].argmax(-1)
    for b in range(B):
        want[b].append(int(last[b]))
    got, sizes = [[int(first[0][b])] for b in range(B)], []
    parents = [[-1, 0, 0, 1, 2, 2, 4, 6], [-1, 0, 1, 2, 3, 4, 5, 6], [-1, 0, 0, 0, 3, 4, 4, -1]]
    good = [[2, 5], [1, 2, 3, 4], [3, 4, 6]]  # nodes that draft what plain decoding finds next
    while min(len(g) for g in got) < 8:
        tokens = torch.from_numpy(rs.randint(0, vocab, (B, 8))).cuda()
        for b in range(B):
            tokens[b, 0] = got[b][-1]
            for k, node in enumerate(good[b]):
                tokens[b, node] = want[b][len(got[b]) + k]
        step = begin_step(treed, tt, 8, parents=parents)
        logits = _forward(m, treed, step, tokens, hq, hkv, d, rope)
        verdict = verify_drafts(tokens, step.parents, logits)
        new = end_tree_step(treed, step, verdict)
        for b in range(B):
            assert len(new[b]) >= len(good[b]) + 1 or new[b] == want[b][len(got[b]):len(got[b]) + len(new[b])]
            got[b] += new[b]
        sizes.append([len(n) for n in new])
        assert [t.length for t in tt] == [9 + len(g) - 1 for g in got]
    for b in range(B):
        n = min(len(got[b]), len(want[b]))
        assert got[b][:n] == want[b][:n], (sizes, got[b], want[b])
        rows = 9 + min(len(got[b]), len(want[b])) - 1
        for layer in range(layers):
            for x, y in zip(plain.gather(layer, pt[b]), treed.gather(layer, tt[b])):
                # the first layer's rows do not depend on attention: the same bits
                if layer == 0:
                    assert torch.equal(x[:rows], y[:rows])
                else:
                    assert float((x[:rows].float() - y[:rows].float()).abs().max()) < 0.1


def test_tree_step_has_no_host_sync_before_its_end():
    from engine.attention import attention_forward_batch, begin_step
    from engine.cache import KVCacheConfig, PagedKVCache
    from kernels.draft_tree import verify_drafts

    cache = PagedKVCache(KVCacheConfig(num_layers=2, num_kv_heads=2, head_dim=64, num_blocks=64, block_size=16))
    tables = [cache.new_sequence() for _ in range(2)]
    rope = rope_tables(64)
    rnd = lambda h, n: torch.randn(2, h, n, 64, device="cuda", dtype=BF16)  # noqa: E731
    p, q, u = probs(2, 6, 512, 1)
    parents = torch.tensor([-1, 0, 0, 1, 1, 2], dtype=torch.int32, device="cuda")
    tokens = drafted(q, parents, 2)

    def step_once():
        s = begin_step(cache, tables, 6, parents=parents)
        for layer in range(2):
            attention_forward_batch(rnd(8, 6), rnd(2, 6), rnd(2, 6), cache, layer, s, rope=rope)
        v = verify_drafts(tokens, parents, p, u, q)
        return s, cache.keep_path(s.block_tables, s.kv_lens, v.path, v.n), v

    step_once()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        s, lens, v = step_once()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert lens.tolist() == [6 + n for n in v.n.tolist()]


def test_two_streams_at_once():
    """Calls that overlap on two streams share nothing: each gives what it gives alone."""
    from kernels.draft_tree import keep_path, tree_attention, verify_drafts

    sets = []
    for i, (D, T) in enumerate(((128, 20), (64, 9))):
        s = setup(6, T, 16, 4, D, 16, BF16, [T + 300 * b for b in range(6)], seed=30 + i)
        p, q, u = probs(6, T, 20000 + i, 31 + i)
        tokens = drafted(q, s["parents"], 32 + i)
        pool = torch.randn(s["k"].shape, device="cuda").to(BF16)
        sets.append((s, (tokens, s["parents"], p, u, q), pool))

    def one(x):
        s, v, pool = x
        out = tree_attention(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"])
        verdict = verify_drafts(*v)
        moved = pool.clone()
        lens = keep_path([moved], s["tables"], s["lens"], verdict.path, verdict.n)
        return [out, *verdict, moved, lens]

    want = [one(x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, x in enumerate(sets):
            with torch.cuda.stream(streams[k]):
                got[k].append(one(x))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))
