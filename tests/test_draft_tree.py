"""CPU checks of the tree-of-drafts operators: what they refuse, before any kernel runs."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import build_ext

    build_ext.build()
    from kernels import _lib

    return _lib.load()


P = ctypes.c_void_p(4096)
S3 = (ctypes.c_int64 * 3)(64, 64, 64)
S2 = (ctypes.c_int64 * 2)(64, 64)


def refused(rc, text, code=None):
    from kernels import _lib

    assert rc == (_lib.CIE_ERR_INVALID if code is None else code)
    assert text in _lib.last_error()


def tree_args(**kw):
    a = dict(q=P, k=P, v=P, tab=P, lens=P, par=P, psb=0, o=P, B=1, Hq=4, Hkv=2, T=5, d=64, nb=8, bs=16, mb=4, qs=S3, os=S3, scale=1.0,
             dt=0, cos=None, sin=None, mp=0, split=0, ws=None, wsb=0, st=None)
    a.update(kw)
    return list(a.values())


def test_tree_attention_refuses(lib):
    from kernels import _lib

    f = lib.cie_tree_attn
    refused(f(*tree_args(q=None)), "null")
    refused(f(*tree_args(par=None)), "null")
    refused(f(*tree_args(Hq=5)), "multiple")
    refused(f(*tree_args(T=1025)), "at most 1024")
    refused(f(*tree_args(T=-1)), "bad shape")
    refused(f(*tree_args(dt=2)), "dtype")
    refused(f(*tree_args(bs=0)), "pool geometry")
    refused(f(*tree_args(mb=1 << 28)), "too large")
    refused(f(*tree_args(qs=(ctypes.c_int64 * 3)(64, 64, 60))), "multiples of 8")
    refused(f(*tree_args(k=ctypes.c_void_p(4104))), "aligned")
    refused(f(*tree_args(split=24)), "multiple of 16")
    for scale in (0.0, -0.5, float("nan"), float("inf")):
        refused(f(*tree_args(scale=scale)), "positive")
    refused(f(*tree_args(cos=P)), "both")
    refused(f(*tree_args(cos=P, sin=P)), "rope_max_pos")
    refused(f(*tree_args(psb=-1)), "stride")
    refused(f(*tree_args(d=96)), "unsupported", _lib.CIE_ERR_UNSUPPORTED)
    refused(f(*tree_args(mb=4096)), "workspace", _lib.CIE_ERR_WORKSPACE)
    assert f(*tree_args(B=0)) == 0 and f(*tree_args(T=0)) == 0
    assert lib.cie_tree_attn_workspace(1, 4, 2, 5, 64, 16, 4096, 0) > 0
    assert lib.cie_tree_attn_workspace(1, 4, 2, 5, 64, 16, 4, 0) == 0
    assert lib.cie_tree_attn_workspace(1, 4, 3, 5, 64, 16, 4, 0) == 0
    assert lib.cie_tree_attn_workspace(1, 4, 2, 5, 64, 16, 1 << 28, 0) == 0


def test_rope_append_tree_refuses(lib):
    f = lib.cie_rope_append_tree
    base = [P, P, P, P, P, P, P, 0, 1, 4, 2, 64, 8, 16, 4, S3, 0, None, None, 0, None]
    bad = lambda i, x: base[:i] + [x] + base[i + 1:]  # noqa: E731
    refused(f(*bad(6, None)), "null")
    refused(f(*bad(7, -1)), "stride")
    refused(f(*bad(9, 1025)), "at most 1024")
    refused(f(*bad(11, 24)), "head_dim")
    assert f(*bad(9, 0)) == 0


def test_verify_refuses(lib):
    f = lib.cie_verify_drafts
    base = dict(tok=P, tsb=5, t64=0, par=P, psb=0, p=P, ps=S2, q=None, qs=None, qr=0, u=P, usb=5, B=1, T=5, V=64, dt=2, out=P, path=P, n=P, st=None)
    go = lambda **kw: f(*{**base, **kw}.values())  # noqa: E731
    refused(go(tok=None), "null")
    refused(go(n=None), "null")
    refused(go(T=0), "bad shape")
    refused(go(V=0), "bad shape")
    refused(go(T=1025), "at most 1024")
    refused(go(V=(1 << 23) + 1), "at most")
    refused(go(dt=3), "dtype")
    refused(go(q=P, qs=S2, qr=0), "draft_rows")
    refused(go(q=P, qs=S2, qr=6), "draft_rows")
    refused(go(q=P, qs=S2, qr=4, u=None), "uniforms")
    refused(go(tsb=-1), "stride")
    assert go(B=0) == 0


def test_keep_path_refuses(lib):
    f = lib.cie_keep_path
    pools = (ctypes.c_void_p * 2)(4096, 8192)
    base = dict(pools=pools, k=2, tab=P, lens=P, path=P, n=P, new=P, B=1, T=5, nb=8, bs=16, mb=4, row=256, st=None)
    go = lambda **kw: f(*{**base, **kw}.values())  # noqa: E731
    refused(go(path=None), "null")
    refused(go(T=0), "bad shape")
    refused(go(T=1025), "at most 1024")
    refused(go(nb=0), "pool geometry")
    refused(go(nb=1 << 28), "too large")
    refused(go(row=24), "row_bytes")
    refused(go(row=0), "row_bytes")
    refused(go(pools=(ctypes.c_void_p * 2)(4096, 8200)), "pool 1")
    refused(go(B=65536), "65535")
    assert go(B=0) == 0


def test_entries_ask_for_cuda_tensors():
    from kernels.draft_tree import keep_path, tree_attention, verify_drafts

    q, pool = torch.zeros(1, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        tree_attention(q, pool, pool, i32([0, 1]).view(1, 2), i32(20), i32(-1, 0, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_drafts(torch.zeros(1, 3, dtype=torch.int64), i32(-1, 0, 1), torch.zeros(1, 3, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        keep_path([pool, pool], i32([0, 1]).view(1, 2), i32(20), i32([0, 1, -1]).view(1, 3), i32(2))


def test_reference_restatement():
    """The 64-bit restatement that the GPU tests use, on cases worked out by hand."""
    from tests.tree_ref import ancestors, depths, verify_ref

    par = [-1, 0, 0, 1, 3, -1]
    assert depths(par) == [0, 1, 1, 2, 3, 0]
    assert ancestors(par)[4].tolist() == [True, True, False, True, True, False]
    p = torch.tensor([[[0.5, 0.3, 0.2]] * 3])
    q = torch.tensor([[[0.1, 0.6, 0.3]] * 3])
    tok, tree = torch.tensor([[0, 1, 2]]), torch.tensor([-1, 0, 0])
    # node 1 drafts 1: 0.4 * 0.6 < 0.3, kept; its row then gives the last token at u0 = 0.79: 1
    assert verify_ref(tok, tree, p, torch.tensor([[0.79, 0.4, 0.0]]), q) == ([[1, 1, -1]], [[0, 1, -1]], [2])
    # refused at u = 0.6: r = [.4, 0, 0], m = 0.4; node 2 drafts 2 with r = 0: refused; token 0
    assert verify_ref(tok, tree, p, torch.tensor([[0.9, 0.6, 0.5]]), q) == ([[0, -1, -1]], [[0, -1, -1]], [1])
    # chosen drafts: 0.6 < 0.3 no; then 0.2 < m = 0.7 times u = 0.2: kept
    assert verify_ref(tok, tree, p, torch.tensor([[0.0, 0.6, 0.2]])) == ([[2, 0, -1]], [[0, 2, -1]], [2])
    assert verify_ref(torch.tensor([[9, 0, 0]]), torch.tensor([-1, 0, 1]), p) == ([[0, 0, 0]], [[0, 1, 2]], [3])


def test_step_checks_trees():
    from engine.attention import _tree_parents, end_tree_step, BatchStep

    assert _tree_parents([-1, 0, 1], 2, 3).tolist() == [-1, 0, 1]
    assert _tree_parents([[-1, 0, 1], [-1, 0, -1]], 2, 3).dtype == torch.int32
    for bad, text in (([-1, 0], "parents must be"), ([-1, 1, 0], "earlier"), ([-1, 0, -2], "earlier"), ([0, 0, 0], "earlier"),
                      ([[-1, 0, 1]] * 3, "parents must be")):
        with pytest.raises(ValueError, match=text):
            _tree_parents(bad, 2, 3)
    step = BatchStep([], 1, [], None, None, None)
    with pytest.raises(ValueError, match="parents"):
        end_tree_step(None, step, None)
