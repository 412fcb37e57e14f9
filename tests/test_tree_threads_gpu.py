"""Tree operators called by two host threads at once: the library's calls are thread-safe."""

from __future__ import annotations

import threading

import pytest
import torch

from tests.test_draft_tree_gpu import _clean_status, run, setup  # noqa: F401

pytestmark = pytest.mark.gpu


def both(fns, calls):
    """Each of ``fns`` ``calls`` times in a thread of its own with a stream of its own; the last results."""
    last, errors, start = [None] * len(fns), [], threading.Barrier(len(fns))

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(calls):
                    last[i] = fns[i]()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001  shown by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(fns))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    return last


@pytest.mark.parametrize("D,small,large", [(32, 40, 1024), (256, 1, 900), (64, 257, 1024)])
def test_trees_of_two_sizes(D, small, large):
    """Both run on one kernel, whose shared memory grows with the tree. The C entry is called in a tight
    loop, where the calls of the two threads interleave most."""
    from kernels import _lib

    lib = _lib.load()
    fns, outs, want, keep = [], [], [], []
    for T in (small, large):
        s = setup(1, T, 1, 1, D, 16, torch.bfloat16, [T + 3], "star", seed=90 + T)
        want.append(run(s))
        out = torch.empty_like(s["q"])
        strides, par = _lib.strides3(out.stride()[:3]), s["parents"]
        ws = torch.empty(max(1, lib.cie_tree_attn_workspace(1, 1, 1, T, D, 16, s["tables"].shape[1], 0)), dtype=torch.uint8, device="cuda")
        args = (s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["tables"].data_ptr(), s["lens"].data_ptr(), par.data_ptr(), 0,
                out.data_ptr(), 1, 1, 1, T, D, s["k"].shape[0], 16, s["tables"].shape[1], strides, strides, D ** -0.5, _lib.CIE_DTYPE_BF16,
                None, None, 0, 0, ws.data_ptr(), ws.numel())

        def call(args=args, what=f"{T} nodes"):
            stream = torch.cuda.current_stream().cuda_stream
            for _ in range(200):
                _lib.check(lib.cie_tree_attn(*args, stream), what)

        fns.append(call)
        outs.append(out)
        keep.append((s, ws))
    torch.cuda.synchronize()
    both(fns, 50)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_verify_of_two_sizes():
    """Long rows and many nodes: more shared memory than a kernel has without asking."""
    from kernels.draft_tree import verify_drafts

    V = 1 << 22
    p = torch.rand(V, generator=torch.Generator(device="cuda").manual_seed(92), device="cuda")
    p /= p.sum()
    calls = []
    for T in (1000, 1024):
        gen = torch.Generator(device="cuda").manual_seed(T)
        tokens = torch.randint(0, V, (1, T), generator=gen, device="cuda")
        u = torch.rand(1, T, generator=gen, device="cuda")
        parents = torch.tensor([-1] + [(i - 1) // 2 for i in range(1, T)], dtype=torch.int32, device="cuda")
        calls.append(lambda tokens=tokens, parents=parents, u=u, T=T: verify_drafts(tokens, parents, p.expand(1, T, V), u))
    want = [f() for f in calls]
    torch.cuda.synchronize()
    got = both(calls, 1500)
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))
