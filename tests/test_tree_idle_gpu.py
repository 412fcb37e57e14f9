"""Padded batches: a few sequences at work among many idle ones."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_draft_tree_gpu import _clean_status, run, setup  # noqa: F401
from tests.tree_ref import assert_within, tree_attention_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,at,longest", [
    (400, [0, 1, 33, 34, 66, 399], 900),       # gaps of 31, 32 and hundreds; sequences cut among CTAs
    (400, [63, 64, 65, 200, 232, 265], 300),   # sequences left whole, dealt out in steps
    (2000, [1999], 2500),
    (2000, [0], 130),
    (500, [], 1),                              # nobody at work
])
@pytest.mark.parametrize("D,T", [(128, 7), (64, 70)])
def test_few_at_work(B, at, longest, D, T):
    rs = np.random.RandomState(B + longest)
    lens = [0] * B
    for b in at:
        lens[b] = T + int(rs.randint(0, longest))
    s = setup(B, T, 4, 2, D, 16, torch.bfloat16, lens, seed=110)
    out = run(s)
    idle = [b for b in range(B) if lens[b] == 0]
    assert float(out[idle].abs().max()) == 0.0
    if at:
        ref, bound = tree_attention_ref(s["q"][at], s["k"], s["v"], s["tables"][at], s["lens"][at], s["parents"][at])
        assert_within(out[at], ref, bound)


def test_idle_sequences_cost_little():
    """16 sequences at work among 4096 slots take a small multiple of their own time (6 when this was
    written; the CTAs' walks through the slots one by one took it to 90)."""
    def us(B):
        lens = [0] * B
        lens[::B // 16] = [2000] * 16
        s = setup(B, 8, 32, 8, 128, 16, torch.bfloat16, lens, seed=111)
        run(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(5):
                run(s)
        best = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            g.replay()
            b.record()
            torch.cuda.synchronize()
            best.append(a.elapsed_time(b) * 200)
        return min(best)

    few, padded = us(16), us(4096)
    assert padded < 20 * few, f"{padded:.0f} us against {few:.0f}"
