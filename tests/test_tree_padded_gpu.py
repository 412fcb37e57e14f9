"""A step over a padded batch, operators together: idle slots (length 0) take part in every call."""

from __future__ import annotations

import pytest
import torch

from tests.test_draft_tree_gpu import _clean_status, drafted, keep_ref, probs, run, setup  # noqa: F401
from tests.tree_ref import assert_within, tree_attention_ref, verify_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("D,T", [(64, 6), (128, 9), (32, 6)])
def test_idle_slots_take_part_in_a_step(D, T, shared):
    """Whatever the verdict on an idle slot (its rows are somebody's leftovers), nothing of it moves,
    its length stays 0 and no status bit is raised."""
    from kernels.draft_tree import keep_path, verify_drafts

    lens = [0, T + 40, 0, 0, T, T + 333]
    s = setup(6, T, 4, 2, D, 16, torch.bfloat16, lens, "chain" if shared else "random", seed=120 + D)
    if shared:
        s["parents"] = s["parents"][0].clone()
    out = run(s)
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"])
    assert_within(out, ref, bound)
    p, q, u = probs(6, T, 700, 121, mix=0.05)                     # drafts that are mostly kept
    tokens = drafted(q, s["parents"], 122)
    got = verify_drafts(tokens, s["parents"], p, u, q)
    assert [x.tolist() for x in got] == list(verify_ref(tokens, s["parents"], p, u, q))
    assert max(got.n.tolist()[b] for b in (0, 2, 3)) > 1          # an idle slot with a path to keep
    pools = [torch.randn(s["k"].shape, device="cuda").to(torch.bfloat16) for _ in range(4)]
    n = [1 if lens[b] == 0 else int(got.n[b]) for b in range(6)]
    want, _ = keep_ref(pools, s["tables"].cpu(), [max(x, T) for x in lens], got.path.cpu(), n, T, 16)
    new = keep_path(pools, s["tables"], s["lens"], got.path, got.n)
    assert new.tolist() == [0 if lens[b] == 0 else lens[b] - T + n[b] for b in range(6)]
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
