"""NaN and infinity in drafted rows: every entry of the output, those of the rows that see them too."""

from __future__ import annotations

import pytest
import torch

from tests.test_draft_tree_gpu import _clean_status, run, setup  # noqa: F401
from tests.tree_ref import assert_within, half_step, tree_attention_ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def row(s, b, node, T):
    """Pool index (block, offset) of a node's slot."""
    t = int(s["lens"][b]) - T + node
    bs = s["k"].shape[1]
    return int(s["tables"][b, t // bs]), t % bs


@pytest.mark.parametrize("split", [0, 64])
@pytest.mark.parametrize("D,T,Hq,hist,bs,dtype", [
    (64, 9, 8, (3, 333), 16, BF16), (64, 9, 8, (3, 333), 16, FP16), (64, 70, 8, (0, 40), 16, FP16), (64, 20, 8, (5, 61), 20, BF16),
    (128, 9, 8, (3, 120), 16, BF16), (128, 50, 16, (2, 300), 16, FP16), (128, 13, 4, (1, 200), 24, FP16),
    (32, 9, 8, (3, 333), 16, FP16), (32, 20, 4, (2, 40), 12, FP16), (32, 40, 8, (7, 100), 16, BF16), (16, 9, 4, (3, 33), 16, FP16),
    (256, 5, 4, (3, 133), 16, FP16), (256, 12, 8, (2, 50), 16, BF16), (256, 9, 4, (4, 70), 20, FP16),
    (64, 260, 4, (3, 30), 16, FP16),
])
def test_bad_columns_of_drafted_rows(D, T, Hq, hist, bs, dtype, split):
    """A few columns of some nodes' V hold NaN or infinities. Finite entries of all rows stay within the
    bound, infinite ones have the sign and NaN the places of the 64-bit restatement (whose weights
    are all far above underflow here: scores differ by less than 20). P has at least 2^-15 on every
    path, so for bf16 the bound's term for a P rounded once, 2^-8 A, shrinks to 2^-15 A."""
    s = setup(2, T, Hq, 2, D, bs, dtype, [T + h for h in hist], "random", seed=60 + D + T)
    for b in range(2):
        for node, col, x in ((T - 1, 0, NAN), (T // 2, 3, INF), (T // 3, 5, -INF), (1, D - 1, INF), (2, D - 1, -INF), (T - 2, 7, -INF)):
            at = row(s, b, node, T)
            s["v"][at[0], at[1], :, col] = x
            s["v"][at[0], at[1], 0, 9] = x            # of one kv head only
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"])
    assert bool(torch.isnan(ref).any()) and bool((ref == INF).any()) and bool((ref == -INF).any())
    if dtype == BF16:
        a, _ = tree_attention_ref(s["q"], s["k"], s["v"].abs(), s["tables"], s["lens"], s["parents"])
        bound = bound - a * (half_step(BF16) - 2.0 ** -15)
    assert_within(run(s, split_tokens=split), ref, bound)


@pytest.mark.parametrize("D,T,dtype", [(64, 9, BF16), (128, 40, FP16), (32, 9, FP16), (256, 5, BF16)])
def test_small_weights_of_infinite_values(D, T, dtype):
    """An infinity that a row gives a weight of about 2^-30 (less than fp16's smallest number) is still one."""
    s = setup(1, T, 4, 2, D, 16, dtype, [T + 50], "chain", seed=70 + D)
    q = torch.zeros_like(s["q"])
    q[..., 0] = 8.0
    s["q"] = q
    s["k"].nan_to_num_(0)
    s["k"][..., 0] = 0.0
    at = row(s, 0, 1, T)
    s["k"][at[0], at[1], :, 0] = -2.625                # score -21: 2^-30 of the others'
    s["v"][at[0], at[1], :, 2] = INF
    s["v"][at[0], at[1], :, 4] = -INF
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"], 1.0)
    assert int((ref == INF).sum()) == 4 * (T - 1) == int((ref == -INF).sum())
    assert_within(run(s, scale=1.0), ref, bound)


@pytest.mark.parametrize("D,T,dtype", [(64, 9, FP16), (128, 40, BF16), (32, 9, BF16), (256, 5, FP16)])
def test_bad_keys_of_drafted_rows(D, T, dtype):
    """A NaN in a node's K makes the rows that see it NaN, and no other entry of the output anything but what it was."""
    s = setup(2, T, 4, 2, D, 16, dtype, [T + 20, T + 200], "random", seed=80 + D)
    for b in range(2):
        at = row(s, b, T // 2, T)
        s["k"][at[0], at[1], 1, 1] = NAN
    ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"])
    assert bool(torch.isnan(ref).any()) and not bool(torch.isnan(ref[:, :2]).any())
    assert_within(run(s), ref, bound)
