"""How many bits of P the tree attention keeps: the output's own rounding is the only one to 16 bits."""

from __future__ import annotations

import pytest
import torch

from tests.test_draft_tree_gpu import _clean_status, run, setup  # noqa: F401
from tests.tree_ref import assert_within, half_step, tree_attention_ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("B,T,Hq,Hkv,D,bs,lens,split", [
    (2, 6, 8, 2, 64, 16, [300, 900], 0),
    (2, 16, 32, 8, 128, 16, [700, 2500], 0),
    (1, 64, 32, 8, 128, 16, [3000], 256),
    (2, 13, 16, 16, 128, 24, [100, 1500], 0),
    (2, 9, 8, 2, 64, 20, [400, 1100], 0),
    (2, 31, 4, 4, 16, 8, [90, 600], 0),
    (2, 40, 8, 4, 32, 16, [41, 1555], 0),
    (2, 12, 4, 2, 256, 16, [100, 1700], 0),
    (1, 300, 2, 2, 64, 16, [1300], 0),
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_p_is_held_in_more_than_16_bits(B, T, Hq, Hkv, D, bs, lens, split, dtype):
    """P in two halves: bf16 p = hi + lo with |lo| < 2^-7 p, exact but for lo's rounding by half a
    step, 2^-8 of it: off by 2^-15 p (fp16: hi rounded, 2^-11 2^-11 = 2^-22 p, inside the 2^-21 of the
    common bound). So of the common bound's term A h for a P rounded once, A = sum_j p_j |v_j|, 2^-15 A
    is left. The sum over hundreds of keys makes many outputs small beside A, where one rounding
    of P (about 2^-9 sqrt(sum p_j^2 v_j^2) at random) shows."""
    s = setup(B, T, Hq, Hkv, D, bs, dtype, lens, seed=40 + D)
    s["k"].nan_to_num_(0)
    s["v"].nan_to_num_(0)
    args = (s["q"], s["k"])
    ref, bound = tree_attention_ref(*args, s["v"], s["tables"], s["lens"], s["parents"])
    if dtype == BF16:
        a, _ = tree_attention_ref(*args, s["v"].abs(), s["tables"], s["lens"], s["parents"])
        bound = bound - a * (half_step(BF16) - 2.0 ** -15)
    assert_within(run(s, split_tokens=split), ref, bound)


@pytest.mark.parametrize("D,Hq,T", [(64, 8, 6), (128, 32, 16), (256, 4, 12)])
def test_scaled_rows(D, Hq, T):
    """The same with scores so far apart that most of P is tiny, and with a small scale."""
    s = setup(2, T, Hq, 2, D, 16, BF16, [400, 1200], seed=50)
    s["k"].nan_to_num_(0)
    s["v"].nan_to_num_(0)
    for scale in (1.0, 0.01):
        ref, bound = tree_attention_ref(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["parents"], scale)
        a, _ = tree_attention_ref(s["q"], s["k"], s["v"].abs(), s["tables"], s["lens"], s["parents"], scale)
        assert_within(run(s, scale=scale), ref, bound - a * (half_step(BF16) - 2.0 ** -15))
