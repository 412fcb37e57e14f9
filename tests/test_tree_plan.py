"""How the tree attention divides its work among CTAs, read off the workspace it asks for."""

from __future__ import annotations

import pytest

from tests.test_draft_tree import lib  # noqa: F401

SLOTS = 2 * 148  # CTAs that run at once on a B200


def ctas(lib, heads, T=4, B=8, d=64):  # noqa: F811
    """Each CTA may leave two partial results of 32 rows: d fp32 values and a log-sum-exp each."""
    n = lib.cie_tree_attn_workspace(B, heads, heads, T, d, 16, 512, 0) - 256
    assert n % (2 * 32 * (d + 1) * 4) == 0
    return n // (2 * 32 * (d + 1) * 4)


@pytest.mark.parametrize("heads", [1, 2, 4, 8, 16, 32, 40, 48, 64, 80, 96, 100, 128, 160, 200, 296, 300, 320, 400, 500])
def test_rounds_of_ctas(lib, heads):  # noqa: F811
    """One round where it fills nine tenths of the slots; else the number of rounds, up to four, after
    which a slot has had the smallest share of a head's list of tiles."""
    n = ctas(lib, heads)
    assert n % heads == 0
    parts = n // heads
    one = SLOTS // heads * heads
    if one and (SLOTS - one) * 10 <= SLOTS:
        # 8 sequences of up to 128 tiles, 8 more each for their borders, at least 4 tiles a CTA
        assert n == min(one, heads * (8 * (128 + 8) // 4))
        return
    share = -(-n // SLOTS) / parts
    best = min(r / (r * SLOTS // heads) for r in range(1, 5) if r * SLOTS >= heads)
    assert share == pytest.approx(best), (n, parts)
