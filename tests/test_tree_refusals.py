"""CPU checks of calls of the tree operators that would go wrong and are refused."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests.test_draft_tree import P, lib, refused  # noqa: F401


def pools(*at):
    return (ctypes.c_void_p * len(at))(*at)


@pytest.mark.parametrize("at,which", [
    ((1 << 20, 2 << 20, 1 << 20), 2),                          # a pool twice
    ((1 << 20, (1 << 20) + 4096), 1),                          # one that begins inside another
    (tuple((i + 1) << 20 for i in range(300)) + (7 << 20,), 300),  # across two launches
])
def test_keep_path_refuses_pools_that_share_memory(lib, at, which):  # noqa: F811
    # 8 blocks of 16 rows of 256 bytes: 32 KB a pool
    rc = lib.cie_keep_path(pools(*at), len(at), P, P, P, P, P, 1, 5, 8, 16, 4, 256, None)
    refused(rc, f"pool {which} shares memory")


@pytest.mark.gpu
def test_keep_path_takes_pools_side_by_side(cuda):
    """Pools that lie next to each other in one tensor share nothing."""
    from kernels.draft_tree import keep_path

    both = torch.arange(2 * 4 * 16 * 2 * 16, device="cuda").view(2, 4, 16, 2, 16).remainder(251).to(torch.bfloat16)
    want = both.clone()
    want[:, 0, 6] = both[:, 0, 8]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens = keep_path([both[0], both[1]], i32(0, 1, 2, 3).view(1, 4), i32(10), i32(0, 3, -1, -1, -1).view(1, 5), i32(2))
    assert lens.tolist() == [7] and torch.equal(both, want)
    with pytest.raises(ValueError, match="pool 2 shares memory"):
        keep_path([both[0], both[1], both[0]], i32(0, 1, 2, 3).view(1, 4), i32(10), i32(0, 3, -1, -1, -1).view(1, 5), i32(2))
    assert torch.equal(both, want)
