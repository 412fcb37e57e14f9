"""Waits that run out while a CTA has the next piece's q and parents on their way to shared memory."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_draft_tree_gpu import _clean_status, run, setup  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,bs,T,Hq", [(128, 16, 30, 16), (64, 20, 9, 16), (64, 16, 100, 8)])
def test_many_pieces_a_cta(cuda, D, bs, T, Hq):
    """Many short sequences: every CTA goes through several pieces. With no time to wait the kernel says so,
    waits for its own copies, and the next calls are right, also of another tree size."""
    from kernels import _lib

    rs = np.random.RandomState(D)
    s = setup(300, T, Hq, 4, D, bs, torch.bfloat16, [T + int(x) for x in rs.randint(0, 700, 300)], seed=100)
    t = setup(40, 5, Hq, 4, D, bs, torch.bfloat16, [5 + int(x) for x in rs.randint(0, 900, 40)], seed=101)
    want = run(s), run(t)
    torch.cuda.synchronize()
    for _ in range(5):
        old = _lib.set_wait_limit(0)
        try:
            run(s)
            torch.cuda.synchronize()
        finally:
            _lib.set_wait_limit(old)
        assert _lib.device_status() == _lib.CIE_DEV_TIMEOUT
        assert torch.equal(run(t), want[1]) and torch.equal(run(s), want[0])
