"""CPU checks of rope_append(parents=): tables, lengths and pools that the kernel would read or write out
of range are refused before it is called."""

from __future__ import annotations

import pytest
import torch


class OnGpu(torch.Tensor):
    """A host tensor that says it is on a GPU: enough to reach the argument checks."""

    @staticmethod
    def __new__(cls, t):
        return t.as_subclass(cls)

    is_cuda = True


@pytest.mark.parametrize("change,text", [
    (dict(block_tables=(1, 4)), "block_tables must be"),       # fewer rows than sequences
    (dict(block_tables=(8,)), "block_tables must be"),
    (dict(start_pos=(1,)), "start_pos"),
    (dict(start_pos=(2, 1)), "start_pos"),
    (dict(k_pool="strided"), "contiguous"),
    (dict(v_pool="strided"), "contiguous"),
])
def test_rope_append_tree_refuses_what_does_not_fit(monkeypatch, change, text):
    from kernels import flash_attention as fa

    called = []
    monkeypatch.setattr(fa, "_require", lambda: type("Lib", (), {"cie_rope_append_tree": lambda *a: called.append(a) or 0})())
    args = dict(k_new=torch.zeros(2, 3, 2, 16), v_new=torch.zeros(2, 3, 2, 16), k_pool=torch.zeros(4, 16, 2, 16), v_pool=torch.zeros(4, 16, 2, 16))
    args = {k: v.to(torch.bfloat16) for k, v in args.items()}
    args.update(block_tables=torch.zeros(2, 4), start_pos=torch.zeros(2), parents=torch.tensor([-1, 0, 1]))
    for name, how in change.items():
        args[name] = torch.zeros(4, 16, 2, 32, dtype=torch.bfloat16)[..., :16] if how == "strided" else torch.zeros(*how)
    for name in ("block_tables", "start_pos", "parents"):
        args[name] = args[name].to(torch.int32)
    with pytest.raises(ValueError, match=text):
        fa.rope_append(**{k: OnGpu(v) for k, v in args.items()})
    assert not called


@pytest.mark.gpu
def test_rope_append_tree_refuses_other_devices(cuda):
    from kernels.flash_attention import rope_append

    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(k_new=z(2, 3, 2, 16), v_new=z(2, 3, 2, 16), k_pool=z(4, 16, 2, 16), v_pool=z(4, 16, 2, 16),
                block_tables=i(2, 4), start_pos=i(2), parents=i(3) - 1)
    for name in ("v_new", "k_pool", "v_pool", "block_tables", "start_pos", "parents"):
        with pytest.raises(RuntimeError, match="one CUDA device"):
            rope_append(**{**good, name: good[name].cpu()})
    rope_append(**good)
