"""CPU checks of the engine's steps over trees of drafts: what they refuse, with nothing changed by it."""

from __future__ import annotations

import pytest
import torch

from engine.cache.allocator import BlockAllocator
from engine.cache.kv_cache import pack_tables


class HostCache:
    """The host side of a PagedKVCache; moves on the device are counted only."""

    device = torch.device("cpu")

    def __init__(self, num_blocks=32, block_size=4):
        self.alloc = BlockAllocator(num_blocks, block_size)
        self.moves = 0

    def device_tables(self, tables):
        return pack_tables(tables, "cpu")

    def keep_path(self, block_tables, kv_lens, path, n):
        self.moves += 1

    def rollback(self, table, new_length):
        self.alloc.rollback(table, new_length)


def state(cache, tables):
    return [(t.length, list(t.blocks)) for t in tables], list(cache.alloc._free)


def verdict(*rows, T):
    """Each row: the new tokens of a sequence."""
    from kernels.draft_tree import Verdict

    n = [len(r) for r in rows]
    pad = [r + [-1] * (T - len(r)) for r in rows]
    path = [list(range(k)) + [-1] * (T - k) for k in n]
    return Verdict(torch.tensor(pad), torch.tensor(path, dtype=torch.int32), torch.tensor(n, dtype=torch.int32))


def test_a_tree_step_ends_once():
    """Ending a step moves rows within the cache: a second time, or after the tables changed, the rows it
    would take have been overwritten or belong to something else."""
    from engine.attention import begin_step, end_tree_step

    cache = HostCache()
    tables = [cache.alloc.new_sequence() for _ in range(2)]
    step = begin_step(cache, tables, 5, parents=[-1, 0, 0, 1, 2])
    v = verdict([7, 8, 9], [4], T=5)
    assert end_tree_step(cache, step, v) == [[7, 8, 9], [4]] and [t.length for t in tables] == [3, 1]
    was = state(cache, tables)
    with pytest.raises(ValueError, match="ended"):
        end_tree_step(cache, step, v)
    assert cache.moves == 1 and state(cache, tables) == was
    step = begin_step(cache, tables, 5, parents=[-1, 0, 0, 1, 2])
    cache.rollback(tables[1], 2)
    was = state(cache, tables)
    with pytest.raises(ValueError, match="ended"):
        end_tree_step(cache, step, v)
    assert cache.moves == 1 and state(cache, tables) == was


@pytest.mark.parametrize("what", ["nodes", "device"])
def test_begin_step_refuses_before_it_reserves(what):
    """Trees that no kernel takes are refused while the tables are as they were, not by the first layer."""
    from engine.attention import begin_step

    cache = HostCache(num_blocks=600)
    tables = [cache.alloc.new_sequence()]
    was = state(cache, tables)
    if what == "nodes":
        with pytest.raises(ValueError, match="at most 1024"):
            begin_step(cache, tables, 1025, parents=[-1] * 1025)
    else:
        parents = FakeCudaTensor(torch.tensor([-1, 0, 0], dtype=torch.int32))
        cache.device = torch.device("cuda", 1)
        with pytest.raises(RuntimeError, match="one CUDA device"):
            begin_step(cache, tables, 3, parents=parents)
    assert state(cache, tables) == was


class FakeCudaTensor(torch.Tensor):
    """An int32 host tensor that says it is on the first GPU."""

    @staticmethod
    def __new__(cls, t):
        return t.as_subclass(cls)

    is_cuda = True
    device = torch.device("cuda", 0)


def test_begin_step_takes_a_sequence_once():
    """Two trees in the same slots of one sequence would overwrite each other and end twice."""
    from engine.attention import begin_step

    cache = HostCache()
    a, b = cache.alloc.new_sequence(), cache.alloc.new_sequence()
    was = state(cache, [a, b])
    with pytest.raises(ValueError, match="twice"):
        begin_step(cache, [a, b, a], 3, parents=[-1, 0, 0])
    assert state(cache, [a, b]) == was
    assert begin_step(cache, [a, b], 3, parents=[-1, 0, 0]).starts == [0, 0]  # equal, but two sequences


@pytest.mark.parametrize("parents", [[-1, 0, 0.5], [-1.0, 0.0, 1.0], torch.tensor([-1, 0, 2 ** 32]), torch.tensor([-1, 0, -1 - 2 ** 32]),
                                     torch.tensor([True, False, False]), [-1, 0, 2 ** 40]])
def test_begin_step_takes_whole_numbers_in_range(parents):
    """Nothing is cut to an index that it is not: fractions and numbers beyond 32 bits are refused."""
    from engine.attention import begin_step

    cache = HostCache()
    tables = [cache.alloc.new_sequence()]
    with pytest.raises(ValueError, match="parent"):
        begin_step(cache, tables, 3, parents=parents)
    assert state(cache, tables) == state(HostCache(), [HostCache().alloc.new_sequence()])


@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.int8, torch.int16])
def test_begin_step_takes_any_kind_of_whole_number(kind):
    from engine.attention import begin_step

    cache = HostCache()
    step = begin_step(cache, [cache.alloc.new_sequence()], 3, parents=torch.tensor([[-1, 0, 1]], dtype=kind))
    assert step.parents.dtype == torch.int32 and step.parents.tolist() == [[-1, 0, 1]]
