"""A step of speculative decoding with a tree of drafted tokens, on B200 (sm_100a).

The reference drafts one greedy chain per step and verifies it on the host
(engine/decode/speculative.py:24-123). Here the drafts of a sequence may form a
tree, a batch of trees is served at once, and nothing waits for the host:

* ``tree_attention``  the T nodes attend over the paged history and over their
                      ancestors (``paged_attention`` is the same for a chain).
* ``verify_drafts``   which nodes are kept and which token follows, by speculative
                      sampling from given uniform numbers, or greedily.
* ``keep_path``       the kept nodes' K/V rows move behind the history, in every
                      layer's pool.

A tree is an int32 tensor ``parents``, (T,) for one tree shared by the batch or
(B, T): parents[i] < i is node i's parent, -1 none. Node 0 is the root, the last
token that is already decided; a chain is ``[-1, 0, 1, ..]``. Smaller trees of a
batch are padded with nodes of parent -1 (and any token), which belong to no path. The nodes sit
in the last T slots of their sequence, written by
``kernels.flash_attention.rope_append(..., parents=parents)``.

Every call is asynchronous on the current stream of its tensors' device, can be
captured into a CUDA graph, and allocates its outputs (and workspace) with torch.
Bad contents of device tensors (parents, tokens, block ids, probabilities) are
reported in the device status word (``kernels._lib.device_status``).
"""

from __future__ import annotations

import ctypes
import math
from array import array
from functools import lru_cache
from operator import attrgetter
from typing import NamedTuple, Sequence

import torch

from kernels import _lib
from kernels.flash_attention import _DTYPES, _kernel_ready, _rope_tables, _require

_PROB_DTYPES = {**_DTYPES, torch.float32: _lib.CIE_DTYPE_FP32}
_I32 = torch.int32
_SHAPE, _DTYPE = attrgetter("shape"), attrgetter("dtype")

# These calls run once per layer or per token, and a small one takes the GPU less time
# than the interpreter needs to describe it: tensors are asked for as little as the
# checks need, and what depends on sizes alone is kept.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


@lru_cache(maxsize=4096)
def _i64s(strides: tuple) -> ctypes.Array:
    """The strides as a C array, read only by the library."""
    return (ctypes.c_int64 * len(strides))(*strides)


@lru_cache(maxsize=4096)
def _tree_workspace(*sizes) -> int:
    """Bytes of workspace; the last of the sizes is the device."""
    with torch.cuda.device(sizes[-1]):
        return _require().cie_tree_attn_workspace(*sizes[:-1])


def _require_lib() -> ctypes.CDLL:
    return _lib._LIB or _require()


def _call(index: int, fn, *args) -> int:
    """fn(*args, stream) on device ``index`` and its current stream."""
    if index == torch.cuda.current_device():
        return fn(*args, _raw_stream(index))
    with torch.cuda.device(index):
        return fn(*args, _raw_stream(index))


class Verdict(NamedTuple):
    """What ``verify_drafts`` decides; -1 fills the rows behind the entries."""

    tokens: torch.Tensor  # (B, T) the kept drafts, then the last token: n[b] entries
    path: torch.Tensor    # (B, T) int32 the kept nodes, root first: n[b] entries
    n: torch.Tensor       # (B,) int32


def _parents(parents: torch.Tensor, B: int, T: int, index: int, what: str
             ) -> tuple[torch.Tensor, int]:
    """(tensor, stride between the sequences' trees)"""
    if parents.dtype is not _I32:
        raise ValueError(f"{what}: parents must be int32, got {parents.dtype}")
    shape = parents.shape
    if shape != (T,) and shape != (B, T):
        raise ValueError(f"{what}: parents must be ({T},) or ({B}, {T}), got {tuple(shape)}")
    if parents.get_device() != index:
        raise RuntimeError(f"{what} requires all tensors on one CUDA device")
    if T > _lib.CIE_MAX_TREE:
        raise ValueError(f"{what}: {T} nodes, at most {_lib.CIE_MAX_TREE}")
    if T > 1 and parents.stride(-1) != 1:
        parents = parents.contiguous()
    return parents, (parents.stride(0) if len(shape) == 2 and B > 1 else 0)


def tree_attention(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    parents: torch.Tensor,
    scale: float | None = None,
    *,
    rope: tuple[torch.Tensor, torch.Tensor] | None = None,
    split_tokens: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of a tree of drafted tokens over each sequence's paged history.

    As ``paged_attention`` (same q, pools, tables, ``rope``, ``split_tokens`` and
    ``out``), with q (B, Hq, T, D) holding one row per node. kv_lens counts the T
    nodes: node i's K/V are in slot kv_lens[b] - T + i. It sees the history
    before them, itself and its ancestors by ``parents``. ``rope`` rotates its q at
    position kv_lens[b] - T + depth. Returns (B, Hq, T, D) in q's dtype; zeros for
    kv_lens[b] = 0. NaN or infinity in a node's K or V reaches only the nodes that
    see it. ``scale`` must be positive (default 1 / sqrt(D)).
    """
    index = q.get_device()
    if index < 0:
        raise RuntimeError("tree_attention requires CUDA tensors")
    if q.ndim != 4:
        raise ValueError(f"q must be (B, Hq, T, D), got {tuple(q.shape)}")
    B, Hq, T, D = q.shape
    shape = k_pool.shape
    if len(shape) != 4 or shape != v_pool.shape:
        raise ValueError("k_pool/v_pool must both be (num_blocks, block_size, Hkv, D)")
    nb, bs, Hkv, Dk = shape
    if Dk != D:
        raise ValueError(f"pool head_dim {Dk} != q head_dim {D}")
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"num_heads {Hq} must be a multiple of num_kv_heads {Hkv}")
    dtype = q.dtype
    if dtype not in _DTYPES or k_pool.dtype is not dtype or v_pool.dtype is not dtype:
        raise ValueError(f"tree_attention expects matching FP16/BF16 q and pools, got "
                         f"{dtype}/{k_pool.dtype}/{v_pool.dtype}")
    if block_tables.dtype is not _I32 or kv_lens.dtype is not _I32:
        raise ValueError("block_tables and kv_lens must be int32")
    tab_shape = block_tables.shape
    if len(tab_shape) != 2 or tab_shape[0] != B or kv_lens.shape != (B,):
        raise ValueError("block_tables must be (B, max_blocks) and kv_lens (B,)")
    if not (k_pool.get_device() == v_pool.get_device() == block_tables.get_device()
            == kv_lens.get_device() == index):
        raise RuntimeError("tree_attention requires all tensors on q's CUDA device")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("k_pool/v_pool must be contiguous")
    k_ptr, v_ptr = k_pool.data_ptr(), v_pool.data_ptr()
    if (k_ptr | v_ptr) & 15:
        raise ValueError("k_pool/v_pool must be 16-byte aligned")
    parents, par_sb = _parents(parents, B, T, index, "tree_attention")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != (B, Hq, T, D) or out.dtype is not dtype or out.get_device() != index:
        raise ValueError(f"out must be a ({B}, {Hq}, {T}, {D}) {dtype} tensor on {q.device}")
    elif out.stride(3) != 1:
        raise ValueError("out must have a unit innermost stride")
    if B == 0 or T == 0 or Hq == 0:
        return out
    qs, q_ptr = q.stride(), q.data_ptr()
    if qs[3] != 1 or (qs[0] | qs[1] | qs[2]) & 7 or q_ptr & 15:
        q = _kernel_ready(q)
        qs, q_ptr = q.stride(), q.data_ptr()
    if not block_tables.is_contiguous():
        block_tables = block_tables.contiguous()
    if not kv_lens.is_contiguous():
        kv_lens = kv_lens.contiguous()
    cos = sin = None
    max_pos = 0
    if rope is not None:
        cos, sin, max_pos = _rope_tables(rope, q.device)
        if cos.shape[1] * 2 != D:
            raise ValueError(f"rope tables are for head_dim {cos.shape[1] * 2}, q has {D}")
        cos, sin = _kernel_ready(cos), _kernel_ready(sin)
    max_blocks = tab_shape[1]
    split_tokens = int(split_tokens)
    ws_bytes = _tree_workspace(B, Hq, Hkv, T, D, bs, max_blocks, split_tokens, index)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    rc = _call(index, _require_lib().cie_tree_attn,
               q_ptr, k_ptr, v_ptr, block_tables.data_ptr(), kv_lens.data_ptr(),
               parents.data_ptr(), par_sb, out.data_ptr(), B, Hq, Hkv, T, D, nb, bs, max_blocks,
               _i64s(qs[:3]), _i64s(out.stride()[:3]),
               1.0 / math.sqrt(D) if scale is None else float(scale), _DTYPES[dtype],
               None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(),
               max_pos, split_tokens, None if ws is None else ws.data_ptr(), ws_bytes)
    if rc:
        _lib.check(rc, "tree_attention")
    return out


def verify_drafts(
    tokens: torch.Tensor,
    parents: torch.Tensor,
    target_probs: torch.Tensor,
    uniforms: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
) -> Verdict:
    """Which drafted tokens are kept, and the token that follows them.

    tokens: (B, T) int32 / int64, node 0 the last token already decided.
    target_probs: (B, T, V) fp32 / fp16 / bf16, row i the target model's
    distribution after node i (unit innermost stride). uniforms: (B, T) fp32 in
    [0, 1), entry i for node i, entry 0 for the last token. draft_probs:
    (B, Td, V), row i the distribution from which the children of node i were
    drawn independently; nodes from Td <= T on are leaves, so a chain of T - 1
    drafts passes its T - 1 rows. None: the children were chosen (the draft's
    best tokens, say) rather than drawn.

    The children x of a node with rows p and q are tested in index order: kept if
    u q(x) m < r(x), where r = p and m = 1 at first; otherwise r becomes
    max(r - m q, 0) and m its sum. If no child is kept the last token is drawn
    from r by its cumulative sum. For rows that sum to 1 the kept tokens are then
    distributed as if drawn from the target alone (16-bit rows: to their rounding; rows
    cut to their likeliest tokens must be normalised again). Without ``uniforms`` the walk is greedy: the child that
    drafted the row's largest entry (the lowest such index) is kept; rows may then be
    logits.

    Returns a ``Verdict``: tokens[b, :n[b]] are the new tokens, the last of them
    not yet in the cache, and path[b, :n[b]] the kept nodes, root first. A row of
    probabilities without a finite positive sum gives the token -1.
    """
    index = target_probs.get_device()
    if index < 0:
        raise RuntimeError("verify_drafts requires CUDA tensors")
    if target_probs.ndim != 3:
        raise ValueError(f"target_probs must be (B, T, V), got {tuple(target_probs.shape)}")
    B, T, V = target_probs.shape
    dtype = target_probs.dtype
    if T == 0 or V == 0:
        raise ValueError("verify_drafts needs at least one node and one token")
    if dtype not in _PROB_DTYPES:
        raise ValueError(f"verify_drafts expects FP32, FP16 or BF16 rows, got {dtype}")
    tok_type = tokens.dtype
    if tok_type is not _I32 and tok_type is not torch.int64:
        raise ValueError(f"tokens must be int32 or int64, got {tok_type}")
    if tokens.shape != (B, T):
        raise ValueError(f"tokens must be ({B}, {T}), got {tuple(tokens.shape)}")
    if tokens.get_device() != index:
        raise RuntimeError("verify_drafts requires all tensors on one CUDA device")
    parents, par_sb = _parents(parents, B, T, index, "verify_drafts")
    if T > 1 and tokens.stride(1) != 1:
        tokens = tokens.contiguous()
    ps = target_probs.stride()
    if ps[2] != 1 and V > 1:
        target_probs = target_probs.contiguous()
        ps = target_probs.stride()
    u_ptr, u_sb, q_ptr, q_strides, Td = None, 0, None, None, 0
    if uniforms is not None:
        if uniforms.dtype is not torch.float32 or uniforms.shape != (B, T):
            raise ValueError(f"uniforms must be a ({B}, {T}) float32 tensor")
        if uniforms.get_device() != index:
            raise RuntimeError("verify_drafts requires all tensors on one CUDA device")
        if T > 1 and uniforms.stride(1) != 1:
            uniforms = uniforms.contiguous()
        u_ptr, u_sb = uniforms.data_ptr(), uniforms.stride(0)
    if draft_probs is not None:
        if uniforms is None:
            raise ValueError("draft_probs are for sampling: pass uniforms too")
        qshape = draft_probs.shape
        if len(qshape) != 3 or qshape[0] != B or qshape[2] != V or not 1 <= qshape[1] <= T:
            raise ValueError(f"draft_probs must be ({B}, 1..{T}, {V}), got {tuple(qshape)}")
        if draft_probs.dtype is not dtype:
            raise ValueError(f"draft_probs must be {dtype} like target_probs")
        if draft_probs.get_device() != index:
            raise RuntimeError("verify_drafts requires all tensors on one CUDA device")
        if draft_probs.stride(2) != 1 and V > 1:
            draft_probs = draft_probs.contiguous()
        Td = qshape[1]
        q_ptr, q_strides = draft_probs.data_ptr(), _i64s(draft_probs.stride()[:2])
    out = torch.empty_like(tokens, memory_format=torch.contiguous_format)
    path = torch.empty_like(out, dtype=_I32)
    n = path.new_empty(B)
    if B:
        rc = _call(index, _require_lib().cie_verify_drafts,
                   tokens.data_ptr(), tokens.stride(0), tok_type is torch.int64,
                   parents.data_ptr(), par_sb, target_probs.data_ptr(), _i64s(ps[:2]), q_ptr,
                   q_strides, Td, u_ptr, u_sb, B, T, V, _PROB_DTYPES[dtype], out.data_ptr(),
                   path.data_ptr(), n.data_ptr())
        if rc:
            _lib.check(rc, "verify_drafts")
    return Verdict(out, path, n)


def keep_path(
    pools: Sequence[torch.Tensor],
    block_tables: torch.Tensor,
    kv_lens: torch.Tensor,
    path: torch.Tensor,
    n: torch.Tensor,
) -> torch.Tensor:
    """Move the kept nodes' rows to the slots behind the history, in place.

    pools: the K and V pools of every layer, each (num_blocks, block_size, Hkv, D),
    all of one shape and dtype, none of them twice. kv_lens: int32 (B,), counting the T nodes. path:
    int32 (B, T) and n: int32 (B,) as ``verify_drafts`` returns them. Slot
    base + i takes the row of slot base + path[b, i] for i < n[b], where
    base = kv_lens[b] - T; nothing of an idle sequence (kv_lens[b] = 0) moves. Rows
    elsewhere stay as they are. Returns the new
    lengths, max(0, base + n[b]), int32 (B,).
    """
    index = path.get_device()
    if index < 0:
        raise RuntimeError("keep_path requires CUDA tensors")
    if path.ndim != 2 or path.dtype is not _I32:
        raise ValueError("path must be int32 (B, T)")
    B, T = path.shape
    if block_tables.dtype is not _I32 or kv_lens.dtype is not _I32 or n.dtype is not _I32:
        raise ValueError("block_tables, kv_lens and n must be int32")
    if block_tables.ndim != 2 or block_tables.shape[0] != B or kv_lens.shape != (B,) \
            or n.shape != (B,):
        raise ValueError("block_tables must be (B, max_blocks), kv_lens and n (B,)")
    if not block_tables.get_device() == kv_lens.get_device() == n.get_device() == index:
        raise RuntimeError("keep_path requires all tensors on one CUDA device")
    if not 1 <= T <= _lib.CIE_MAX_TREE:
        raise ValueError(f"keep_path: {T} nodes, 1 to {_lib.CIE_MAX_TREE} are served")
    if len(pools) == 0:
        raise ValueError("keep_path needs at least one pool")
    shape, dtype = pools[0].shape, pools[0].dtype
    if len(shape) != 4:
        raise ValueError("pools must be (num_blocks, block_size, Hkv, D)")
    if dtype not in _DTYPES:
        raise ValueError(f"keep_path expects FP16/BF16 pools, got {dtype}")
    if list(map(_SHAPE, pools)).count(shape) != len(pools) \
            or set(map(_DTYPE, pools)) != {dtype} \
            or not all(map(torch.Tensor.is_contiguous, pools)):
        raise ValueError("pools must be contiguous and of one shape and dtype")
    if set(map(torch.Tensor.get_device, pools)) != {index}:
        raise RuntimeError("keep_path requires all tensors on one CUDA device")
    new_lens = torch.empty_like(kv_lens, memory_format=torch.contiguous_format)
    if B == 0:
        return new_lens
    if not block_tables.is_contiguous():
        block_tables = block_tables.contiguous()
    kv_lens, path, n = kv_lens.contiguous(), path.contiguous(), n.contiguous()
    ptrs = array("Q", map(torch.Tensor.data_ptr, pools))
    rc = _call(index, _require_lib().cie_keep_path,
               ptrs.buffer_info()[0], len(pools), block_tables.data_ptr(), kv_lens.data_ptr(), path.data_ptr(),
               n.data_ptr(), new_lens.data_ptr(), B, T, shape[0], shape[1],
               block_tables.shape[1], shape[2] * shape[3] * 2)
    if rc:
        _lib.check(rc, "keep_path")
    return new_lens
