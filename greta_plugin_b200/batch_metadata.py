"""Metadata of a packed serving batch from the requests' lengths, on the GPU.

The packed calls of this package (packed_dynamic_conv_triton,
packed_causal_conv1d, packed_selective_scan) take `starts` and `has_initial`,
and the attention layers between them a slot in their paged cache for every
token. packed_batch_metadata makes all of them in one launch from lengths that
may live on the device only (no host synchronisation), so a step whose lengths
change from replay to replay can be captured in a CUDA graph. The reference
takes these tensors from vLLM's metadata (greta_vllm/conv.py:73-103), which is
built on the host.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _capi
from .causal_conv import same_device

MAX_REQUESTS = 16384


class PackedBatch(NamedTuple):
    starts: torch.Tensor                  # [N + 1] int32 token offsets
    has_initial: torch.Tensor             # [N] int8: the request has cached tokens
    seq_idx: torch.Tensor                 # [T] int32 request of each token, -1 behind the last
    positions: torch.Tensor               # [T] int64 position in its request, 0 behind the last
    slot_map: Optional[torch.Tensor]      # [T] int64 slot in the paged cache, -1 for none
    blocks_used: Optional[torch.Tensor]   # [1] int32 new blocks that the step asks for


def packed_batch_metadata(query_lens: torch.Tensor, context_lens: torch.Tensor, num_tokens: int,
                          block_tables: Optional[torch.Tensor] = None, block_size: int = 0,
                          free_blocks: Optional[torch.Tensor] = None) -> PackedBatch:
    """The metadata of a step that adds query_lens[i] tokens (0: none) to request
    i, which has context_lens[i] cached.

    query_lens, context_lens: [N] int32; negative lengths count as 0.
    num_tokens: rows T of the packed tensors, at least the sum of query_lens;
    tokens past it are dropped (the offsets end at T), though their blocks are
    asked for like the others'.

    With block_tables ([N, M] int32, contiguous rows, updated in place) the
    requests' tables grow by the blocks that their new tokens begin, taken from
    the front of free_blocks ([K] int32) in request order, and every token gets
    its slot: block * block_size + position % block_size. blocks_used is the
    number of blocks asked for: above K, the list ran out, and the entries and
    slots without a block are -1, as are slots past the table's width M. It counts
    the blocks of all query_lens: those that only dropped tokens would begin, and
    those past the table's width, stand in no table, so a caller whose T may be
    below the sum clamps query_lens first, or those blocks are lost to it.
    """
    for name, t in (("query_lens", query_lens), ("context_lens", context_lens)):
        if t.dim() != 1 or t.dtype != torch.int32:
            raise ValueError(f"{name} must be a 1-d int32 tensor, got {t.dtype} {tuple(t.shape)}")
    N, T = query_lens.numel(), int(num_tokens)
    if context_lens.numel() != N:
        raise ValueError(f"context_lens has {context_lens.numel()} entries, query_lens {N}")
    if N > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests, got {N}")
    if T < 0:
        raise ValueError(f"num_tokens must not be negative, got {T}")
    paged = block_tables is not None
    if paged:
        if block_tables.dim() != 2 or block_tables.shape[0] != N or block_tables.dtype != torch.int32:
            raise ValueError(f"block_tables must be [{N}, M] int32, got {block_tables.dtype} "
                             f"{tuple(block_tables.shape)}")
        if block_tables.shape[1] > 1 and block_tables.stride(1) != 1 or \
                N > 1 and block_tables.stride(0) < block_tables.shape[1]:
            raise ValueError("block_tables must have contiguous, separate rows because it is updated in-place")
        if block_size < 1:
            raise ValueError(f"block_size must be at least 1, got {block_size}")
        if free_blocks is None or free_blocks.dim() != 1 or free_blocks.dtype != torch.int32:
            raise ValueError("block_tables need free_blocks, a 1-d int32 tensor")
    elif free_blocks is not None:
        raise ValueError("free_blocks without block_tables")
    same_device("query_lens", query_lens, context_lens=context_lens, block_tables=block_tables,
                free_blocks=free_blocks)
    dev = query_lens.device
    if not query_lens.is_cuda:
        raise ValueError("packed_batch_metadata requires CUDA tensors")
    query_lens, context_lens = query_lens.contiguous(), context_lens.contiguous()
    free_blocks = None if free_blocks is None else free_blocks.contiguous()
    # int32 and int64 results share a buffer each (an allocation costs as much as
    # a third of the kernel's launch)
    starts, seq_idx, used = torch.split_with_sizes(query_lens.new_empty(N + T + 2), (N + 1, T, 1))
    init = torch.empty(N, dtype=torch.int8, device=dev)
    if paged:
        positions, slot_map = torch.empty((2, T), dtype=torch.int64, device=dev).unbind()
    else:
        positions, slot_map, used = torch.empty(T, dtype=torch.int64, device=dev), None, None
    p = _capi.addr
    # a table without entries has no address of its own
    width = block_tables.shape[1] if paged else 0
    table = (p(block_tables) or p(used)) if paged else None
    _capi.call("greta_ssm_batch_metadata", query_lens, p(query_lens), p(context_lens), N, T, p(starts), p(init),
               p(seq_idx), p(positions), table, max(block_tables.stride(0), width) if paged else 0, width,
               block_size if paged else 0, p(free_blocks), free_blocks.numel() if paged else 0, p(slot_map), p(used))
    return PackedBatch(starts, init, seq_idx, positions, slot_map, used)


__all__ = ["PackedBatch", "packed_batch_metadata"]
