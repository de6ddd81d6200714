"""The care of a paged KV cache's blocks: sequences forked, live blocks moved together, in every layer's K and V in one
call. No reference counterpart beyond the block-prefix copy (kv_copy.py); the engine's block manager decides which blocks
are whose, these move the bytes and rewrite the tables on the device.

``kv`` is the engine's contiguous [layers, 2, blocks, block_size, kv_heads, ...] cache as ``runner.allocate_kv_cache``
makes it, bf16 or 4-bit (uint8, last dimension 68). Tables and lengths are the forward context's: int32 on the GPU,
entries past a row's context ignored. Nothing synchronizes; calls can be captured into HIP graphs.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..ops import _as_i32, _check_cuda, _flat
from ..ops_fp4 import ROW_BYTES, _ids, _on, _table


def pages_of(kv: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(planes, blocks, block_size, slot bytes, scale bytes) of a cache [layers, 2, blocks, block_size, kv_heads, width]."""
    if kv.dim() != 6 or kv.shape[1] != 2:
        raise ValueError(f"kv must be [layers, 2, blocks, block_size, kv_heads, width], got {tuple(kv.shape)}")
    if not kv.is_contiguous():
        raise ValueError("kv must be contiguous")
    layers, kvs, blocks, block_size, heads, width = kv.shape
    if kv.dtype == torch.uint8:
        if width != ROW_BYTES:
            raise ValueError(f"a uint8 cache is 4-bit: its last dimension must be {ROW_BYTES}, got {width}")
        return layers * kvs, blocks, block_size, heads * 64, heads * 4
    return layers * kvs, blocks, block_size, heads * width * kv.element_size(), 0


def _context(kv: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, *more: torch.Tensor):
    dev = _check_cuda(kv, block_tables, context_lens, *more)
    if block_tables.dim() != 2 or block_tables.shape[0] < context_lens.numel():
        raise ValueError("block_tables must be [B, max_blocks] and context_lens [B]")
    bt, bt_stride = _table(block_tables)
    return dev, bt, bt_stride, _as_i32(_flat(context_lens), "context_lens")


def fork_kv_blocks(kv: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, parents: torch.Tensor,
                   new_blocks: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Children that go on from where rows ``parents`` ([F], rows of block_tables [B, max_blocks], a row may be forked
    several times) are: each shares its parent's full blocks, and the filled slots of a partly filled last block are copied
    to new_blocks[i], which takes its place. Returns the children's tables int32 [F, max_blocks] (-1 past the context) and
    lengths int32 [F].

    ``new_blocks`` ([F]) are blocks that no table names, no two the same; one whose parent ends with a full block stays
    unused. A parent outside the batch gives an empty child; a partly filled block that is not in the cache, or a new block
    that is not, leaves -1 in the child's table."""
    planes, blocks, bs, slot, scale = pages_of(kv)
    dev, bt, bt_stride, lens = _context(kv, block_tables, context_lens, parents, new_blocks)
    who, fresh = _ids(parents, "parents"), _ids(new_blocks, "new_blocks")
    n, mb = who.numel(), bt.shape[1]
    if fresh.numel() != n:
        raise ValueError("fork_kv_blocks: one new block per parent")
    tables = torch.empty(n, mb, dtype=torch.int32, device=dev)
    child_lens = torch.empty(n, dtype=torch.int32, device=dev)
    if n == 0:
        return tables, child_lens
    lib = _lib.load()
    with _on(dev):
        _lib.check(lib.vox_fork_kv_blocks(kv.data_ptr(), planes, blocks, bs, slot, scale, bt.data_ptr(), bt_stride, mb,
                                          lens.data_ptr(), lens.numel(), who.data_ptr(), fresh.data_ptr(), n,
                                          tables.data_ptr(), child_lens.data_ptr(), _lib.stream_handle(dev)),
                   "fork_kv_blocks")
    return tables, child_lens


def compact_kv_blocks(kv: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Moves the live blocks (those that a row of block_tables [B, max_blocks] names within context_lens [B]) to the front
    of the cache: with L of them, those at or past L go to the dead blocks below L, the lowest to the lowest; a block
    shared by several rows moves once. A sequence is freed by leaving it out (or by a length of 0): afterwards the blocks
    from L on are free.

    Returns the tables with the new numbers (int32 [B, max_blocks], -1 past the context, entries that name no block as
    they were), the new number of every block (int32 [blocks], -1: dead), and L (int32 [1]). At most 2^18 blocks."""
    planes, blocks, bs, slot, scale = pages_of(kv)
    dev, bt, bt_stride, lens = _context(kv, block_tables, context_lens)
    batch, mb = lens.numel(), bt.shape[1]
    tables = torch.empty(batch, mb, dtype=torch.int32, device=dev)
    book = torch.empty(3 * blocks + 2, dtype=torch.int32, device=dev)
    remap, live, moves = book[:blocks], book[blocks:blocks + 1], book[blocks + 1:]
    lib = _lib.load()
    with _on(dev):
        _lib.check(lib.vox_compact_kv_blocks(kv.data_ptr(), planes, blocks, bs, slot, scale, bt.data_ptr(), bt_stride, mb,
                                             lens.data_ptr(), batch if mb else 0, tables.data_ptr(), remap.data_ptr(),
                                             live.data_ptr(), moves.data_ptr(), _lib.stream_handle(dev)),
                   "compact_kv_blocks")
    return tables, remap, live
