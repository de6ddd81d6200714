"""Eviction from a paged KV cache by what its tokens have received of the attention (``ops_weights`` adds it up), for every
layer and kv head apart. No reference counterpart.

``kv`` is the engine's contiguous [layers, 2, blocks, block_size, kv_heads, ...] cache as ``runner.allocate_kv_cache`` makes
it, 16-bit or 4-bit (uint8, last dimension 68), ``key_weights`` fp32 [layers, rows, kv_heads, width] as
``runner.allocate_key_weights`` makes it. Nothing synchronizes; calls can be captured into HIP graphs.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..ops_fp4 import _ids, _on, _table
from .kv_pages import _context, pages_of


def evict_kv_tokens(kv: torch.Tensor, key_weights: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                    budget: int, *, recent: int = 0, sinks: int = 0, weight_rows: torch.Tensor | None = None,
                    new_blocks: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Brings every sequence longer than ``budget`` down to it: its first ``sinks`` and last ``recent`` tokens stay, and of
    the others, in every layer and kv head apart, the budget - sinks - recent with the largest weight (of equal ones the
    earliest; NaN counts as larger than any number). They move in their order to the first ``budget`` slots of the sequence
    and their weights to the first places of its row; the slots and places behind keep what they held. Sequences within the
    budget, and those whose row (``weight_rows`` [B], sequence b's is row b where it is left out) is outside
    key_weights, stay as they are.

    Returns the tables (int32 [B, max_blocks], -1 behind the blocks still in use) and lengths (int32 [B]) to go on with. The
    keys hold the positions they were stored with: the next token's position is that of the text, its slot that of the
    length (``evicted`` of ``runner.prepare_decode_context``).

    A block that several rows name (a forked prefix) must not be written: ``new_blocks`` int [B, max_blocks] names blocks,
    which no row names, that take the place of the sequence's own as it is brought down (-1: its own). Every row over the
    budget needs one for each block among its first ceil(budget / block_size) that another row names too;
    ``checks.eviction_violations`` looks a step over.

    A block that was written no longer holds the text that it was filled from: its tokens are others in every layer and kv head.
    Where blocks are found again by their text (a prefix cache's hashes), those written in place and the new ones lose their
    hash, a sequence that was brought down registers none for its further blocks, and a block whose hash is to stay needs a new
    one in its place."""
    planes, blocks, bs, slot, scale = pages_of(kv)
    layers, hk = planes // 2, kv.shape[4]
    if slot % hk or (slot // hk) % 16 or slot // hk > 4096:
        raise ValueError(f"evict_kv_tokens: a token's head must be a multiple of 16 bytes up to 4096, got {slot // max(hk, 1)}")
    if key_weights.dtype != torch.float32:
        raise TypeError(f"evict_kv_tokens: key_weights must be fp32, got {key_weights.dtype}")
    if key_weights.dim() != 4 or key_weights.shape[0] != layers or key_weights.shape[2] != hk or not key_weights.is_contiguous():
        raise ValueError(f"evict_kv_tokens: key_weights must be contiguous [{layers}, rows, {hk}, width], got "
                         f"{tuple(key_weights.shape)}")
    if budget <= 0 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"evict_kv_tokens: budget {budget} must be positive and hold sinks {sinks} and recent {recent}")
    more = [t for t in (weight_rows, new_blocks) if t is not None]
    dev, bt, bt_stride, lens = _context(kv, block_tables, context_lens, key_weights, *more)
    batch, mb = lens.numel(), bt.shape[1]
    if key_weights.shape[3] < mb * bs:
        raise ValueError(f"evict_kv_tokens: key_weights hold {key_weights.shape[3]} tokens a row, the tables reach {mb * bs}")
    rows = None
    if weight_rows is not None:
        if weight_rows.numel() != batch:
            raise ValueError("evict_kv_tokens: weight_rows must hold one row per sequence")
        rows = _ids(weight_rows, "weight_rows")
    elif key_weights.shape[1] < batch:
        raise ValueError(f"evict_kv_tokens: key_weights have {key_weights.shape[1]} rows for {batch} sequences")
    into, into_stride = None, 0
    if new_blocks is not None:
        if new_blocks.dim() != 2 or new_blocks.shape[0] < batch or new_blocks.shape[1] != mb:
            raise ValueError(f"evict_kv_tokens: new_blocks must be [{batch}, {mb}], got {tuple(new_blocks.shape)}")
        into, into_stride = _table(new_blocks)
    tables = torch.empty(batch, mb, dtype=torch.int32, device=dev)
    left = torch.empty(batch, dtype=torch.int32, device=dev)
    if batch == 0:
        return tables, left
    if mb == 0 or layers == 0 or key_weights.shape[1] == 0:
        raise ValueError("evict_kv_tokens: empty cache, tables or weights")
    if budget >= mb * bs:  # (nothing is longer)
        budget, sinks, recent = mb * bs, 0, 0
    lib = _lib.load()
    with _on(dev):
        moves = torch.empty(layers, batch, hk, budget + 1, 2, dtype=torch.int32, device=dev)
        _lib.check(lib.vox_evict_kv_tokens(kv.data_ptr(), layers, blocks, bs, hk, slot // hk, scale // hk, bt.data_ptr(),
                                           bt_stride, mb, lens.data_ptr(), batch, key_weights.data_ptr(),
                                           None if rows is None else rows.data_ptr(), key_weights.shape[1],
                                           key_weights.shape[3], int(budget), int(sinks), int(recent),
                                           None if into is None else into.data_ptr(), into_stride, moves.data_ptr(),
                                           tables.data_ptr(), left.data_ptr(), _lib.stream_handle(dev)),
                   "evict_kv_tokens")
    return tables, left
