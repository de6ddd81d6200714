"""CPU restatement of forking and compacting a paged cache (test infrastructure only; see oracle/__init__.py)."""

from __future__ import annotations

import torch


def copy_slots(kv: torch.Tensor, src: int, dst: int, n: int) -> None:
    """The first n slots of block src over those of block dst in every plane of kv [layers, 2, blocks, block_size, HK,
    width]; a 4-bit cache (uint8, width 68) keeps its slots' codes and scales in two runs."""
    if kv.dtype != torch.uint8:
        kv[:, :, dst, :n] = kv[:, :, src, :n].clone()
        return
    bs, hk = kv.shape[3], kv.shape[4]
    flat = kv.view(*kv.shape[:3], -1)
    at = bs * hk * 64
    flat[:, :, dst, :n * hk * 64] = flat[:, :, src, :n * hk * 64].clone()
    flat[:, :, dst, at:at + n * hk * 4] = flat[:, :, src, at:at + n * hk * 4].clone()


def fork(kv: torch.Tensor, tables, lens, parents, new_blocks):
    """In place on kv; the children's tables and lengths as lists."""
    blocks, bs, width = kv.shape[2], kv.shape[3], len(tables[0])
    child_tables, child_lens = [], []
    for p, fresh in zip(parents, new_blocks):
        n = min(max(lens[p], 0), width * bs) if 0 <= p < len(lens) else 0
        row = list(tables[p][:n // bs]) if n else []
        if n % bs:
            src = tables[p][n // bs]
            ok = 0 <= src < blocks and 0 <= fresh < blocks
            if ok:
                copy_slots(kv, src, fresh, n % bs)
            row.append(fresh if ok else -1)
        child_tables.append(row + [-1] * (width - len(row)))
        child_lens.append(n)
    return child_tables, child_lens


def compact(kv: torch.Tensor, tables, lens):
    """In place on kv; the new tables, every block's new number and how many live, as lists."""
    blocks, bs = kv.shape[2], kv.shape[3]
    rows = [row[:max(0, -(-n // bs))] for row, n in zip(tables, lens)]
    live = sorted({b for row in rows for b in row if 0 <= b < blocks})
    holes = [b for b in range(len(live)) if b not in set(live)]
    remap = [-1] * blocks
    for b in live:
        if b < len(live):
            remap[b] = b
    for src, dst in zip([b for b in live if b >= len(live)], holes):
        remap[src] = dst
        copy_slots(kv, src, dst, bs)
    new = [[remap[b] if 0 <= b < blocks else b for b in row] + [-1] * (len(full) - len(row))
           for row, full in zip(rows, tables)]
    return new, remap, len(live)


def head_rows(kv: torch.Tensor):
    """A token's head of every plane in one run: views [layers, 2, blocks, block_size, HK, ...] of kv's bytes, a 4-bit cache's
    codes and scales apart."""
    if kv.dtype != torch.uint8:
        return [kv]
    layers, two, blocks, bs, hk, width = kv.shape
    flat = kv.view(layers, two, blocks, -1)
    return [flat[..., :bs * hk * 64].view(layers, two, blocks, bs, hk, 64),
            flat[..., bs * hk * 64:].view(layers, two, blocks, bs, hk, 4)]
