"""CPU restatement of attention that adds up what every key receives, and of eviction by it (test infrastructure only; see
oracle/__init__.py). float64; written key by key and sequence by sequence."""

from __future__ import annotations

import torch

from oracle.kvpages import head_rows


def attend(q, k, v, scale, counts=None):
    """q [n, H, D], the last n positions of keys k / v [m, HK, D]; counts [m] (bool): keys that take weight. o [n, H, D],
    zeros for a row without keys, the probabilities [H, n, m], and for tolerances the sums of p |v| [n, H, D] and the
    scores' magnitudes sum |q_d k_d| scale [H, n, m]."""
    n, H, m, group = q.shape[0], q.shape[1], k.shape[0], q.shape[1] // k.shape[1]
    q = q.double().transpose(0, 1)
    k, v = (x.double().repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
    seen = torch.arange(m)[None] <= torch.arange(n)[:, None] + (m - n)
    if counts is not None:
        seen = seen & counts[None]
    # (a key that no row counts may hold anything)
    used = seen.any(0)[None, :, None]
    k, v = torch.where(used, k, 0.0), torch.where(used, v, 0.0)
    x = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, float("-inf"))
    p = torch.softmax(x, -1)
    p = torch.where(seen.any(1)[None, :, None], p, 0.0)
    size = q.abs() @ k.abs().transpose(1, 2) * scale
    return (p @ v).transpose(0, 1), p, (p @ v.abs()).transpose(0, 1), size


def add(row, p, new):
    """Adds p [H, n, m] to one sequence's row of weights [HK, width] in place; the last ``new`` tokens start with theirs."""
    hk, m = row.shape[0], p.shape[2]
    got = p.sum(1).view(hk, p.shape[0] // hk, m).sum(1)
    old = max(m - new, 0)
    row[:, :old] += got[:, :old]
    row[:, old:m] = got[:, old:]


def keys_of(cache, table, n):
    """The first n tokens of a sequence [n, HK, D] through its block table, and which lie in blocks of the cache."""
    blocks, bs = cache.shape[:2]
    out, ok = torch.zeros(n, *cache.shape[2:], dtype=cache.dtype), torch.zeros(n, dtype=torch.bool)
    for c in range(-(-n // bs)):
        b, a, e = int(table[c]), c * bs, min(n, (c + 1) * bs)
        if 0 <= b < blocks:
            out[a:e], ok[a:e] = cache[b, :e - a], True
    return out, ok


def kept(w, n, budget, sinks, recent):
    """The tokens (ascending) of n with weights w [>= n] that stay: NaN above every number, of equal ones the earliest."""
    if n <= budget:
        return list(range(n))

    def key(i):
        x = float(w[i])
        return (0, 0.0, i) if x != x else (1, -x, i)

    mid = sorted(range(sinks, n - recent), key=key)[:budget - sinks - recent]
    return sorted([*range(sinks), *mid, *range(n - recent, n)])


def evict(kv, weights, tables, lens, budget, sinks=0, recent=0, rows=None, new_blocks=None):
    """In place on kv [layers, 2, blocks, block_size, HK, width] and weights [layers, rows, HK, width]; the new tables and
    lengths as lists."""
    layers, _, blocks, bs, hk, _ = kv.shape
    reach = len(tables[0]) * bs
    new_tables, new_lens = [], []
    for b, (table, n) in enumerate(zip(tables, lens)):
        n, r = min(max(n, 0), reach), b if rows is None else rows[b]
        drops = n > budget and 0 <= r < weights.shape[1]
        left = budget if drops else n
        into = list(table)
        if drops and new_blocks is not None:
            into = [x if x >= 0 else t for x, t in zip(new_blocks[b], table)]
        used = -(-left // bs)
        new_tables.append(into[:used] + [-1] * (len(table) - used))
        new_lens.append(left)
        if not drops:
            continue
        for layer in range(layers):
            for g in range(hk):
                w = weights[layer, r, g]
                stay = kept(w, n, budget, sinks, recent)
                w[:left] = w[stay].clone()
                for part in head_rows(kv):
                    old = part[layer, :, :, :, g].clone()
                    for j, i in enumerate(stay):
                        src, dst = table[i // bs], into[j // bs]
                        if 0 <= src < blocks and 0 <= dst < blocks:
                            part[layer, :, dst, j % bs, g] = old[:, src, i % bs]
    return new_tables, new_lens
