"""CPU restatement of the 4-bit KV cache (test infrastructure only; see oracle/__init__.py), in 64 bits.

OCP MXFP4: 32 channels share a scale 2^(b - 127) (255: not a number); a value is a sign and one of GRID times it. A plane is
uint8 [blocks, block_size, HK, 68]; a block's bytes are its codes [block_size][HK][64], then its scales
[block_size][HK][4]; channel 2i is the low nibble of byte i."""

from __future__ import annotations

import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize_group(x) -> tuple[list[int], int]:
    """32 floats as (codes, scale byte), one value at a time."""
    x = [float(v) for v in x]
    if not all(math.isfinite(v) for v in x):
        return [0] * len(x), 255
    amax = max(abs(v) for v in x)
    e = -126
    while amax > 7 * 2.0 ** e and e < 125:  # (6 x 2^125 is the last that bf16 holds)
        e += 1
    codes = []
    for v in x:
        a = min(abs(v) / 2.0 ** e, 6.0)
        off = [abs(a - g) for g in GRID]
        best = [c for c in range(8) if off[c] == min(off)]
        code = next((c for c in best if c % 2 == 0), best[0])
        codes.append(code + (8 if math.copysign(1.0, v) < 0 else 0))
    return codes, e + 127


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [N, HK, 128] as codes uint8 [N, HK, 64] and scales uint8 [N, HK, 4]."""
    n, hk, d = x.shape
    codes, scales = torch.empty(n, hk, d, dtype=torch.uint8), torch.empty(n, hk, d // 32, dtype=torch.uint8)
    groups = x.double().view(n, hk, d // 32, 32).tolist()
    for i in range(n):
        for g in range(hk):
            for j in range(d // 32):
                c, b = quantize_group(groups[i][g][j])
                codes[i, g, 32 * j:32 * j + 32] = torch.tensor(c, dtype=torch.uint8)
                scales[i, g, j] = b
    return codes[..., 0::2] | (codes[..., 1::2] << 4), scales


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes [..., 64] and scales [..., 4] stand for, float64 [..., 128]."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64)
    v = grid[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return v * s.repeat_interleave(32, -1)


def parts(cache: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Copies of a plane's codes [blocks, block_size, HK, 64] and scales [blocks, block_size, HK, 4]."""
    blocks, bs, hk, _ = cache.shape
    flat = cache.reshape(blocks, -1)
    n = bs * hk * 64
    return flat[:, :n].reshape(blocks, bs, hk, 64).clone(), flat[:, n:].reshape(blocks, bs, hk, 4).clone()


def plane(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The plane [blocks, block_size, HK, 68] that holds codes and scales."""
    blocks, bs, hk, _ = codes.shape
    return torch.cat((codes.reshape(blocks, -1), scales.reshape(blocks, -1)), 1).view(blocks, bs, hk, 68)


def cache_values(cache: torch.Tensor) -> torch.Tensor:
    """A plane's values, float64 [blocks, block_size, HK, 128]."""
    return values(*parts(cache))


def store(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots) -> None:
    """In place: rows quantised into their slots, those outside the cache left out."""
    bs = k_cache.shape[1]
    for rows, cache in ((key, k_cache), (value, v_cache)):
        codes, scales = parts(cache)
        c, s = quantize(rows)
        for i, slot in enumerate(torch.as_tensor(slots).tolist()):
            if 0 <= slot < cache.shape[0] * bs:
                codes[slot // bs, slot % bs], scales[slot // bs, slot % bs] = c[i], s[i]
        cache.copy_(plane(codes, scales))
