"""4-bit caches at the top of bf16's range: finite rows stay finite, and what one head or row sees does not show in others."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4
from tests._util import randn
from tests.test_fp4_gpu import BS, D, DEV, SCALE, _check, _cu, _gen, _plane, _pool, _reach, _varlen, WIDE
from voxcpm2_arabic_dialects_turbo_amd.ops_fp4 import (decode_attention_fp4, load_kvcache_fp4, store_kvcache_fp4,
                                                       varlen_attention_fp4)

pytestmark = pytest.mark.gpu


def test_finite_rows_load_finite():
    """Every bf16 value of the highest two binades as a group's largest: held as the oracle says, in magnitude at most 6 x
    2^125, and at most a quarter of the value off."""
    top = torch.arange(0x7e80, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    rows = randn(_gen(1), top.numel(), 2, D) * (torch.finfo(torch.bfloat16).max / 8)
    rows[:, 0, 5::32], rows[:, 1, ::32] = top[:, None], -top[:, None]
    assert rows.isfinite().all()
    kc = torch.zeros(4, 64, 2, 68, dtype=torch.uint8)
    vc = kc.clone()
    kd, vd = kc.to(DEV), vc.to(DEV)
    slots = torch.arange(256, dtype=torch.int32)
    store_kvcache_fp4(rows.to(DEV), rows.flip(0).contiguous().to(DEV), kd, vd, slots.to(DEV))
    fp4.store(rows, rows.flip(0), kc, vc, slots)
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)
    k, v = (x.double().cpu() for x in load_kvcache_fp4(kd, vd, slots.to(DEV)))
    assert k.isfinite().all() and v.isfinite().all() and k.abs().max() == 6 * 2.0 ** 125
    assert torch.equal(k, fp4.cache_values(kc).view(256, 2, D)) and torch.equal(v, fp4.cache_values(vc).view(256, 2, D))
    held, want = k[:, 0, 5::32], top.double()[:, None]
    assert ((held - want).abs() <= want / 4).all()


def _large_value(hk, seed):
    """Three sequences whose keys are 0 in the last kv head (so every probability is 1 over the keys it sees, and no sum passes
    fp32) and whose values there hold one row of bf16's largest, at position 150 of the second."""
    gen = _gen(seed)
    lens = [200, 300, 70]
    kc, vc, tables = _pool(gen, lens, hk)
    codes, scales = fp4.parts(kc)
    codes[:, :, hk - 1] = 0
    kc = fp4.plane(codes, scales)
    row = torch.full((1, hk, D), 0.5, dtype=torch.bfloat16)
    row[:, hk - 1, 32:64] = torch.finfo(torch.bfloat16).max
    slot = int(tables[1, 150 // BS]) * BS + 150 % BS
    kd, vd = kc.to(DEV), vc.to(DEV)
    zero = torch.zeros_like(row)
    store_kvcache_fp4(zero.to(DEV), row.to(DEV), kd, vd, torch.tensor([slot], device=DEV))
    fp4.store(zero, row, kc, vc, [slot])
    assert torch.equal(vd.cpu(), vc)
    return gen, lens, kc, vc, tables, kd, vd


@WIDE
@pytest.mark.parametrize("hk", [1, 2])
def test_decode_over_the_largest_values(hk, wide):
    gen, lens, kc, vc, tables, kd, vd = _large_value(hk, 10 + hk)
    q = randn(gen, 3, 8 * hk, D)
    o = decode_attention_fp4(q.to(DEV), kd, vd, torch.tensor(lens, device=DEV), _reach(tables, wide), SCALE)
    assert o.isfinite().all()
    _check(o, *_varlen(q, kc, vc, tables, [1, 1, 1], lens))


@pytest.mark.parametrize("hk", [1, 2])
@pytest.mark.parametrize("more", [0, 200])
def test_varlen_over_the_largest_values(hk, more):
    """Rows that see the value and rows before it, in launches of few and of many workgroups."""
    gen, lens, kc, vc, tables, kd, vd = _large_value(hk, 20 + hk)
    new = [200, 200, 70] + [2] * more
    lens, tables = lens + [2] * more, torch.cat([tables, tables[:1].expand(more, -1)])
    q = randn(gen, sum(new), 8 * hk, D)
    o = varlen_attention_fp4(q.to(DEV), kd, vd, cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens), max_seqlen_q=200,
                             block_table=tables.to(DEV), softmax_scale=SCALE)
    assert o.isfinite().all()
    _check(o, *_varlen(q, kc, vc, tables, new, lens))
