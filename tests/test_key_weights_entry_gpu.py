"""Steps that Attention.forward takes with key weights as it does without. Tolerances as in test_key_weights_gpu."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4
from oracle import key_weights as ref
from tests._util import randn
from tests.test_key_weights_gpu import D, DEV, SCALE, Want, _i32
from voxcpm2_arabic_dialects_turbo_amd import ops, runner
from voxcpm2_arabic_dialects_turbo_amd.context import reset_context, set_context
from voxcpm2_arabic_dialects_turbo_amd.layers import Attention

pytestmark = pytest.mark.gpu
H, HK, BS = 16, 2, 256


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float4_e2m1fn_x2])
def test_decode_steps_with_more_rows_than_queries(dtype):
    """Every row goes to its slot, the queries attend and add, two steps."""
    gen = torch.Generator().manual_seed(3)
    layer = Attention(H, D, SCALE, HK)
    runner.allocate_kv_cache([layer], 8, BS, dtype=dtype, device=DEV).zero_()
    runner.allocate_key_weights([layer], 4, 2 * BS, device=DEV)
    tables, lens, rows = [[5, 1], [0, -1], [3, 7]], [260, 9, 255], [2, 0, 3]
    w = torch.full((4, HK, 2 * BS), float("nan"))
    for n, r in zip(lens, rows):
        w[r, :, :n - 1] = torch.rand(HK, n - 1, generator=gen)
    layer.key_weights.copy_(w.to(DEV))
    four_bit = dtype != torch.bfloat16
    caches = [c.cpu() for c in (layer.k_cache, layer.v_cache)]
    try:
        for _ in range(2):
            slots = [tables[b][(n - 1) // BS] * BS + (n - 1) % BS for b, n in enumerate(lens)] + [6 * BS + 3, -1, 2 * BS]
            q, k, v = randn(gen, 3, H, D), randn(gen, 6, HK, D), randn(gen, 6, HK, D)
            set_context(False, slot_mapping=_i32(slots), context_lens=_i32(lens), block_tables=_i32(tables), weight_rows=_i32(rows))
            o = layer(q.to(DEV), k.to(DEV), v.to(DEV))
            if four_bit:
                fp4.store(k, v, *caches, torch.tensor(slots, dtype=torch.int32))
            else:
                for c, x in zip(caches, (k, v)):
                    for i, s in enumerate(slots):
                        if s >= 0:
                            c[s // BS, s % BS] = x[i]
            assert all(torch.equal(a.cpu(), c) for a, c in zip((layer.k_cache, layer.v_cache), caches))
            values = [fp4.cache_values(c) if four_bit else c for c in caches]
            want = Want(w)
            for b, (n, r) in enumerate(zip(lens, rows)):
                keys, vals = (ref.keys_of(c, tables[b], n)[0] for c in values)
                size = (q[b].double().abs().view(HK, -1, D) @ keys.double().abs().permute(1, 2, 0)).max()
                x = SCALE * float(2.0 ** -13 * size + 2.0 ** -18 * q[b].abs().max() * keys.double().abs().sum(-1).max()) if four_bit else 0.0
                want.sequence(q[b:b + 1], keys, vals, None, r, 1, more=2 * x * (1 + 2 * x))
            want.check(o.reshape(3, H, D), layer.key_weights)
            w, lens = layer.key_weights.cpu(), [n + 1 for n in lens]
    finally:
        reset_context()
        ops.forget_plans()
