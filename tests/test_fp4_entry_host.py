"""Entry points around the 4-bit caches on the CPU: allocation, the module's dispatch, the wrappers (nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from voxcpm2_arabic_dialects_turbo_amd import layers, runner
from voxcpm2_arabic_dialects_turbo_amd.context import reset_context, set_context
from voxcpm2_arabic_dialects_turbo_amd.kernels import prefill_attn
from voxcpm2_arabic_dialects_turbo_amd.layers import Attention

BF16, U8, I32 = torch.bfloat16, torch.uint8, torch.int32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, None])
def test_16_bit_caches_need_no_4_bit_type_of_torch(monkeypatch, dtype):
    monkeypatch.delattr(torch, "float4_e2m1fn_x2")
    mods = [Attention(16, 128, 0.1, 2) for _ in range(2)]
    held = torch.get_default_dtype() if dtype is None else dtype
    kv = runner.allocate_kv_cache(mods, 2, 256, dtype=dtype, device="cpu")
    assert kv.shape == (2, 2, 2, 256, 2, 128) and kv.dtype == held
    assert runner.kv_cache_block_bytes(mods, 256, dtype) * 2 == kv.numel() * kv.element_size()
    assert runner.allocate_kv_cache([mods[0], Attention(8, 128, 0.1, 1)], 2, 256, dtype=dtype, device="cpu") is None
    assert mods[0].k_cache.shape == (2, 256, 2, 128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float4_e2m1fn_x2])
def test_decode_steps_with_more_rows_than_queries_store_then_attend(monkeypatch, dtype):
    """Every row goes to its slot and the queries attend, over caches of either kind; with a row per query one call does both."""
    calls = []
    for name in ("decode_attention", "decode_attention_fp4", "store_kvcache", "flash_attn_with_kvcache"):
        def fake(*args, _name=name, **kw):
            calls.append((_name, args, kw))
            return torch.zeros(args[0].shape, dtype=BF16)
        monkeypatch.setattr(layers, name, fake)
    m = Attention(16, 128, 0.1, 2)
    runner.allocate_kv_cache([m], 4, 256, dtype=dtype, device="cpu")
    q = torch.zeros(3, 16, 128, dtype=BF16)
    lens, tables = torch.zeros(3, dtype=I32), torch.zeros(3, 1, dtype=I32)
    try:
        for rows, want in ((5, ["store_kvcache", "flash_attn_with_kvcache"]),
                           (3, ["decode_attention" if dtype == BF16 else "decode_attention_fp4"])):
            calls.clear()
            k, slots = torch.zeros(rows, 2, 128, dtype=BF16), torch.zeros(rows, dtype=I32)
            set_context(False, slot_mapping=slots, context_lens=lens, block_tables=tables)
            assert m(q, k, k).shape == (3, 1, 16, 128)
            assert [c[0] for c in calls] == want
            assert rows == 3 or (calls[0][1][0] is k and calls[0][1][4] is slots and calls[1][1][1] is m.k_cache)
    finally:
        reset_context()


def test_the_paged_prefill_wrapper_takes_4_bit_caches(monkeypatch):
    calls = []
    monkeypatch.setattr(prefill_attn, "varlen_attention_fp4", lambda *args, **kw: calls.append((args, kw)))
    q, cu, bt = torch.zeros(5, 16, 128, dtype=BF16), torch.zeros(3, dtype=I32), torch.zeros(2, 1, dtype=I32)
    kc, vc = (torch.zeros(2, 64, 2, 68, dtype=U8) for _ in range(2))
    o = prefill_attn.paged_prefill_attention(q, kc, vc, bt, cu, cu, 3, 0.1)
    ((args, kw),) = calls
    assert o.shape == (5, 16 * 128) and o.dtype == BF16 and kw["out"].data_ptr() == o.data_ptr()
    assert args[0] is q and args[1] is kc and args[2] is vc and kw["block_table"] is bt and kw["causal"]
    assert kw["max_seqlen_q"] == 3 and kw["softmax_scale"] == 0.1
    with pytest.raises(NotImplementedError, match="4-bit"):
        prefill_attn.paged_prefill_attention(q, kc, vc, bt, cu, cu, 3, 0.1, quant=True)
