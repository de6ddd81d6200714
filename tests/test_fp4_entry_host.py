"""Entry points around the 4-bit caches on the CPU: allocation, the module's dispatch, the wrappers (nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from voxcpm2_arabic_dialects_turbo_amd import runner
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
