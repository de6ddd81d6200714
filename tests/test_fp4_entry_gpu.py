"""Entry points around the 4-bit caches on the GPU."""

from __future__ import annotations

import pytest
import torch

from tests._util import randn
from tests.test_fp4_gpu import D, DEV, SCALE, _check, _cu, _gen, _pool, _varlen
from voxcpm2_arabic_dialects_turbo_amd.kernels.prefill_attn import paged_prefill_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,lens", [([5, 63, 0, 17], [300, 63, 40, 512]), ([1] * 30 + [60], [40 + 7 * i for i in range(31)])])
def test_paged_prefill_over_4_bit_caches(new, lens):
    """The wrapper's layouts: strided query rows in, [T, H * D] out; prefills over prefixes and a step of mostly decode rows."""
    gen = _gen(sum(new))
    kc, vc, tables = _pool(gen, lens, 2)
    rows = randn(gen, sum(new), 20 * D)
    q = rows[:, :16 * D].view(-1, 16, D)
    o = paged_prefill_attention(rows.to(DEV)[:, :16 * D].view(-1, 16, D), kc.to(DEV), vc.to(DEV), tables.to(DEV), _cu(new),
                                _cu(lens), max(new), SCALE)
    assert o.shape == (sum(new), 16 * D)
    _check(o.view(-1, 16, D), *_varlen(q, kc, vc, tables, new, lens))
