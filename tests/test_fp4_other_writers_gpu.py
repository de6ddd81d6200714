"""4-bit planes that other programs have written: the store's scales end at 2^125, the format's at 2^127, where codes stand for
more than bf16 holds. Such a value is no number to the attention: it shows in the heads and rows that see it, in its group of
32 channels, and nowhere else; what bf16 holds counts at any scale."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4
from tests._util import randn
from tests.test_fp4_gpu import BS, D, DEV, SCALE, STEP, WIDE, _check, _cu, _gen, _pool, _reach, _varlen
from voxcpm2_arabic_dialects_turbo_amd.ops_fp4 import decode_attention_fp4, load_kvcache_fp4, varlen_attention_fp4

pytestmark = pytest.mark.gpu

# (scale byte, code, whether bf16 holds it): 3 x 2^126, 4 x 2^126, -6 x 2^126, -1.5 x 2^127, 2 x 2^127, -3 x 2^127, 6 x 2^127
CASES = [(253, 5, True), (253, 6, False), (253, 15, False), (254, 11, True), (254, 4, False), (254, 13, False),
         (254, 7, False)]


def _planes(hk, byte, code, seed):
    """Three sequences; the keys of the last kv head are 0 (every probability 1 over the keys it sees, so no sum passes fp32),
    and at position 150 of the second its values of channels 32 to 63 are 0 but for one, channel 41, of that byte and code."""
    gen = _gen(seed)
    lens = [200, 300, 70]
    kc, vc, tables = _pool(gen, lens, hk)
    codes, scales = fp4.parts(kc)
    codes[:, :, hk - 1] = 0
    kc = fp4.plane(codes, scales)
    codes, scales = fp4.parts(vc)
    block, at = int(tables[1, 150 // BS]), 150 % BS
    codes[block, at, hk - 1, 16:32] = 0
    codes[block, at, hk - 1, 16 + 9 // 2] = code << 4
    scales[block, at, hk - 1, 1] = byte
    return gen, lens, kc, fp4.plane(codes, scales), tables, block * BS + at


def _compare(o, want, tol, nan):
    assert torch.equal(o.isnan().cpu(), nan) and not o.isinf().any()
    _check(torch.where(nan, 0.0, o.float().cpu()), torch.where(nan, 0.0, want), tol.nan_to_num(0.0, 0.0))


@WIDE
@pytest.mark.parametrize("hk", [1, 2])
@pytest.mark.parametrize("byte,code,held", CASES)
def test_decode(hk, byte, code, held, wide):
    gen, lens, kc, vc, tables, _ = _planes(hk, byte, code, 10 * byte + code + hk)
    q = randn(gen, 3, 8 * hk, D)
    o = decode_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, device=DEV), _reach(tables, wide), SCALE)
    nan = torch.zeros(o.shape, dtype=torch.bool)
    nan[1, 8 * (hk - 1):, 32:64] = not held
    _compare(o, *_varlen(q, kc, vc, tables, [1, 1, 1], lens), nan)


@pytest.mark.parametrize("hk", [1, 2])
@pytest.mark.parametrize("more", [0, 200])
@pytest.mark.parametrize("byte,code,held", CASES)
def test_varlen(hk, more, byte, code, held):
    gen, lens, kc, vc, tables, _ = _planes(hk, byte, code, 10 * byte + code + hk)
    new = [200, 200, 70] + [2] * more
    lens, tables = lens + [2] * more, torch.cat([tables, tables[:1].expand(more, -1)])
    q = randn(gen, sum(new), 8 * hk, D)
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=200, block_table=tables.to(DEV), softmax_scale=SCALE)
    nan = torch.zeros(o.shape, dtype=torch.bool)
    nan[200 + 50:400, 8 * (hk - 1):, 32:64] = not held  # the second's queries stand at 100 to 299
    _compare(o, *_varlen(q, kc, vc, tables, new, lens), nan)


@pytest.mark.parametrize("hk", [1, 2])
@pytest.mark.parametrize("byte,code,held", CASES)
def test_mixed_steps(hk, byte, code, held):
    """The prompt sees the value from its 51st query on, a decode row over the same blocks sees it, the others do not."""
    gen, lens, kc, vc, tables, _ = _planes(hk, byte, code, 10 * byte + code + hk)
    new, lens = [1, 200, 1] + [1] * 30, lens + [300] + [100 + i for i in range(29)]
    tables = torch.cat([tables, tables[1:2].expand(30, -1)])
    q = randn(gen, sum(new), 8 * hk, D)
    assert 4 * sum(new) <= len(new) * 200
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=200, block_table=tables.to(DEV), softmax_scale=SCALE)
    nan = torch.zeros(o.shape, dtype=torch.bool)
    nan[1 + 50:201, 8 * (hk - 1):, 32:64] = not held
    nan[202, 8 * (hk - 1):, 32:64] = not held
    _compare(o, *_varlen(q, kc, vc, tables, new, lens), nan)


@pytest.mark.parametrize("byte,code,held", CASES)
def test_load(byte, code, held):
    """A value that bf16 does not hold is an infinity of its sign, by bf16's own rounding."""
    _, _, kc, vc, _, slot = _planes(2, byte, code, 5)
    _, v = load_kvcache_fp4(kc.to(DEV), vc.to(DEV), torch.tensor([slot], device=DEV))
    want = fp4.cache_values(vc).view(-1, 2, D)[slot].to(torch.bfloat16)
    assert torch.equal(v[0].cpu(), want) and bool(want.isinf().any()) == (not held)
