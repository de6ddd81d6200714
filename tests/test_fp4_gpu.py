"""GPU parity of the 4-bit KV cache operators against the oracle in 64 bits.

The store and the load are exact. The attention is over the values the cache holds, which the oracle takes as they are, so
what an output may be off by is what the kernels round: the output (half a step of bf16, 2^-8 of the value), every
probability (the same, so 2^-8 of the attention over |V|), and the scores: the scaled MFMA's sum is off by at most 2^-13
of sum |q||k| (measured: 2^-13.4 at worst over operands whose scales spread over 2^12), which an exponential turns into
that many parts of the probability, in the sum of a row and in its norm."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as ref
from oracle import fp4
from tests._util import paged_pool, randn
from voxcpm2_arabic_dialects_turbo_amd import ops, runner
from voxcpm2_arabic_dialects_turbo_amd.context import reset_context
from voxcpm2_arabic_dialects_turbo_amd.kernels import kv_pages
from voxcpm2_arabic_dialects_turbo_amd.layers import Attention
from voxcpm2_arabic_dialects_turbo_amd.ops_fp4 import (decode_attention_fp4, fp4_parts, load_kvcache_fp4,
                                                       store_kvcache_fp4, varlen_attention_fp4)

pytestmark = pytest.mark.gpu
DEV = "cuda"
D, BS = 128, 256
SCALE = D ** -0.5
STEP = torch.finfo(torch.bfloat16).eps / 2


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _plane(gen, blocks, bs, hk):
    """A plane of random codes whose scales lie around 2^0 (values of normal size), on the CPU."""
    codes = torch.randint(0, 256, (blocks, bs, hk, 64), generator=gen, dtype=torch.uint8)
    return fp4.plane(codes, torch.randint(123, 128, (blocks, bs, hk, 4), generator=gen, dtype=torch.uint8))


def _pool(gen, lens, hk, bs=BS, spare=2, extra_cols=0):
    need = sum(-(-n // bs) for n in lens)
    _, _, tables = paged_pool(gen, lens, need + spare, bs, 1, 1, extra_cols)
    return _plane(gen, need + spare, bs, hk), _plane(gen, need + spare, bs, hk), tables


def _attend(q, k, v, causal, scale):
    """One sequence in 64 bits: the output [n, H, 128] and how far a kernel may be off it."""
    o = ref.attend(q.double(), k, v, causal, scale).view(q.shape)
    size = ref.attend(q.double(), k, v.abs(), causal, scale).view(q.shape)
    group = q.shape[1] // k.shape[1]
    s = torch.einsum("qhd,khd->hqk", q.double().abs(), k.abs().repeat_interleave(group, 1)).amax(-1)  # [H, n]
    off = (2.0 ** -13 * abs(scale) * s).transpose(0, 1)[..., None]
    return o, STEP * o.abs() + (STEP + 2 * off + 2.0 ** -14) * size


def _check(out, want, tol, what=""):
    out = out.double().cpu()
    bad = ~((out - want).abs() <= tol + 1e-30)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst " \
                          f"{float(((out - want).abs() / tol.clamp_min(1e-30)).max()):.3g} of the tolerance"


def _varlen(q, kc, vc, tables, new, lens, causal=True, scale=SCALE):
    kv, vv = fp4.cache_values(kc), fp4.cache_values(vc)
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        first = max(0, n - m) if causal else (n if m == 0 else 0)  # queries before every key see none
        if n > first:
            k, v = (ref.gather_pages(c, tables[b], m) for c in (kv, vv))
            out[at + first:at + n], tol[at + first:at + n] = _attend(q[at + first:at + n], k, v, causal, scale)
        at += n
    return out, tol


def _cu(lens):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32).to(DEV)


# ---------------------------------------------------------------------------------------------------------------------
# store and load


@pytest.mark.parametrize("hk", [1, 2, 3])
@pytest.mark.parametrize("bs", [64, 256])
def test_store_and_load_are_the_oracles(hk, bs):
    gen = _gen(10 * hk + bs)
    n, blocks = 23, 3
    rows = (randn(gen, n, 3 * hk * D).float() * torch.exp2(torch.randint(-20, 20, (n, 1), generator=gen).float()))
    rows = rows.to(torch.bfloat16)
    rows[3] = 0.0
    rows[4, ::2] = -0.0
    k, v = rows[:, :hk * D].view(n, hk, D), rows[:, hk * D:2 * hk * D].view(n, hk, D)
    slots = torch.randperm(blocks * bs, generator=gen)[:n].to(torch.int32)
    slots[5], slots[6], slots[7] = -1, blocks * bs, 2 ** 31 - 1
    kc, vc = _plane(gen, blocks, bs, hk), _plane(gen, blocks, bs, hk)
    kd, vd, rd = kc.to(DEV), vc.to(DEV), rows.to(DEV)
    store_kvcache_fp4(rd[:, :hk * D].view(n, hk, D), rd[:, hk * D:2 * hk * D].view(n, hk, D), kd, vd, slots.to(DEV))
    fp4.store(k, v, kc, vc, slots)
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)  # stored slots, and every other byte as it was
    for got, part in zip(fp4_parts(kd), fp4.parts(kc)):
        assert torch.equal(got.cpu(), part)
    at = torch.cat((slots, slots[:3], torch.tensor([0, 0, -5], dtype=torch.int32)))
    lk, lv = load_kvcache_fp4(kd, vd, at.to(DEV).long())
    for got, cache in ((lk, kc), (lv, vc)):
        flat = fp4.cache_values(cache).view(-1, hk, D)
        ok = (at >= 0) & (at < blocks * bs)
        want = torch.where(ok[:, None, None], flat[at.clamp(0, blocks * bs - 1).long()], 0.0)
        assert torch.equal(got.double().cpu(), want)


def test_store_of_every_bf16_value_and_tie():
    """Each finite bf16 value as a group's largest, beside values on every tie of the grid."""
    top = torch.arange(0, 0x7f80, 37, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    n = top.numel()
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.125, -0.25, -0.75, -1.25, -5.0, 0.2490234375, 5.03125])
    rows = torch.zeros(n, 1, D, dtype=torch.bfloat16)
    rows[:, 0, 0::32] = top[:, None]
    exp = torch.frexp(top.float())[1]
    for i, t in enumerate(ties.tolist()):
        for g in range(4):
            rows[:, 0, 32 * g + 1 + i] = torch.ldexp(torch.full((n,), t), exp - 2 - (g % 3)).to(torch.bfloat16)
    blocks = -(-n // 64)
    kc = torch.zeros(blocks, 64, 1, 68, dtype=torch.uint8)
    kd, vd = kc.to(DEV), kc.to(DEV)
    slots = torch.arange(n, dtype=torch.int32)
    store_kvcache_fp4(rows.to(DEV), rows.flip(0).contiguous().to(DEV), kd, vd, slots.to(DEV))
    vc = kc.clone()
    fp4.store(rows, rows.flip(0), kc, vc, slots)
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)


def test_store_of_infinities_and_nans_marks_their_groups():
    rows = randn(_gen(3), 4, 2, D)
    rows[0, 0, 5], rows[1, 1, 40], rows[2, 0, 127], rows[2, 0, 0] = float("inf"), float("nan"), -float("inf"), 3e38
    kd = torch.zeros(1, 64, 2, 68, dtype=torch.uint8, device=DEV)
    vd = kd.clone()
    slots = torch.tensor([9, 3, 60, 0], dtype=torch.int32, device=DEV)
    store_kvcache_fp4(rows.to(DEV), rows.to(DEV), kd, vd, slots)
    k, v = load_kvcache_fp4(kd, vd, slots)
    want = ~rows.isfinite().view(4, 2, 4, 32).all(-1)
    assert torch.equal(k.isnan().view(4, 2, 4, 32).all(-1).cpu(), want) and torch.equal(v.isnan().cpu(), k.isnan().cpu())
    assert torch.equal(k.isnan().view(4, 2, 4, 32).any(-1).cpu(), want)


@pytest.mark.parametrize("offset", [1, 3])
def test_store_of_unaligned_rows(offset):
    gen = _gen(offset)
    x = randn(gen, 300 * 517 + 8).to(DEV)
    k = x[offset:offset + 300 * 517].view(300, 517)[:, :256].view(300, 2, D)
    v = x[offset:offset + 300 * 517].view(300, 517)[:, 260:516].view(300, 2, D)
    a = [torch.zeros(2, 256, 2, 68, dtype=torch.uint8, device=DEV) for _ in range(4)]
    slots = torch.randperm(512, generator=gen)[:300].to(torch.int32).to(DEV)
    store_kvcache_fp4(k, v, a[0], a[1], slots)
    store_kvcache_fp4(k.contiguous(), v.contiguous(), a[2], a[3], slots)
    assert torch.equal(a[0], a[2]) and torch.equal(a[1], a[3])


def test_store_of_one_row_for_every_token_and_of_none():
    row = randn(_gen(4), 1, 2, D).to(DEV)
    caches = [torch.zeros(1, 64, 2, 68, dtype=torch.uint8, device=DEV) for _ in range(2)]
    slots = torch.arange(5, dtype=torch.int32, device=DEV)
    store_kvcache_fp4(row.expand(5, 2, D), row.expand(5, 2, D), *caches, slots)
    k, _ = load_kvcache_fp4(*caches, slots)
    assert (k == k[:1]).all() and k.abs().sum() > 0
    store_kvcache_fp4(row[:0], row[:0], *caches, slots[:0])
    assert load_kvcache_fp4(*caches, slots[:0])[0].shape == (0, 2, D)


def test_ids_past_int32_name_nothing():
    """64-bit slots and block ids that int32 does not hold lie outside the cache, not where their low half points."""
    gen = _gen(6)
    kc, vc, tables = _pool(gen, [100, 100], 2)
    row = randn(gen, 2, 2, D).to(DEV)
    kd, vd = kc.to(DEV), vc.to(DEV)
    store_kvcache_fp4(row, row, kd, vd, torch.tensor([2 ** 32 + 3, -2 ** 33], device=DEV))
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)
    assert not load_kvcache_fp4(kd, vd, torch.tensor([2 ** 32], device=DEV))[0].any()
    wide = tables.long()
    wide[1] += 2 ** 32
    q = randn(gen, 2, 16, D)
    o = decode_attention_fp4(q.to(DEV), kd, vd, torch.tensor([100, 100], device=DEV), wide.to(DEV), SCALE)
    assert (o[1] == 0).all()
    want, tol = _varlen(q, kc, vc, tables, [1, 1], [100, 100])
    _check(o[:1], want[:1], tol[:1])


# ---------------------------------------------------------------------------------------------------------------------
# decode


def _reach(tables, wide, bs=BS):
    """Tables on the GPU; wide: with columns behind them, so that they reach more than 8192 16-token steps, from where the
    decode kernels have eight waves a workgroup instead of four."""
    if wide:
        cols = 8192 * 16 // (bs * len(tables)) + 1
        tables = torch.nn.functional.pad(tables, (0, max(0, cols - tables.shape[1])), value=-1)
    return tables.to(DEV)


WIDE = pytest.mark.parametrize("wide", [False, True])


@WIDE
@pytest.mark.parametrize("heads,hk", [(16, 2), (8, 1), (16, 1), (1, 1), (2, 2), (6, 2), (5, 1)])
@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [17, 0, 300], [15, 16, 31, 32, 33, 63, 64, 65, 255, 256, 257, 512, 0, 1]])
def test_decode_matches_the_oracle(heads, hk, lens, wide):
    gen = _gen(heads * 100 + hk + len(lens))
    kc, vc, tables = _pool(gen, lens, hk, extra_cols=1)
    q = randn(gen, len(lens), heads, D)
    o = decode_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                             _reach(tables, wide), SCALE)
    _check(o, *_varlen(q, kc, vc, tables, [1] * len(lens), lens))


@WIDE
@pytest.mark.parametrize("bs", [64, 128, 192, 512])
@pytest.mark.parametrize("batch,hi", [(3, 5000), (70, 700), (260, 90)])
def test_decode_over_block_sizes_and_batches(bs, batch, hi, wide):
    gen = _gen(bs + batch)
    lens = torch.randint(1, hi, (batch,), generator=gen).tolist()
    kc, vc, tables = _pool(gen, lens, 2, bs)
    q = randn(gen, batch, 16, D)
    o = decode_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, device=DEV),
                             _reach(tables, wide, bs), 0.05)
    _check(o, *_varlen(q, kc, vc, tables, [1] * batch, lens, scale=0.05))


def test_decode_of_more_sequences_than_a_launch_and_wide_tables():
    gen = _gen(7)
    lens = torch.randint(0, 150, (700,), generator=gen).tolist()
    kc, vc, tables = _pool(gen, lens, 1, 64, extra_cols=9)
    q = randn(gen, 700, 8, D)
    o = decode_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, device=DEV), tables.to(DEV), SCALE)
    _check(o, *_varlen(q, kc, vc, tables, [1] * 700, lens))


@WIDE
def test_decode_is_the_same_twice_and_with_any_workgroups(wide):
    gen = _gen(8)
    lens = [3000, 40, 700, 1, 0, 2222]
    kc, vc, tables = _pool(gen, lens, 2)
    q = randn(gen, len(lens), 16, D)
    args = (q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, device=DEV), _reach(tables, wide), SCALE)
    a = decode_attention_fp4(*args)
    assert torch.equal(a, decode_attention_fp4(*args))
    for plan in ("a", "a", "b", "a"):  # recorded, read back, recorded, recorded
        assert torch.equal(a, decode_attention_fp4(*args, plan=plan))
    want = _varlen(q, kc, vc, tables, [1] * len(lens), lens)
    from voxcpm2_arabic_dialects_turbo_amd import _lib
    try:
        for wgs in (1, 7, 300):
            _lib.load().vox_set_decode_workgroups(wgs)
            _check(decode_attention_fp4(*args), *want, f"{wgs} workgroups")
    finally:
        _lib.load().vox_set_decode_workgroups(0)


@WIDE
def test_decode_with_rising_scores_and_large_scales(wide):
    """Scores that rise along the context (the running maximum moves all the time), and values far from 1."""
    gen = _gen(9)
    lens = [900, 333]
    kc, vc, tables = _pool(gen, lens, 2)
    codes, scales = fp4.parts(kc)
    for b, n in enumerate(lens):
        for j in range(n):
            codes[tables[b, j // BS], j % BS] = 0x22  # every channel 1
            scales[tables[b, j // BS], j % BS] = 118 + (12 * j) // n
    kc = fp4.plane(codes, scales)
    vcodes, vscales = fp4.parts(vc)
    vc = fp4.plane(vcodes, vscales + 80)  # 2^80
    q = randn(gen, 2, 16, D).abs()
    o = decode_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, device=DEV),
                             _reach(tables, wide), SCALE)
    _check(o, *_varlen(q, kc, vc, tables, [1, 1], lens))


@WIDE
def test_decode_masks_unmapped_blocks_and_what_lies_behind_the_context(wide):
    """A block outside the cache has no weight; scales that are not numbers behind the context do not show."""
    gen = _gen(11)
    lens = [700, 500, 600]
    kc, vc, tables = _pool(gen, lens, 2)
    for cache in (kc, vc):
        codes, scales = fp4.parts(cache)
        for b, n in enumerate(lens):
            if n % BS:
                scales[tables[b, n // BS], n % BS:] = 255
        cache.copy_(fp4.plane(codes, scales))
    bad = tables.clone()
    bad[0, 1], bad[1, 0], bad[2] = -1, 10 ** 6, -1
    q = randn(gen, 3, 16, D)
    o = decode_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, device=DEV), _reach(bad, wide), SCALE)
    kv, vv = fp4.cache_values(kc), fp4.cache_values(vc)
    for b, keep in ((0, [*range(256), *range(512, 700)]), (1, [*range(256, 500)])):
        k, v = (ref.gather_pages(c, tables[b], lens[b])[keep] for c in (kv, vv))
        want, tol = _attend(q[b:b + 1], k, v, True, SCALE)
        _check(o[b:b + 1], want, tol, f"sequence {b}")
    assert (o[2] == 0).all()


@WIDE
@pytest.mark.parametrize("hk", [1, 2])
def test_decode_with_values_that_are_not_numbers(hk, wide):
    """A NaN group of a value row shows in its kv head's heads and its channels alone; one of a key row in its kv head's
    heads; a NaN query head in itself."""
    gen = _gen(12)
    lens, heads = [300, 300, 300, 300], 8 * hk
    kc, vc, tables = _pool(gen, lens, hk)
    codes, scales = fp4.parts(vc)
    scales[tables[0, 1], 7, hk - 1, 2] = 255
    vc = fp4.plane(codes, scales)
    codes, scales = fp4.parts(kc)
    scales[tables[1, 0], 200, 0, 1] = 255
    kc = fp4.plane(codes, scales)
    q = randn(gen, 4, heads, D)
    q[2, 3, 77] = float("nan")
    q[3, 1, 0] = float("inf")
    o = decode_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(lens, device=DEV),
                             _reach(tables, wide), SCALE).cpu()
    want = torch.zeros(4, heads, D, dtype=torch.bool)
    want[0, 8 * (hk - 1):, 64:96] = True
    want[1, :8] = True
    want[2, 3] = True
    want[3, 1] = True
    assert torch.equal(o.isnan(), want)


@WIDE
@pytest.mark.parametrize("batch,hk", [(1, 2), (37, 2), (37, 1), (600, 2)])
def test_decode_that_stores_is_store_then_decode(batch, hk, wide):
    gen = _gen(20 + batch + hk)
    lens = torch.randint(1, 600, (batch,), generator=gen).tolist()
    if batch > 3:
        lens[3] = 0  # a padded row: its slot is -1
    kc, vc, tables = _pool(gen, lens, hk)
    rows = randn(gen, batch, (8 * hk + 2 * hk) * D).to(DEV)
    q = rows[:, :8 * hk * D].view(batch, 8 * hk, D)
    k, v = (rows[:, (8 + i) * hk * D:(9 + i) * hk * D].view(batch, hk, D) for i in (0, 1))
    slots = torch.tensor([ref.slot_of(tables[b], n - 1, BS) if n else -1 for b, n in enumerate(lens)], dtype=torch.int32)
    a, b = (kc.to(DEV), vc.to(DEV)), (kc.to(DEV), vc.to(DEV))
    args = (torch.tensor(lens, dtype=torch.int32, device=DEV), _reach(tables, wide), SCALE)
    o = decode_attention_fp4(q, *a, *args, key=k, value=v, slot_mapping=slots.to(DEV))
    store_kvcache_fp4(k, v, *b, slots.to(DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    _check(o, *_decode_ref(q.cpu(), b[0].cpu(), b[1].cpu(), tables, lens))


def _decode_ref(q, kc, vc, tables, lens):
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    kv, vv = fp4.cache_values(kc), fp4.cache_values(vc)
    for b, n in enumerate(lens):
        if n:
            out[b:b + 1], tol[b:b + 1] = _attend(q[b:b + 1], *(ref.gather_pages(c, tables[b], n) for c in (kv, vv)), True,
                                                 SCALE)
    return out, tol


def test_decode_past_32_bit_offsets():
    """A cache of over 4 GiB a plane: blocks at its end."""
    blocks, hk = 130_000, 2
    if torch.cuda.mem_get_info()[0] < 4 * blocks * BS * hk * 68:
        pytest.skip("not enough GPU memory")
    kd = torch.zeros(blocks, BS, hk, 68, dtype=torch.uint8, device=DEV)
    vd = torch.zeros(blocks, BS, hk, 68, dtype=torch.uint8, device=DEV)
    gen = _gen(13)
    n = 400
    rows = randn(gen, n, 2, D).to(DEV)
    table = torch.tensor([[blocks - 1, blocks - 7]], dtype=torch.int32, device=DEV)
    slots = torch.cat((torch.arange(BS) + (blocks - 1) * BS, torch.arange(n - BS) + (blocks - 7) * BS)).to(torch.int32)
    store_kvcache_fp4(rows, rows, kd, vd, slots.to(DEV))
    k, v = load_kvcache_fp4(kd, vd, slots.to(DEV))
    c, s = fp4.quantize(rows.cpu())
    want = fp4.values(c, s)
    assert torch.equal(k.double().cpu(), want) and torch.equal(v.double().cpu(), want)
    q = randn(gen, 20, 16, D)
    o = decode_attention_fp4(q[:1].to(DEV), kd, vd, torch.tensor([n], device=DEV), table, SCALE)
    _check(o, *_attend(q[:1], want, want, True, SCALE))
    o = varlen_attention_fp4(q.to(DEV), kd, vd, cu_seqlens_q=_cu([20]), cu_seqlens_k=_cu([n]), max_seqlen_q=20,
                             block_table=table, softmax_scale=SCALE)
    _check(o, *_attend(q, want, want, True, SCALE))


# ---------------------------------------------------------------------------------------------------------------------
# varlen


@pytest.mark.parametrize("heads,hk", [(16, 2), (8, 1), (16, 1), (3, 3), (32, 8), (128, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_varlen_matches_the_oracle(heads, hk, causal):
    gen = _gen(heads + hk)
    new, lens = [1, 5, 63, 130, 0, 17, 64], [1, 300, 63, 260, 40, 512, 65]
    kc, vc, tables = _pool(gen, lens, hk)
    q = randn(gen, sum(new), heads, D)
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=max(new), block_table=tables.to(DEV), softmax_scale=SCALE, causal=causal)
    _check(o, *_varlen(q, kc, vc, tables, new, lens, causal))


@pytest.mark.parametrize("bs", [64, 192, 1024])
def test_varlen_over_block_sizes_and_strided_rows(bs):
    gen = _gen(bs)
    new, lens = [200, 33, 1, 90], [1500, 33, 700, 95]
    kc, vc, tables = _pool(gen, lens, 2, bs, extra_cols=2)
    rows = randn(gen, sum(new), 20 * D)
    q = rows[:, :16 * D].view(-1, 16, D)
    out = torch.full((sum(new) + 3, 24, D), 7.0, dtype=torch.bfloat16, device=DEV)
    o = varlen_attention_fp4(rows.to(DEV)[:, :16 * D].view(-1, 16, D), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new),
                             cu_seqlens_k=_cu(lens), max_seqlen_q=200, block_table=tables.to(DEV), softmax_scale=SCALE,
                             out=out[:sum(new), :16])
    _check(o, *_varlen(q, kc, vc, tables, new, lens))
    assert (out[sum(new):] == 7).all() and (out[:, 16:] == 7).all()  # nothing but its rows


def test_varlen_queries_that_see_no_key():
    gen = _gen(31)
    new, lens = [70, 9, 40], [20, 0, 40]
    kc, vc, tables = _pool(gen, lens, 2)
    q = randn(gen, sum(new), 16, D)
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=70, block_table=tables.to(DEV), softmax_scale=SCALE)
    want, tol = _varlen(q, kc, vc, tables, new, lens)
    assert (want[:50] == 0).all() and (want[70:79] == 0).all()
    _check(o, want, tol)


def test_varlen_of_mixed_steps_takes_the_decode_kernels():
    gen = _gen(32)
    new, lens = [1] * 40 + [150, 2] + [1] * 20, torch.randint(1, 900, (62,), generator=gen).tolist()
    lens[40], lens[41], lens[5], lens[50] = 400, 3, 0, 1
    kc, vc, tables = _pool(gen, lens, 2)
    q = randn(gen, sum(new), 16, D)
    want = _varlen(q, kc, vc, tables, new, lens)
    args = dict(cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens), max_seqlen_q=150, block_table=tables.to(DEV),
                softmax_scale=SCALE)
    assert 4 * sum(new) <= len(new) * 150
    _check(varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), **args), *want)
    for plan in ("a", "a", "b"):  # recorded, read back, recorded
        _check(varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), plan=plan, **args), *want)
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu([1] * 62), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=1, block_table=tables.to(DEV), softmax_scale=SCALE)[:62]
    _check(o, *_decode_ref(q[:62], kc, vc, tables, lens))


@pytest.mark.parametrize("heads,hk", [(16, 2), (8, 1), (16, 1), (2, 1)])
@pytest.mark.parametrize("prompts,decodes,hi", [(1, 10, 90), (2, 70, 300), (7, 200, 600), (4, 250, 330), (3, 300, 200)])
@pytest.mark.parametrize("causal", [True, False])
def test_varlen_of_prompts_between_decode_rows(heads, hk, prompts, decodes, hi, causal):
    """One launch for both kinds of rows (two past 256 sequences), few prompts and many: rows without a key, sequences
    without a query, blocks that are none, and rows behind the last sequence, which stay as they were."""
    gen = _gen(heads + decodes + hi)
    n = prompts + decodes
    new, lens = [1] * n, torch.randint(1, 500, (n,), generator=gen).tolist()
    at = torch.randperm(n, generator=gen)[:prompts].tolist()
    for i, b in enumerate(at):
        new[b] = hi - 13 * i
        lens[b] = new[b] + (0, 50, 700)[i % 3]
    one = [b for b in range(n) if new[b] == 1]
    lens[one[0]], new[one[1]] = 0, 0
    kc, vc, tables = _pool(gen, lens, hk, 64)
    bad = tables.clone()
    bad[one[2], 0] = -1
    lens[one[2]] = 60  # its only block is none
    q = randn(gen, sum(new) + 5, heads, D)
    want, tol = _varlen(q[:sum(new)], kc, vc, tables, new, lens, causal)
    row = sum(new[:one[2]])
    want[row] = tol[row] = 0.0
    out = torch.full((sum(new) + 5, heads, D), 7.0, dtype=torch.bfloat16, device=DEV)
    assert 4 * len(q) <= n * hi  # the call is mostly decode rows
    key = (heads, hk, n, hi, causal)
    for plan in (None, key, key):
        out.fill_(7.0)
        varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=hi, block_table=bad.to(DEV), softmax_scale=SCALE, causal=causal, out=out, plan=plan)
        _check(out[:sum(new)], want, tol)
        assert (out[sum(new):] == 7).all()


def test_varlen_masks_unmapped_blocks_and_values_that_are_not_numbers():
    """NaN groups show in the rows that see them, in their channels; not in rows before them, nor behind the sequence."""
    gen = _gen(33)
    new, lens = [100, 60], [300, 190]
    kc, vc, tables = _pool(gen, lens, 2)
    codes, scales = fp4.parts(vc)
    scales[tables[0, 1], 300 - 256:] = 255       # behind the sequence
    scales[tables[1, 0], 160, 1, 3] = 255        # position 160 of the second: its queries are 130 to 189
    vc = fp4.plane(codes, scales)
    codes, scales = fp4.parts(kc)
    scales[tables[0, 1], 300 - 256:] = 255
    kc = fp4.plane(codes, scales)
    bad = tables.clone()
    bad[0, 0] = -1
    q = randn(gen, 160, 16, D)
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=100, block_table=bad.to(DEV), softmax_scale=SCALE).cpu()
    nan = torch.zeros(160, 16, D, dtype=torch.bool)
    nan[100 + 30:, 8:, 96:] = True
    assert torch.equal(o.isnan(), nan)
    kv, vv = fp4.cache_values(kc), fp4.cache_values(vc)
    k, v = (ref.gather_pages(c, tables[0], 300)[256:] for c in (kv, vv))  # queries 200 to 299, keys 256 to 299
    assert (o[:56] == 0).all()
    _check(o[56:100], *_attend(q[56:100], k, v, True, SCALE))
    k, v = (ref.gather_pages(c, tables[1], 190) for c in (kv, vv.nan_to_num(0.0)))
    want, tol = _attend(q[100:], k, v, True, SCALE)
    _check(torch.where(nan[100:], want.to(torch.bfloat16), o[100:]), want, tol + STEP * nan[100:])


@pytest.mark.parametrize("heads,hk", [(16, 2), (3, 3), (64, 1), (128, 1)])
@pytest.mark.parametrize("more", [0, 200])
def test_varlen_of_few_and_many_workgroups(heads, hk, more):
    """The same sequences alone and among so many others that a launch takes the variant for full chips: masks, blocks that
    are none, values that are not numbers and rows without a key in both."""
    gen = _gen(1000 + heads + more)
    new, lens = [70, 37, 9, 100, 33], [200, 300, 4, 100, 0]
    new, lens = new + [2] * more, lens + [2 + i for i in range(more)]
    kc, vc, tables = _pool(gen, lens, hk, 64)
    codes, scales = fp4.parts(vc)
    scales[tables[0, 3], 0, hk - 1, 1] = 255  # position 192 of the first: its queries are 130 to 199
    vc = fp4.plane(codes, scales)
    bad = tables.clone()
    bad[1, 1], bad[3, 1] = kc.shape[0], -5
    q = randn(gen, sum(new), heads, D)
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=100, block_table=bad.to(DEV), softmax_scale=SCALE).cpu()
    nan = torch.zeros(sum(new), heads, D, dtype=torch.bool)
    nan[62:70, heads - heads // hk:, 32:64] = True
    assert torch.equal(o.isnan(), nan)
    kv, vv = fp4.cache_values(kc), fp4.cache_values(vc).nan_to_num(0.0)
    want, tol = _varlen(q, kc, fp4.plane(codes, torch.where(scales == 255, 0, scales)), tables, new, lens)
    # the second's keys without 64 to 127 (its queries 263 to 299 see all others before them), the fourth's first 64 only
    k, v = (torch.cat([ref.gather_pages(c, tables[1], 300)[:64], ref.gather_pages(c, tables[1], 300)[128:]])
            for c in (kv, vv))
    want[70:107], tol[70:107] = _attend(q[70:107], k, v, True, SCALE)
    k, v = (ref.gather_pages(c, tables[3], 64) for c in (kv, vv))
    want[116:180], tol[116:180] = _attend(q[116:180], k, v, True, SCALE)
    want[180:216], tol[180:216] = _attend(q[180:216], k, v, False, SCALE)
    _check(torch.where(nan, want.to(torch.bfloat16), o), want, tol + STEP * nan * want.abs())


@pytest.mark.parametrize("more", [0, 200])
def test_varlen_of_queries_that_are_not_numbers(more):
    gen = _gen(35 + more)
    new, lens = [40, 30] + [2] * more, [200, 70] + [5] * more
    kc, vc, tables = _pool(gen, lens, 2)
    q = randn(gen, sum(new), 16, D)
    want, tol = _varlen(q, kc, vc, tables, new, lens)
    q[3, 2, 5], q[45, 15, 127] = float("nan"), float("-inf")
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=40, block_table=tables.to(DEV), softmax_scale=SCALE).cpu()
    nan = torch.zeros(o.shape, dtype=torch.bool)
    nan[3, 2], nan[45, 15] = True, True
    assert torch.equal(o.isnan(), nan)
    _check(torch.where(nan, want.to(torch.bfloat16), o), want, tol + STEP * nan * want.abs())


def test_varlen_of_long_contexts():
    gen = _gen(34)
    new, lens = [40, 300], [9000, 4097]
    kc, vc, tables = _pool(gen, lens, 2)
    q = randn(gen, sum(new), 16, D)
    o = varlen_attention_fp4(q.to(DEV), kc.to(DEV), vc.to(DEV), cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens),
                             max_seqlen_q=300, block_table=tables.to(DEV), softmax_scale=SCALE)
    _check(o, *_varlen(q, kc, vc, tables, new, lens))


# ---------------------------------------------------------------------------------------------------------------------
# together, as an engine uses them


def test_flash_attn_entry_points_take_4_bit_caches():
    gen = _gen(40)
    lens = [300, 77]
    kc, vc, tables = _pool(gen, lens, 2)
    kd, vd, td = kc.to(DEV), vc.to(DEV), tables.to(DEV)
    dev_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = randn(gen, 2, 5, 16, D)
    o = ops.flash_attn_with_kvcache(q[:, :1].to(DEV), kd, vd, cache_seqlens=dev_lens, block_table=td, causal=True)
    assert o.shape == (2, 1, 16, D)
    _check(o[:, 0], *_varlen(q[:, 0], kc, vc, tables, [1, 1], lens))
    want = _varlen(q.reshape(10, 16, D), kc, vc, tables, [5, 5], lens)
    o = ops.flash_attn_with_kvcache(q.to(DEV), kd, vd, cache_seqlens=dev_lens, block_table=td, causal=True)
    _check(o.view(10, 16, D), *want)
    o = ops.flash_attn_varlen_func(q.reshape(10, 16, D).to(DEV), kd, vd, _cu([5, 5]), _cu(lens), 5, 300, causal=True,
                                   block_table=td)
    _check(o, *want)


@pytest.mark.parametrize("hk", [1, 2])
def test_engine_steps_through_attention_forward(hk):
    """A prompt stored and attended over its own rows, a second one over the cached prefix, decode steps eagerly and as a
    captured graph replayed over moving lengths: two layers of 4-bit caches, every output against the cache's values."""
    gen = _gen(41 + hk)
    heads = 8 * hk
    layers = [Attention(heads, D, SCALE, hk) for _ in range(2)]
    kv = runner.allocate_kv_cache(layers, 8, BS, dtype=torch.float4_e2m1fn_x2, device=DEV)
    kv.zero_()
    assert runner.kv_cache_block_bytes(layers, BS, torch.float4_e2m1fn_x2) * 8 == kv.numel()
    tasks = [runner.RunnerTask([5, 2], 250, 0, BS), runner.RunnerTask([7], 37, 0, BS)]

    def rows(n):
        x = randn(gen, 2, n, heads + 2 * hk, D).to(DEV)
        return [(x[i, :, :heads], x[i, :, heads:heads + hk], x[i, :, heads + hk:]) for i in range(2)]

    def check(o, q, new, lens, i, what):
        tables = [t.block_table + [-1] * (2 - len(t.block_table)) for t in tasks]
        _check(o, *_varlen(q.cpu(), layers[i].k_cache.cpu(), layers[i].v_cache.cpu(), torch.tensor(tables), new, lens), what)

    try:
        runner.prepare_prefill_context(tasks, BS, device=DEV)
        for i, (q, k, v) in enumerate(rows(287)):
            o = layers[i](q, k, v)
            kk, vv = (torch.tensor_split(t.cpu().double(), [250]) for t in (k, v))
            want = [_attend(a, b, c, True, SCALE) for a, b, c in zip(torch.tensor_split(q.cpu(), [250]), kk, vv)]
            tol = torch.cat([w[1] for w in want])
            _check(o, torch.cat([w[0] for w in want]), tol, f"prompt, layer {i}")
        for t, n in zip(tasks, (270, 40)):
            t.num_cached_tokens, t.seq_length = t.seq_length, n
        runner.prepare_prefill_context(tasks, BS, device=DEV)
        for i, (q, k, v) in enumerate(rows(23)):
            check(layers[i](q, k, v), q, [20, 3], [270, 40], i, f"prefix, layer {i}")

        bufs = runner.DecodeGraphBuffers(4, 2, device=DEV)
        static = [tuple(t.clone() for t in r) for r in rows(4)]
        graph = None
        for step in range(4):
            for t in tasks:
                t.num_cached_tokens, t.seq_length = t.seq_length, t.seq_length + 1
            runner.prepare_decode_context(tasks, BS, device=DEV)
            if step == 0:  # eager
                for i, (q, k, v) in enumerate(rows(2)):
                    o = layers[i](q, k, v)
                    assert o.shape == (2, 1, heads, D)
                    check(o[:, 0], q, [1, 1], [t.seq_length for t in tasks], i, f"decode, layer {i}")
                continue
            bufs.load()
            bufs.bind(4)
            for dst, src in zip(static, rows(4)):
                for a, b in zip(dst, src):
                    a.copy_(b)
            if graph is None:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    [layer(*r) for layer, r in zip(layers, static)]
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    outs = [layer(*r) for layer, r in zip(layers, static)]
            graph.replay()
            torch.cuda.synchronize()
            for i in range(2):
                check(outs[i][:2, 0], static[i][0][:2], [1, 1], [t.seq_length for t in tasks], i, f"step {step}, layer {i}")
                assert (outs[i][2:] == 0).all()
    finally:
        reset_context()


def test_streams_forked_and_compacted_between_steps():
    """Two prompts stored in two layers, forked into takes, decode steps that store, a step that mixes a new prompt with
    them, some takes freed and the pool compacted: every output against what the cache holds, the last step's again
    bit for bit after the compaction."""
    gen = _gen(51)
    heads, hk, blocks, cols = 16, 2, 24, 6
    layers = [Attention(heads, D, SCALE, hk) for _ in range(2)]
    kv = runner.allocate_kv_cache(layers, blocks, BS, dtype=torch.float4_e2m1fn_x2, device=DEV)
    kv.random_(0, 120)  # (no scale that is none)
    tables = torch.full((2, cols), -1, dtype=torch.int32)
    tables[0, :3], tables[1, :2] = torch.tensor([21, 4, 17]), torch.tensor([9, 23])
    lens = [600, 300]

    def rows(n):
        x = randn(gen, 2, n, heads + 2 * hk, D).to(DEV)
        return [(x[i, :, :heads], x[i, :, heads:heads + hk], x[i, :, heads + hk:]) for i in range(2)]

    def slots(tables, new, lens):
        return torch.tensor([ref.slot_of(tables[b], j, BS) for b, (n, m) in enumerate(zip(new, lens)) for j in range(m - n, m)],
                            dtype=torch.int32, device=DEV)

    def step(tables, new, lens, r):
        outs = []
        for i, (q, k, v) in enumerate(r):
            kc, vc = kv[i, 0], kv[i, 1]
            if max(new) == 1:
                o = decode_attention_fp4(q, kc, vc, torch.tensor(lens, device=DEV), tables.to(DEV), SCALE, key=k, value=v,
                                         slot_mapping=slots(tables, new, lens), plan=(*lens, *tables.flatten().tolist()))
            else:
                store_kvcache_fp4(k, v, kc, vc, slots(tables, new, lens))
                o = varlen_attention_fp4(q, kc, vc, cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens), max_seqlen_q=max(new),
                                         block_table=tables.to(DEV), softmax_scale=SCALE)
            _check(o, *_varlen(q.cpu(), kc.cpu(), vc.cpu(), tables, new, lens))
            outs.append(o)
        return outs

    step(tables, lens, lens, rows(900))
    ct, cl = kv_pages.fork_kv_blocks(kv, tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                     torch.tensor([0, 1, 0], device=DEV), torch.tensor([1, 2, 3], device=DEV))
    assert cl.tolist() == [600, 300, 600]
    tables, lens = torch.cat([tables, ct.cpu()]), lens + cl.tolist()
    for _ in range(2):
        lens = [n + 1 for n in lens]
        step(tables, [1] * 5, lens, rows(5))
    tables = torch.cat([tables, torch.tensor([[11, 12] + [-1] * (cols - 2)], dtype=torch.int32)])
    lens = [n + 1 for n in lens] + [280]
    assert 4 * 285 <= 6 * 280
    step(tables, [1] * 5 + [280], lens, rows(285))
    keep = [0, 2, 3, 5]
    tables, lens = tables[keep], [lens[b] for b in keep]
    lens = [n + 1 for n in lens]
    r = rows(4)
    before = step(tables, [1] * 4, lens, r)
    moved, remap, live = kv_pages.compact_kv_blocks(kv, tables.to(DEV), torch.tensor(lens, device=DEV))
    moved = moved.cpu()
    assert int(live) == len({b for row in tables.tolist() for b in row if b >= 0}) == moved.max() + 1
    assert ((moved < 0) == (tables < 0)).all() and torch.equal(moved[0, :2], moved[1, :2])  # (children share full blocks)
    for a, b in zip(before, step(moved, [1] * 4, lens, r)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("seed", range(30))
def test_random_steps(seed):
    """Decode, prefill and mixed steps of random head layouts, block sizes, lengths, strides, unmapped blocks, table widths
    and decode grids, planned or not, causal or not."""
    from voxcpm2_arabic_dialects_turbo_amd import _lib
    gen = _gen(7000 + seed)

    def pick(*of):
        return of[int(torch.randint(0, len(of), (1,), generator=gen))]

    heads, hk = pick((16, 2), (8, 1), (16, 1), (4, 2), (2, 2), (1, 1), (8, 2))
    bs, kind, wgs = pick(64, 128, 256, 320), pick("decode", "store", "varlen", "mixed"), pick(0, 0, 0, 3, 77, 1000)
    n = pick(1, 2, 9, 33, 65, 130, 280)
    top = pick(20, 90, 700, 3000) if n < 60 else pick(20, 90, 400)
    lens = torch.randint(0, top + 1, (n,), generator=gen).tolist()
    new = [1] * n
    if kind == "varlen":
        new = torch.randint(0, pick(3, 40, 200), (n,), generator=gen).tolist()
    elif kind == "mixed":
        new[int(torch.randint(0, n, (1,), generator=gen))] = pick(2, 31, 257)
    if kind == "store" and heads // hk > 8:
        kind = "decode"
    lens = [max(a, b) if pick(True, True, False) or kind == "store" else b for a, b in zip(new, lens)]
    kc, vc, tables = _pool(gen, lens, hk, bs, extra_cols=pick(0, 1, 40))
    scale = pick(SCALE, 0.02, 0.3)
    causal = pick(True, True, False) if kind in ("varlen", "mixed") else True
    t = sum(new)
    pad = pick(0, 3)
    q = randn(gen, max(t, 1) + pad, heads * D + pick(0, 2 * hk * D))[:, :heads * D].unflatten(1, (heads, D))
    qd, kd, vd = q.to(DEV), kc.to(DEV), vc.to(DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    plans = (None, ("random", seed), ("random", seed))
    try:
        if wgs:
            _lib.load().vox_set_decode_workgroups(wgs)
        for plan in plans:
            if kind in ("decode", "store"):
                kw = {}
                if kind == "store":
                    rows = randn(gen, n, 2 * hk * D).to(DEV)
                    k, v = rows[:, :hk * D].unflatten(1, (hk, D)), rows[:, hk * D:].unflatten(1, (hk, D))
                    slots = torch.tensor([ref.slot_of(tables[b], m - 1, bs) if m else -1 for b, m in enumerate(lens)],
                                         dtype=torch.int32, device=DEV)
                    kw = dict(key=k, value=v, slot_mapping=slots)
                    want_k, want_v = kd.clone(), vd.clone()
                    store_kvcache_fp4(k, v, want_k, want_v, slots)
                o = decode_attention_fp4(qd[:n], kd, vd, lens_d, tables.to(DEV), scale, plan=plan, **kw)
                if kind == "store":
                    assert torch.equal(kd, want_k) and torch.equal(vd, want_v)
                _check(o, *_varlen(q[:n], kd.cpu(), vd.cpu(), tables, new, lens, scale=scale), f"{kind}, plan {plan}")
            else:
                out = torch.full((len(q), heads, D), 7.0, dtype=torch.bfloat16, device=DEV)
                varlen_attention_fp4(qd, kd, vd, cu_seqlens_q=_cu(new), cu_seqlens_k=_cu(lens), max_seqlen_q=max(new),
                                     block_table=tables.to(DEV), softmax_scale=scale, causal=causal, out=out, plan=plan)
                _check(out[:t], *_varlen(q[:t], kc, vc, tables, new, lens, causal, scale), f"{kind}, plan {plan}")
                assert (out[t:] == 7).all()
    finally:
        _lib.load().vox_set_decode_workgroups(0)


def test_calls_on_two_streams_do_not_share_scratch():
    gen = _gen(50)
    lens = [[4000, 30, 2500], [100, 3900, 1200]]
    sets = [(*_pool(gen, n, 2), randn(gen, 3, 16, D), n) for n in lens]
    streams = [torch.cuda.Stream() for _ in sets]
    dev = [(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.tensor(n, device=DEV), t.to(DEV)) for kc, vc, t, q, n in sets]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(decode_attention_fp4(*dev[i], SCALE))
    torch.cuda.synchronize()
    for i, (kc, vc, t, q, n) in enumerate(sets):
        want = _varlen(q, kc, vc, t, [1] * 3, n)
        for o in outs[i]:
            _check(o, *want)


def test_a_captured_graph_and_eager_calls_between_its_replays():
    gen = _gen(51)
    lens = [1500, 700]
    kc, vc, tables = _pool(gen, lens, 2)
    q, kd, vd, td = randn(gen, 2, 16, D).to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    cu_q, cu_k = _cu([1, 1]), _cu(lens)
    eager = decode_attention_fp4(q, kd, vd, n, td, SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode_attention_fp4(q, kd, vd, n, td, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = decode_attention_fp4(q, kd, vd, n, td, SCALE)
        b = varlen_attention_fp4(q, kd, vd, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=1, block_table=td,
                                 softmax_scale=SCALE)
    for _ in range(4):
        a.zero_()
        graph.replay()
        decode_attention_fp4(q.flip(0).contiguous(), kd, vd, n, td, SCALE)
        torch.cuda.synchronize()
        assert torch.equal(a, eager) and torch.equal(b, eager)
