"""Key weights of chunks over 4-bit keys that bf16 does not hold: the format's scales end at 2^127, where codes stand for 2^128
and more. Such a key is a number to the attention, whose scores come from the codes, so it takes its weight like any other.

Tolerances as in test_key_weights_gpu. What the query's two fp8 parts leave (2^-18 of the row's largest magnitude a channel)
counts at the channels where the query is not 0: a 0 is held exactly."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4
from oracle import key_weights as ref
from tests._util import paged_pool, randn
from tests.test_fp4_other_writers_gpu import CASES
from tests.test_key_weights_gpu import D, DEV, SCALE, Want, _i32, _received
from voxcpm2_arabic_dialects_turbo_amd.ops_weights import varlen_attention_weights

pytestmark = pytest.mark.gpu
BS, FAR = 64, 41  # FAR: the channel of the values past bf16


def _queries(gen, n, h, kind):
    """"zero": nothing at channel FAR. "small": every magnitude in [2^-123, 2^-122), so that 6 x 2^127 gives a score of some 10.
    "large": [2^123, 2^124) at channels 64 to 95 and nothing elsewhere, so that the least scales there give one of some 3."""
    if kind == "zero":
        q = randn(gen, n, h, D)
        q[..., FAR] = 0
        return q
    sign = torch.randint(0, 2, (n, h, D), generator=gen) * 2.0 - 1
    q = sign * (1 + torch.rand(n, h, D, generator=gen)).to(torch.bfloat16).clamp(max=1.9921875)
    if kind == "small":
        return (q * 2.0 ** -123).to(torch.bfloat16)
    q[..., :64], q[..., 96:] = 0, 0
    return (q * 2.0 ** 123).to(torch.bfloat16)


@pytest.mark.parametrize("kind", ["zero", "small", "large"])
@pytest.mark.parametrize("seqs,h,hk", [
    ([(60, 200)], 16, 2), ([(60, 60)], 8, 1), ([(130, 300)] * 30, 16, 2), ([(130, 300)] * 60, 16, 2),
    ([(1, 90 + i) for i in range(21)] + [(90, 190)], 16, 2), ([(700, 700)], 8, 1)])
def test_chunks(seqs, h, hk, kind):
    """Half key blocks and whole ones, direct and persistent grids, parts, decode rows beside a chunk. Each sequence has two such
    keys at its last kv head, a case of its own, beside groups of the least scales."""
    gen = torch.Generator().manual_seed(len(seqs) + h + len(kind))
    lens, T, cu_q, cu_k = [m for _, m in seqs], sum(n for n, _ in seqs), [0], [0]
    for n, m in seqs:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    need = sum(-(-n // BS) for n in lens) + 1
    _, _, tables = paged_pool(gen, lens, need, BS, 1, 1)
    planes = []
    for x in range(2):
        codes = torch.randint(0, 256, (need * BS, hk, 64), generator=gen, dtype=torch.uint8)
        scales = torch.randint(123, 128, (need * BS, hk, 4), generator=gen, dtype=torch.uint8)
        least = codes[..., 32:48].clone()
        if x == 0 and kind == "large":
            codes[..., 32:48] = 0
        for b, (n, m) in enumerate(seqs if x == 0 else []):
            byte, code, _ = CASES[(b + 1) % len(CASES)]
            for at in {5, m - n}:
                slot = int(tables[b, at // BS]) * BS + at % BS
                codes[slot, hk - 1, 16:32] = 0
                codes[slot, hk - 1, FAR // 2] = code << 4
                codes[slot, hk - 1, 32:48] = least[slot, hk - 1]
                scales[slot, hk - 1] = torch.tensor([125, byte, b % 3, 126], dtype=torch.uint8)
        planes.append(fp4.plane(codes.view(need, BS, hk, 64), scales.view(need, BS, hk, 4)))
    q, w = _queries(gen, T, h, kind), _received(gen, len(seqs), hk, tables.shape[1] * BS)
    for b, (n, m) in enumerate(seqs):
        w[b, :, m - n:m] = float("nan")
    wd = w.to(DEV)
    o = varlen_attention_weights(q.to(DEV), None, None, wd, cu_seqlens_q=_i32(cu_q), cu_seqlens_k=_i32(cu_k),
                                 max_seqlen_q=max(n for n, _ in seqs), max_seqlen_k=max(lens), softmax_scale=SCALE,
                                 block_table=tables.to(DEV), k_cache=planes[0].to(DEV), v_cache=planes[1].to(DEV))
    kv, vv = (fp4.cache_values(c) for c in planes)
    want = Want(w)
    for b, (n, m) in enumerate(seqs):
        (k, _), (v, _) = (ref.keys_of(c, tables[b], m) for c in (kv, vv))
        qb = q[cu_q[b]:cu_q[b + 1]].double()
        size = (qb.abs().view(n, hk, -1, D).transpose(0, 1).reshape(hk, -1, D) @ k.abs().permute(1, 2, 0)).max()
        live = (qb != 0).any(0).any(0)
        x = SCALE * float(2.0 ** -13 * size + 2.0 ** -18 * qb.abs().max() * k.abs()[..., live].sum(-1).max())
        assert x < 0.05
        want.sequence(q[cu_q[b]:cu_q[b + 1]], k, v, None, b, n, more=2 * x * (1 + 2 * x))
    want.check(o, wd)
