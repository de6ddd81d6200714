"""Key weights where a call's lengths pass what its tables reach or what it says: the attention's and the weights' kernels end a
context at the same place. Tolerances as in test_key_weights_gpu."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4
from oracle import key_weights as ref
from tests._util import paged_pool, randn
from tests.test_key_weights_gpu import D, DEV, SCALE, Want, _i32, _received
from voxcpm2_arabic_dialects_turbo_amd.ops_weights import decode_attention_weights, varlen_attention_weights

pytestmark = pytest.mark.gpu
H, HK, BS = 16, 2, 64


def _caches(gen, reach, batch, four_bit):
    """Caches of `batch` sequences whose tables reach `reach` tokens each: on the GPU, and their values and tables."""
    need = batch * reach // BS
    kc, vc, tables = paged_pool(gen, [reach] * batch, need, BS, HK)
    if not four_bit:
        return (kc.to(DEV), vc.to(DEV)), (kc, vc), tables
    planes = [fp4.plane(torch.randint(0, 256, (need, BS, HK, 64), generator=gen, dtype=torch.uint8),
                        torch.randint(123, 128, (need, BS, HK, 4), generator=gen, dtype=torch.uint8)) for _ in range(2)]
    return tuple(c.to(DEV) for c in planes), tuple(fp4.cache_values(c) for c in planes), tables


def _more(q, k, four_bit):
    """What the 4-bit caches' scores add to a probability's tolerance."""
    if not four_bit:
        return 0.0
    n = q.shape[0]
    size = (q.double().abs().view(n, HK, -1, D).transpose(0, 1).reshape(HK, -1, D) @ k.abs().permute(1, 2, 0)).max()
    x = SCALE * float(2.0 ** -13 * size + 2.0 ** -18 * q.abs().max() * k.abs().sum(-1).max())
    return 2 * x * (1 + 2 * x)


def _varlen(seed, seqs, reach, max_k, four_bit):
    """seqs: (queries, keys) as the call says them. A context ends at the tables' reach, its queries are its last tokens; keys
    at and past max_k count in the softmax and take no weight."""
    gen = torch.Generator().manual_seed(seed)
    caches, values, tables = _caches(gen, reach, len(seqs), four_bit)
    cu = torch.tensor([(0, 0), *seqs]).cumsum(0)
    q, w = randn(gen, int(cu[-1, 0]), H, D), _received(gen, len(seqs), HK, max(max_k, reach) + 64)
    for b, (n, m) in enumerate(seqs):  # a new token's place may hold anything
        m = min(m, reach)
        w[b, :, m - n:min(m, max_k)] = float("nan")
    wd = w.to(DEV)
    o = varlen_attention_weights(q.to(DEV), None, None, wd, cu_seqlens_q=_i32(cu[:, 0].tolist()),
                                 cu_seqlens_k=_i32(cu[:, 1].tolist()), max_seqlen_q=max(n for n, _ in seqs), max_seqlen_k=max_k,
                                 softmax_scale=SCALE, block_table=tables.to(DEV), k_cache=caches[0], v_cache=caches[1])
    want = Want(w)
    for b, (n, m) in enumerate(seqs):
        m = min(m, reach)
        k, v = (ref.keys_of(c, tables[b], m)[0] for c in values)
        qb, before = q[cu[b, 0]:cu[b + 1, 0]], want.w[b].clone()
        want.sequence(qb, k, v, None, b, n, more=_more(qb, k, four_bit))
        want.w[b][:, max_k:] = before[:, max_k:]
        want.tol[b][:, max_k:] = 0
    want.check(o, wd)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("seqs", [
    [(20, 250), (40, 192), (30, 100), (1, 300), (3, 192)], [(100, 1000), (150, 193)]])
def test_chunks_past_their_tables(seqs, four_bit):
    _varlen(len(seqs), seqs, 192, 1000, four_bit)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("seqs", [
    [(1, 250), (1, 192), (1, 193), (1, 100), (1, 1000)], [(1, 200 + i) for i in range(20)] + [(60, 230)]])
def test_decode_rows_past_their_tables(seqs, four_bit):
    """Decode rows alone, and beside a chunk."""
    _varlen(10 + len(seqs), seqs, 192, 1000, four_bit)


@pytest.mark.parametrize("four_bit", [False, True])
def test_decode_contexts_past_their_tables(four_bit):
    """The last token that the table reaches is the newest one."""
    gen = torch.Generator().manual_seed(40)
    caches, values, tables = _caches(gen, 192, 4, four_bit)
    lens = [193, 192, 50, 100000]
    q, w = randn(gen, 4, H, D), _received(gen, 4, HK, 192)
    for b, n in enumerate(lens):
        w[b, :, min(n, 192) - 1] = float("nan")
    wd = w.to(DEV)
    o = decode_attention_weights(q.to(DEV), *caches, _i32(lens), tables.to(DEV), SCALE, wd)
    want = Want(w)
    for b, n in enumerate(lens):
        k, v = (ref.keys_of(c, tables[b], min(n, 192))[0] for c in values)
        want.sequence(q[b:b + 1], k, v, None, b, 1, more=_more(q[b:b + 1], k, four_bit))
    want.check(o, wd)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("seqs", [
    [(1, 150), (1, 90), (1, 100), (1, 101), (1, 192)],
    [(1, 80 + 5 * i) for i in range(20)] + [(60, 150)],
    [(20, 150), (40, 192), (1, 150)]])
def test_keys_past_what_the_call_says(seqs, four_bit):
    """The same on the decode kernels as on the chunk's."""
    _varlen(30 + len(seqs), seqs, 192, 100, four_bit)
