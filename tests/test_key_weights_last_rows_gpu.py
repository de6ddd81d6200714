"""Key weights of a step that has fewer queries than new tokens, as a model's last layer has where only the last row of every
sequence goes on: every token of the step starts with what these queries give it. Tolerances as in test_key_weights_gpu."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp4
from oracle import key_weights as ref
from tests._util import paged_pool, randn
from tests.test_key_weights_gpu import D, DEV, SCALE, Want, _i32, _received
from voxcpm2_arabic_dialects_turbo_amd import ops, runner
from voxcpm2_arabic_dialects_turbo_amd.context import get_context, reset_context
from voxcpm2_arabic_dialects_turbo_amd.layers import Attention
from voxcpm2_arabic_dialects_turbo_amd.ops_weights import varlen_attention_weights

pytestmark = pytest.mark.gpu
H, HK, BS = 16, 2, 256


@pytest.fixture(autouse=True)
def _context():
    yield
    reset_context()
    ops.forget_plans()


def _step(gen, cached, dtype):
    """A layer, the tasks of a step and its rows; the layer's weights are NaN, as another sequence may have left them, but for
    the cached tokens'."""
    layer = Attention(H, D, SCALE, HK)
    runner.allocate_kv_cache([layer], num_blocks=32, block_size=BS, dtype=dtype, device=DEV)
    if dtype == torch.bfloat16:
        for c in (layer.k_cache, layer.v_cache):
            c.copy_(randn(gen, *c.shape).to(DEV))
    else:
        for c in (layer.k_cache, layer.v_cache):
            c.copy_(fp4.plane(torch.randint(0, 256, (32, BS, HK, 64), generator=gen, dtype=torch.uint8),
                              torch.randint(123, 128, (32, BS, HK, 4), generator=gen, dtype=torch.uint8)))
    runner.allocate_key_weights([layer], 6, 3 * BS, device=DEV)
    lengths, rows = [40, 300, 513, 7], [4, 0, -1, 2]
    perm, tasks, at = torch.randperm(32, generator=gen).tolist(), [], 0
    w = torch.full((6, HK, 3 * BS), float("nan"))
    for n, c, r in zip(lengths, cached, rows):
        nb = -(-n // BS)
        tasks.append(runner.RunnerTask(perm[at:at + nb], n, c, BS))
        at += nb
        if r >= 0:
            w[r, :, :c] = 3 * torch.rand(HK, c, generator=gen)
    layer.key_weights.copy_(w.to(DEV))
    new = [n - c for n, c in zip(lengths, cached)]
    q, k, v = randn(gen, len(tasks), H, D), randn(gen, sum(new), HK, D), randn(gen, sum(new), HK, D)
    return layer, tasks, rows, new, w, q, k, v


def _last_rows(layer, q, k, v):
    """One query per sequence, set on the live context around the call."""
    ctx = get_context()
    saved = ctx.cu_seqlens_q, ctx.max_seqlen_q
    ctx.cu_seqlens_q, ctx.max_seqlen_q = torch.arange(q.shape[0] + 1, dtype=torch.int32, device=DEV), 1
    try:
        return layer(q, k, v)
    finally:
        ctx.cu_seqlens_q, ctx.max_seqlen_q = saved


def _expect(layer, tasks, rows, new, w, q, k, v, paged):
    want, at, four_bit = Want(w), 0, layer.k_cache.dtype == torch.uint8
    caches = [fp4.cache_values(c.cpu()) if four_bit else c.cpu() for c in (layer.k_cache, layer.v_cache)]
    for b, (t, n, r) in enumerate(zip(tasks, new, rows)):
        keys, vals = (ref.keys_of(c, t.block_table, t.seq_length)[0] for c in caches) if paged else \
            (k[at:at + n], v[at:at + n])
        at += n
        more = 0.0
        if four_bit and paged:
            size = (q[b].double().abs().view(HK, -1, D) @ keys.abs().permute(1, 2, 0)).max()
            x = SCALE * float(2.0 ** -13 * size + 2.0 ** -18 * q[b].abs().max() * keys.abs().sum(-1).max())
            more = 2 * x * (1 + 2 * x)
        want.sequence(q[b:b + 1], keys, vals, None, r, n, more=more)
    return want


DTYPES = [torch.bfloat16, torch.float4_e2m1fn_x2]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cached", [[0, 0, 0, 0], [0, 260, 100, 3]])
def test_last_rows_start_the_steps_tokens(cached, dtype):
    """Packed and through block tables, over caches of both kinds."""
    gen = torch.Generator().manual_seed(5 + sum(cached))
    layer, tasks, rows, new, w, q, k, v = _step(gen, cached, dtype)
    runner.prepare_prefill_context(tasks, BS, device=DEV, weight_rows=rows)
    o = _last_rows(layer, q.to(DEV), k.to(DEV), v.to(DEV))
    _expect(layer, tasks, rows, new, w, q, k, v, any(cached)).check(o, layer.key_weights)


def test_last_rows_beside_whole_steps():
    """A layer of all rows, one of the last rows and one of all rows again in one context: each starts its own tokens."""
    gen = torch.Generator().manual_seed(9)
    layer, tasks, rows, new, w, q, k, v = _step(gen, [0, 260, 100, 3], torch.bfloat16)
    runner.prepare_prefill_context(tasks, BS, device=DEV, weight_rows=rows)
    whole = randn(gen, sum(new), H, D)
    layer(whole.to(DEV), k.to(DEV), v.to(DEV))
    first = layer.key_weights.clone()
    layer.key_weights.copy_(w.to(DEV))
    o = _last_rows(layer, q.to(DEV), k.to(DEV), v.to(DEV))
    _expect(layer, tasks, rows, new, w, q, k, v, True).check(o, layer.key_weights)
    layer.key_weights.copy_(w.to(DEV))
    layer(whole.to(DEV), k.to(DEV), v.to(DEV))
    assert torch.equal(layer.key_weights.view(torch.int32), first.view(torch.int32))


@pytest.mark.parametrize("cached", [[0, 0, 0, 0], [0, 260, 100, 3]])
def test_captured_last_rows(cached):
    gen = torch.Generator().manual_seed(10)
    layer, tasks, rows, new, w, q, k, v = _step(gen, cached, torch.bfloat16)
    qd, kd, vd, wd = q.to(DEV), k.to(DEV), v.to(DEV), w.to(DEV)
    runner.prepare_prefill_context(tasks, BS, device=DEV, weight_rows=rows)
    _last_rows(layer, qd, kd, vd)
    layer.key_weights.copy_(wd)
    eager, ew = _last_rows(layer, qd, kd, vd).clone(), layer.key_weights.clone()
    _expect(layer, tasks, rows, new, w, q, k, v, any(cached)).check(eager, ew)
    ones = torch.arange(5, dtype=torch.int32, device=DEV)
    ctx = get_context()
    ctx.cu_seqlens_q, ctx.max_seqlen_q = ones, 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = layer(qd, kd, vd)
    for _ in range(4):
        layer.key_weights.copy_(wd)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, eager) and torch.equal(layer.key_weights.view(torch.int32), ew.view(torch.int32))


@pytest.mark.parametrize("bs", [None, 64])
def test_fewer_queries_than_new_tokens(bs):
    """The operator itself: the last queries of each sequence, rows in any order and none, a sequence of new tokens without any
    query (they start with nothing), one whose new tokens are all that it has, int64 index tensors."""
    gen = torch.Generator().manual_seed(20)
    seqs = [(3, 40, 100), (1, 1, 70), (0, 30, 90), (20, 20, 20), (2, 150, 150), (4, 33, 65)]  # queries, new, keys
    rows = [3, 0, 5, 1, -1, 2]
    if bs is None:
        seqs = [(n, m, m) for n, _, m in seqs]
    lens, cu = [m for _, _, m in seqs], np.cumsum([(0, 0, 0), *seqs], 0)
    q = randn(gen, int(cu[-1, 0]), 16, D)
    w = _received(gen, 8, 2, 256)
    for (_, new, m), r in zip(seqs, rows):
        if r >= 0:
            w[r, :, m - new:m] = float("nan")
    kw = {}
    if bs:
        kc, vc, tables = paged_pool(gen, lens, 20, bs, 2)
        keys = [tuple(ref.keys_of(c, tables[b], m)[0] for c in (kc, vc)) for b, m in enumerate(lens)]
        kd = vd = None
        kw.update(block_table=tables.to(DEV), k_cache=kc.to(DEV), v_cache=vc.to(DEV))
    else:
        k, v = randn(gen, int(cu[-1, 2]), 2, D), randn(gen, int(cu[-1, 2]), 2, D)
        keys = [(k[a:e], v[a:e]) for a, e in zip(cu[:, 2], cu[1:, 2])]
        kd, vd = k.to(DEV), v.to(DEV)
    wd = w.to(DEV)
    o = varlen_attention_weights(q.to(DEV), kd, vd, wd, _i32(rows), cu_seqlens_q=_i32(cu[:, 0].tolist()),
                                 cu_seqlens_k=_i32(cu[:, 2].tolist()), max_seqlen_q=20, max_seqlen_k=max(lens),
                                 softmax_scale=SCALE, cu_seqlens_new=torch.tensor(cu[:, 1].copy(), device=DEV), **kw)
    want = Want(w)
    for b, (n, new, m) in enumerate(seqs):
        want.sequence(q[cu[b, 0]:cu[b + 1, 0]], *keys[b], None, rows[b], new)
        if n == 0 and rows[b] >= 0:
            want.w[rows[b], :, m - new:m] = 0
    want.check(o, wd)
