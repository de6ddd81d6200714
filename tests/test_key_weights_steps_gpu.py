"""Steps that add to key weights, through Attention.forward: prompts, captured decode steps, eviction, decode steps behind it,
forks evicted into blocks of their own, several streams and graphs. Every step is held to the float64 oracle from the state
that the GPU had before it; tolerances as in test_key_weights_gpu."""

from __future__ import annotations

import pytest
import torch

from oracle import key_weights as ref
from tests._util import randn
from tests.test_key_weights_gpu import D, DEV, SCALE, Want, _i32
from voxcpm2_arabic_dialects_turbo_amd import ops, runner
from voxcpm2_arabic_dialects_turbo_amd.context import get_context, reset_context
from voxcpm2_arabic_dialects_turbo_amd.kernels.kv_evict import evict_kv_tokens
from voxcpm2_arabic_dialects_turbo_amd.kernels.kv_pages import fork_kv_blocks
from voxcpm2_arabic_dialects_turbo_amd.layers import Attention
from voxcpm2_arabic_dialects_turbo_amd.ops_weights import decode_attention_weights, varlen_attention_weights

pytestmark = pytest.mark.gpu
H, HK, BS = 16, 2, 256


@pytest.fixture(autouse=True)
def _context():
    yield
    reset_context()
    ops.forget_plans()


class Engine:
    """Layers over one pool, with the oracle's copy of it."""

    def __init__(self, layers=2, blocks=24, rows=6, reach=1024, seed=0):
        self.gen = torch.Generator().manual_seed(seed)
        self.layers = [Attention(H, D, SCALE, HK) for _ in range(layers)]
        self.kv = runner.allocate_kv_cache(self.layers, blocks, BS, device=DEV)
        self.kv.zero_()
        self.weights = runner.allocate_key_weights(self.layers, rows, reach, device=DEV)
        self.weights.fill_(float("nan"))  # (whatever the last sequences left)

    def rows(self, n):
        return randn(self.gen, n, H, D), randn(self.gen, n, HK, D), randn(self.gen, n, HK, D)

    def step(self, tasks, rows, prefill, run=None, evicted=None, graphs=False):
        """One step of every layer, checked."""
        kw = dict(device=DEV, weight_rows=rows, evicted=evicted)
        if prefill:
            runner.prepare_prefill_context(tasks, BS, graphs=graphs, **kw)
        else:
            runner.prepare_decode_context(tasks, BS, **kw)
        new = [t.seq_length - t.num_cached_tokens for t in tasks] if prefill else [1] * len(tasks)
        kv, weights = self.kv.cpu(), self.weights.cpu()
        data = [self.rows(sum(new)) for _ in self.layers]
        if run is None:
            outs = [layer(*(x.to(DEV) for x in d)) for layer, d in zip(self.layers, data)]
        else:
            outs = run(data)
        for i, (q, k, v) in enumerate(data):
            want, at = Want(weights[i]), 0
            for t, n, r in zip(tasks, new, rows):
                for j in range(n):
                    p = t.seq_length - n + j
                    kv[i, 0, t.block_table[p // BS], p % BS], kv[i, 1, t.block_table[p // BS], p % BS] = k[at + j], v[at + j]
                keys, vals = (ref.keys_of(kv[i, c], t.block_table, t.seq_length)[0] for c in (0, 1))
                want.sequence(q[at:at + n], keys, vals, None, r, n)
                at += n
            want.check(outs[i].reshape(sum(new), H, D), self.weights[i])
        assert torch.equal(self.kv.cpu(), kv)

    def evict(self, tasks, rows, budget, sinks, recent, new_blocks=None):
        kv, weights = self.kv.cpu(), self.weights.cpu()
        width = max(len(t.block_table) for t in tasks)
        tables = [t.block_table + [-1] * (width - len(t.block_table)) for t in tasks]
        lens = [t.seq_length for t in tasks]
        t, n = evict_kv_tokens(self.kv, self.weights, _i32(tables), _i32(lens), budget, recent=recent, sinks=sinks,
                               weight_rows=_i32(rows), new_blocks=None if new_blocks is None else _i32(new_blocks))
        want_t, want_n = ref.evict(kv, weights, tables, lens, budget, sinks, recent, rows, new_blocks)
        assert t.tolist() == want_t and n.tolist() == want_n
        assert torch.equal(self.kv.cpu(), kv) and torch.equal(self.weights.cpu().view(torch.int32), weights.view(torch.int32))
        lost = [a - b for a, b in zip(lens, want_n)]
        for task, row, m in zip(tasks, want_t, want_n):
            task.block_table, task.seq_length = [b for b in row if b >= 0], m
        return lost


def _next(task, spare):
    task.num_cached_tokens = task.seq_length
    task.seq_length += 1
    if task.seq_length > len(task.block_table) * BS:
        task.block_table.append(spare.pop())


def test_a_text_read_evicted_and_gone_on_with():
    """Prompts, decode steps, eviction, a chunk and decode steps behind it, and eviction again, two layers, three sequences
    in rows of any order; the planned decode calls of a step share their layout."""
    e, spare = Engine(), list(range(12, 24))
    tasks = [runner.RunnerTask([0, 1], 400, 0), runner.RunnerTask([2], 30, 0), runner.RunnerTask([3, 4, 5], 700, 0)]
    rows = [4, 0, 2]
    e.step(tasks, rows, True)
    for _ in range(2):
        for t in tasks:
            _next(t, spare)
        e.step(tasks, rows, False)
    lost = e.evict(tasks, rows, 250, 4, 50)
    assert lost == [152, 0, 452]
    for t in tasks:  # new text behind what is left: a chunk over the caches
        t.num_cached_tokens, t.seq_length = t.seq_length, t.seq_length + 40
        while t.seq_length > len(t.block_table) * BS:
            t.block_table.append(spare.pop())
    e.step(tasks, rows, True, evicted=lost)
    for _ in range(2):
        for t in tasks:
            _next(t, spare)
        e.step(tasks, rows, False, evicted=lost)
    again = e.evict(tasks, rows, 60, 0, 60)
    assert again == [232, 14, 232]  # (30 + 2 + 40 + 2 - 60)
    for t in tasks:
        _next(t, spare)
    e.step(tasks, rows, False, evicted=[a + b for a, b in zip(lost, again)])


def test_a_sequence_without_a_row_beside_others():
    e, spare = Engine(), list(range(12, 24))
    tasks = [runner.RunnerTask([0, 1], 300, 0), runner.RunnerTask([2], 30, 0)]
    e.step(tasks, [-1, 3], True)
    for t in tasks:
        _next(t, spare)
    e.step(tasks, [-1, 3], False)
    assert e.weights[:, :3].isnan().all() and e.evict(tasks, [-1, 3], 20, 1, 1) == [0, 11]


def test_captured_decode_steps():
    """One graph replayed over steps of other sequences, lengths and rows, with eager steps and eviction between."""
    e, spare = Engine(), list(range(12, 24))
    bufs = runner.DecodeGraphBuffers(4, 4, device=DEV, key_weights=True)
    tasks = [runner.RunnerTask([0, 1], 400, 0), runner.RunnerTask([2], 30, 0), runner.RunnerTask([3], 200, 0)]
    rows = [4, 0, 2]
    e.step(tasks, rows, True)
    static = [[torch.zeros(4, h, D, dtype=torch.bfloat16, device=DEV) for h in (H, HK, HK)] for _ in e.layers]
    bufs.bind(4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):  # (padded rows: nothing is stored or added)
        before = e.weights.clone()
        for layer, s in zip(e.layers, static):
            layer(*s)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(e.weights.nan_to_num(7.0), before.nan_to_num(7.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [layer(*s) for layer, s in zip(e.layers, static)]

    def run(data):
        bufs.load()
        n = data[0][0].shape[0]
        for s, d in zip(static, data):
            for x, y in zip(s, d):
                x.zero_()
                x[:n] = y.to(DEV)
        graph.replay()
        torch.cuda.synchronize()
        return [o[:n].clone() for o in outs]

    for i in range(5):
        for t in tasks:
            _next(t, spare)
        e.step(tasks, rows, False, run=run)
        if i == 1:
            assert e.evict(tasks, rows, 150, 2, 40) == [252, 0, 52]
        if i == 2:
            for t in tasks:
                _next(t, spare)
            e.step(tasks, rows, False)  # eager, in between
            tasks, rows = tasks[::-1][:2], rows[::-1][:2]


def test_captured_chunk_and_eviction():
    """A chunk and the eviction behind it in one graph, replayed over other contents of its buffers."""
    gen = torch.Generator().manual_seed(9)
    h, hk, bs, n, m = 8, 1, 64, 40, 300
    tables = torch.tensor([[5, 0, 3, 7, 1]], dtype=torch.int32)
    kv = torch.zeros(1, 2, 8, bs, hk, D, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(n, h, D, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(1, 1, hk, 320, device=DEV)
    args = dict(cu_seqlens_q=_i32([0, n]), cu_seqlens_k=_i32([0, m]), max_seqlen_q=n, max_seqlen_k=m, softmax_scale=SCALE,
                block_table=tables.to(DEV))
    lens = _i32([m])

    def step():
        o = varlen_attention_weights(q, None, None, w[0], k_cache=kv[0, 0], v_cache=kv[0, 1], **args)
        return o, *evict_kv_tokens(kv, w, args["block_table"], lens, 100, recent=n, sinks=3)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        kv0, q0 = randn(gen, 1, 2, 8, bs, hk, D), randn(gen, n, h, D)
        w0 = torch.rand(1, 1, hk, 320, generator=gen)
        results = []
        for run in (graph.replay, None):
            kv.copy_(kv0)
            q.copy_(q0)
            w.copy_(w0)
            outs = step() if run is None else (run(), got)[1]
            torch.cuda.synchronize()
            results.append([x.clone() for x in (*outs, kv, w)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        assert results[0][2].tolist() == [100] and results[0][1].tolist() == [[5, 0, -1, -1, -1]]


def test_takes_of_one_text_are_evicted_into_blocks_of_their_own():
    """Two children of a parent share its full blocks; each goes on, and is brought down into new blocks, the parent's blocks
    as they were; the parent goes on from them."""
    e = Engine(blocks=20)
    parent = runner.RunnerTask([0, 1, 2], 600, 0)
    e.step([parent], [0], True)
    t, n = fork_kv_blocks(e.kv, _i32([parent.block_table]), _i32([600]), _i32([0, 0]), _i32([3, 4]))
    takes = [runner.RunnerTask(row, m, m) for row, m in zip(t.tolist(), n.tolist())]
    e.weights[:, 1:3] = e.weights[:, :1]
    for _ in range(3):
        for task in (parent, *takes):
            _next(task, [])
        e.step([parent, *takes], [0, 1, 2], False)
    kept = e.kv[:, :, :3].clone()
    lost = e.evict(takes, [1, 2], 300, 4, 64, [[5, 6, -1], [7, 8, -1]])
    assert lost == [303, 303] and [t.block_table for t in takes] == [[5, 6], [7, 8]]
    assert torch.equal(e.kv[:, :, :3], kept)
    for task in (parent, *takes):
        _next(task, [])
    e.step([parent, *takes], [0, 1, 2], False, evicted=[0, *lost])


def test_mixed_step():
    """Chunks, prompts and one-query rows of long contexts in one step through the block tables."""
    e, spare = Engine(blocks=24), list(range(16, 24))
    tasks = [runner.RunnerTask([0, 1, 2, 3], 1000, 0), runner.RunnerTask([4], 100, 0), runner.RunnerTask([5, 6], 500, 0)]
    e.step(tasks, [0, 1, 2], True)
    for t in tasks:
        _next(t, spare)
    tasks[1].seq_length += 29  # (a chunk of 30)
    e.step([*tasks, runner.RunnerTask([7], 64, 0)], [0, 1, 2, 5], True)


def test_calls_on_another_stream_and_device_argument():
    """Two streams at once, each with its own weights: unplanned calls do not share scratch."""
    gen = torch.Generator().manual_seed(4)
    lens, width = [700, 90], 768
    kc, vc = randn(gen, 6, BS, HK, D).to(DEV), randn(gen, 6, BS, HK, D).to(DEV)
    tables, n = _i32([[0, 1, 2], [3, -1, -1]]), _i32(lens)
    qs = [randn(gen, 2, H, D).to(DEV) for _ in range(8)]
    want = []
    for q in qs:
        w = torch.zeros(2, HK, width, device=DEV)
        want.append((decode_attention_weights(q, kc, vc, n, tables, SCALE, w), w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            w = torch.zeros(2, HK, width, device=DEV)
            got.append((decode_attention_weights(q, kc, vc, n, tables, SCALE, w), w))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_planned_step_is_the_unplanned_one():
    """Layers that reuse a step's layout, with lengths that change between steps."""
    gen = torch.Generator().manual_seed(5)
    kc, vc = randn(gen, 12, BS, HK, D).to(DEV), randn(gen, 12, BS, HK, D).to(DEV)
    tables = _i32([[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]])
    for step, lens in enumerate(([700, 90, 1024], [701, 91, 1], [1024, 0, 512])):
        for layer in range(3):
            q = randn(gen, 3, H, D).to(DEV)
            a, b = torch.ones(3, HK, 1024, device=DEV), torch.ones(3, HK, 1024, device=DEV)
            x = decode_attention_weights(q, kc, vc, _i32(lens), tables, SCALE, a, plan=("step", step))
            y = decode_attention_weights(q, kc, vc, _i32(lens), tables, SCALE, b)
            assert torch.equal(x, y) and torch.equal(a, b)
    assert get_context().weight_rows is None


def test_layers_with_and_without_weights_in_one_planned_step():
    """Calls of both kinds, riding stores and varlen calls among them, under one plan key: each as without a plan."""
    gen = torch.Generator().manual_seed(6)
    kc, vc = randn(gen, 12, BS, HK, D).to(DEV), randn(gen, 12, BS, HK, D).to(DEV)
    tables, lens = _i32([[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]]), [700, 90, 1024]
    slots = _i32([699, 4 * BS + 89, 8 * BS + 1023])
    cu_k = _i32([0, 700, 790, 1814])
    kw = dict(cu_seqlens_q=_i32([0, 1, 2, 3]), cu_seqlens_k=cu_k, max_seqlen_q=1, max_seqlen_k=1024, softmax_scale=SCALE,
              block_table=tables, k_cache=kc, v_cache=vc)
    new = dict(key=randn(gen, 3, HK, D).to(DEV), value=randn(gen, 3, HK, D).to(DEV), slot_mapping=slots)
    decode_attention_weights(randn(gen, 3, H, D).to(DEV), kc, vc, _i32(lens), tables, SCALE,
                             torch.ones(3, HK, 1024, device=DEV), **new)  # (the rows are there from here on)
    for kind in "wdwwvdswsvvw":
        q = randn(gen, 3, H, D).to(DEV)
        got = []
        for plan in (("one", 1), None) if kind != "d" else (("one", 1), ("other", kind)):
            w = torch.ones(3, HK, 1024, device=DEV)
            if kind == "d":
                o = ops.decode_attention(q, kc, vc, _i32(lens), tables, SCALE, plan=plan)
            elif kind == "v":
                o = varlen_attention_weights(q, None, None, w, **kw, plan=plan)
            else:
                o = decode_attention_weights(q, kc, vc, _i32(lens), tables, SCALE, w, plan=plan,
                                             **(new if kind == "s" else {}))
            got.append((o, w))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
        assert got[0][0].isfinite().all() and (kind == "d" or (got[0][1] != 1).any())


def test_a_text_over_4_bit_caches():
    """Prompts, decode steps and evictions through the module over 4-bit caches: the calls' own outputs and weights, and tokens
    that go on from what an eviction left."""
    gen = torch.Generator().manual_seed(7)
    layers = [Attention(H, D, SCALE, HK) for _ in range(2)]
    kv = runner.allocate_kv_cache(layers, 12, BS, dtype=torch.uint8 if not hasattr(torch, "float4_e2m1fn_x2")
                                  else torch.float4_e2m1fn_x2, device=DEV)
    weights = runner.allocate_key_weights(layers, 4, 1024, device=DEV)
    weights.fill_(float("nan"))
    tasks, rows = [runner.RunnerTask([0, 1], 300, 0), runner.RunnerTask([2], 30, 0)], [3, 1]
    runner.prepare_prefill_context(tasks, BS, device=DEV, weight_rows=rows)
    for layer in layers:
        layer(randn(gen, 330, H, D).to(DEV), randn(gen, 330, HK, D).to(DEV), randn(gen, 330, HK, D).to(DEV))
    spare = list(range(3, 12))
    for step in range(6):
        for t in tasks:
            _next(t, spare)
        runner.prepare_decode_context(tasks, BS, device=DEV, weight_rows=rows)
        ctx = get_context()
        for i, layer in enumerate(layers):
            q, k, v = randn(gen, 2, H, D).to(DEV), randn(gen, 2, HK, D).to(DEV), randn(gen, 2, HK, D).to(DEV)
            kv2, w2 = kv[i].clone(), weights[i].clone()
            o = layer(q, k, v)
            o2 = decode_attention_weights(q, kv2[0], kv2[1], ctx.context_lens, ctx.block_tables, SCALE, w2, ctx.weight_rows,
                                          key=k, value=v, slot_mapping=ctx.slot_mapping)
            assert torch.equal(o.reshape(o2.shape), o2) and torch.equal(kv[i], kv2)
            assert torch.equal(weights[i].view(torch.int32), w2.view(torch.int32))
            for t, r in zip(tasks, rows):
                assert weights[i, r, :, :t.seq_length].isfinite().all() and weights[i, r, :, t.seq_length].isnan().all() \
                    or step > 3
        if step == 3:
            lens = [t.seq_length for t in tasks]
            tables = [tasks[0].block_table, tasks[1].block_table + [-1]]
            new, left = evict_kv_tokens(kv, weights, _i32(tables), _i32(lens), 100, recent=20, sinks=4, weight_rows=_i32(rows))
            assert left.tolist() == [100, lens[1]]
            tasks[0].block_table, tasks[0].seq_length = [b for b in new[0].tolist() if b >= 0], 100


def test_a_chunk_over_what_an_eviction_left_in_a_4_bit_cache():
    """A prompt, an eviction, a chunk and a mixed step behind it through the module: as the calls over the same cache."""
    gen = torch.Generator().manual_seed(8)
    layer = Attention(H, D, SCALE, HK)
    kv = runner.allocate_kv_cache([layer], 12, BS, dtype=getattr(torch, "float4_e2m1fn_x2", torch.uint8), device=DEV)
    weights = runner.allocate_key_weights([layer], 5, 1024, device=DEV)
    rows = lambda n: (randn(gen, n, H, D).to(DEV), randn(gen, n, HK, D).to(DEV), randn(gen, n, HK, D).to(DEV))  # noqa: E731
    runner.prepare_prefill_context([runner.RunnerTask([0, 1, 2], 700, 0)], BS, device=DEV, weight_rows=[2])
    layer(*rows(700))
    new, left = evict_kv_tokens(kv, weights, _i32([[0, 1, 2]]), _i32([700]), 300, recent=50, sinks=4, weight_rows=_i32([2]))
    assert new.tolist() == [[0, 1, -1]] and left.tolist() == [300]
    steps = [([runner.RunnerTask([0, 1], 380, 300)], [2]),
             ([runner.RunnerTask([0, 1], 381, 380)] + [runner.RunnerTask([3 + i], 1, 0) for i in range(6)] +
              [runner.RunnerTask([9], 60, 0)], [2, 0, 1, -1, -1, -1, -1, 4])]
    for tasks, where in steps:
        runner.prepare_prefill_context(tasks, BS, device=DEV, weight_rows=where, evicted=[400] + [0] * (len(tasks) - 1),
                                       graphs=True)
        ctx, (q, k, v) = get_context(), rows(sum(t.seq_length - t.num_cached_tokens for t in tasks))
        kv2, w2 = kv[0].clone(), weights[0].clone()
        o = layer(q, k, v)
        ops.store_kvcache(k, v, kv2[0], kv2[1], ctx.slot_mapping)
        o2 = varlen_attention_weights(q, None, None, w2, ctx.weight_rows, cu_seqlens_q=ctx.cu_seqlens_q,
                                      cu_seqlens_k=ctx.cu_seqlens_k, max_seqlen_q=ctx.max_seqlen_q,
                                      max_seqlen_k=ctx.max_seqlen_k, softmax_scale=SCALE, block_table=ctx.block_tables,
                                      k_cache=kv2[0], v_cache=kv2[1])
        assert torch.equal(o.reshape(o2.shape), o2) and torch.equal(kv[0], kv2) and torch.equal(weights[0], w2)
        assert o2.isfinite().all() and weights[0, 2, :, :380].isfinite().all() and (weights[0, 2, :, 300:380] > 0).all()
