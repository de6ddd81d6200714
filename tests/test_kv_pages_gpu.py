"""GPU parity of forking, compacting and copying a paged cache's blocks against the oracle: bit-exact, bf16 and 4-bit."""

from __future__ import annotations

import pytest
import torch

from oracle import kvpages
from voxcpm2_arabic_dialects_turbo_amd.kernels.kv_copy import copy_kv_block_prefix
from voxcpm2_arabic_dialects_turbo_amd.kernels.kv_pages import compact_kv_blocks, fork_kv_blocks

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _kv(gen, layers, blocks, bs, hk, fp4):
    if fp4:
        return torch.randint(0, 256, (layers, 2, blocks, bs, hk, 68), generator=gen, dtype=torch.uint8)
    return torch.randn(layers, 2, blocks, bs, hk, 128, generator=gen).to(torch.bfloat16)


def _int(rows):
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def _same(got, want):
    assert torch.equal(got.cpu(), torch.tensor(want, dtype=torch.int32).view(got.shape))


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("bs,hk", [(256, 2), (64, 1), (64, 3)])
def test_fork(fp4, bs, hk):
    """Full, partial, empty, single-token and over-long parents; one forked several times; parents and blocks that are
    none; unused new blocks."""
    gen = torch.Generator().manual_seed(bs + hk)
    kv = _kv(gen, 3, 20, bs, hk, fp4)
    tables = [[3, 9, 1], [4, -1, 7], [0, 2, 5], [6, -1, 99]]
    lens = [2 * bs + 17, bs, 9 * bs, 1]
    parents = [0, 1, 0, 2, 3, -1, 4, 0, 0]
    fresh = [10, 11, 12, 13, 14, 15, 16, 25, -1]
    d = kv.to(DEV)
    t, n = fork_kv_blocks(d, _int(tables), _int(lens), _int(parents), _int(fresh))
    want_t, want_n = kvpages.fork(kv, tables, lens, parents, fresh)
    _same(t, want_t)
    _same(n, want_n)
    assert torch.equal(d.cpu(), kv)


@pytest.mark.parametrize("fp4", [False, True])
def test_fork_of_a_block_that_is_not_in_the_cache_leaves_no_entry(fp4):
    kv = _kv(torch.Generator().manual_seed(1), 1, 4, 64, 1, fp4)
    d = kv.to(DEV)
    t, n = fork_kv_blocks(d, _int([[1, -1], [1, 7]]), _int([70, 70]), _int([0, 1]), _int([2, 3]))
    _same(t, [[1, -1], [1, -1]])
    _same(n, [70, 70])
    assert torch.equal(d.cpu(), kv)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("blocks,batch,hi,layers", [(40, 6, 1000, 2), (1, 1, 256, 1), (33, 12, 256, 1), (64, 3, 200, 3),
                                                    (2000, 60, 900, 1), (5000, 400, 700, 1)])
def test_compact(fp4, blocks, batch, hi, layers):
    gen = torch.Generator().manual_seed(blocks + batch)
    bs, hk = (256, 1) if blocks < 100 else (64, 1)
    kv = _kv(gen, layers, blocks, bs, hk, fp4) if blocks < 100 or fp4 else \
        torch.randn(layers, 2, blocks, bs, hk, 8, generator=gen).to(torch.bfloat16)
    width = -(-hi // bs) + 1
    lens = torch.randint(0, hi + 1, (batch,), generator=gen).tolist()
    perm = torch.randperm(blocks, generator=gen).tolist()
    tables, at = [], 0
    for n in lens:
        need = -(-n // bs)
        row = [perm[(at + i) % blocks] for i in range(need)]  # (a small pool: blocks shared by rows)
        at += need
        tables.append(row + [0] * (width - need))  # stale entries past the context name blocks, too
    d = kv.to(DEV)
    t, remap, live = compact_kv_blocks(d, _int(tables), _int(lens))
    want_t, want_r, want_n = kvpages.compact(kv, tables, lens)
    _same(t, want_t)
    _same(remap, want_r)
    _same(live, [want_n])
    assert torch.equal(d.cpu(), kv)
    # compacted: nothing moves any more
    t2, remap2, live2 = compact_kv_blocks(d, t, _int(lens))
    assert torch.equal(t2, t) and int(live2) == want_n and torch.equal(d.cpu(), kv)
    _same(remap2, [b if b < want_n else -1 for b in range(blocks)])


@pytest.mark.parametrize("fp4", [False, True])
def test_compact_of_nothing_and_of_everything(fp4):
    kv = _kv(torch.Generator().manual_seed(2), 2, 6, 64, 1, fp4)
    d = kv.to(DEV)
    t, remap, live = compact_kv_blocks(d, _int([[1, 2], [3, 4]]), _int([0, 0]))
    _same(t, [[-1, -1], [-1, -1]])
    _same(remap, [-1] * 6)
    assert int(live) == 0
    t, remap, live = compact_kv_blocks(d, torch.empty(0, 2, dtype=torch.int32, device=DEV), _int([]))
    assert t.shape == (0, 2) and int(live) == 0
    t, remap, live = compact_kv_blocks(d, _int([[5, 1, 3], [0, 2, 4]]), _int([192, 192]))
    _same(t, [[5, 1, 3], [0, 2, 4]])
    assert int(live) == 6 and torch.equal(d.cpu(), kv)
    t, remap, live = compact_kv_blocks(d, _int([[5, -1, 9], [5, 5, 77]]), _int([192, 100]))  # entries that are no blocks
    kvpages.compact(kv, [[5, -1, 9], [5, 5, 77]], [192, 100])
    _same(t, [[0, -1, 9], [0, 0, -1]])
    _same(remap, [-1] * 5 + [0])
    assert int(live) == 1 and torch.equal(d.cpu(), kv)


def test_compact_of_the_most_blocks():
    """Live blocks at the end of a cache of 2^18 blocks, whose bitmap is the largest the plan takes."""
    blocks = 1 << 18
    bits = torch.arange(2 * blocks * 8).to(torch.int16).view(1, 2, blocks, 1, 1, 8)
    d = bits.view(torch.bfloat16).to(DEV)
    t, remap, live = compact_kv_blocks(d, _int([[blocks - 1, 7, blocks - 2], [1, blocks // 2, -1]]), _int([3, 2]))
    _same(t, [[4, 0, 3], [1, 2, -1]])
    _same(live, [5])
    new = {1: 1, 7: 0, blocks // 2: 2, blocks - 2: 3, blocks - 1: 4}
    want = torch.full((blocks,), -1, dtype=torch.int32)
    for a, b in new.items():
        want[a] = b
        bits[:, :, b] = bits[:, :, a]
    assert torch.equal(remap.cpu(), want)
    assert torch.equal(d.cpu().view(torch.int16), bits)


def test_fork_from_no_rows():
    """Every parent is outside a batch of none: empty children."""
    kv = torch.zeros(1, 2, 4, 64, 1, 68, dtype=torch.uint8, device=DEV)
    tables, lens = fork_kv_blocks(kv, torch.empty(0, 3, dtype=torch.int32, device=DEV),
                                  torch.empty(0, dtype=torch.int32, device=DEV), _int([0, 5]), _int([1, 2]))
    _same(tables, [[-1, -1, -1], [-1, -1, -1]])
    _same(lens, [0, 0])


def test_copy_block_prefix_of_a_4_bit_cache():
    kv = _kv(torch.Generator().manual_seed(3), 5, 12, 256, 2, True)
    d = kv.to(DEV)
    entries = [(3, 10, 50), (5, 7, 256), (0, 11, 300), (1, 2, 0), (4, 6, 1), (8, 9, 255)]
    copy_kv_block_prefix(d, entries)
    for src, dst, n in entries:
        if n > 0:
            kvpages.copy_slots(kv, src, dst, min(n, 256))
    assert torch.equal(d.cpu(), kv)


def test_fork_and_compact_in_a_graph():
    gen = torch.Generator().manual_seed(4)
    kv = _kv(gen, 4, 30, 256, 2, False)
    tables, lens, parents, fresh = [[20, 21, 22], [25, 26, 27]], [600, 700], [1, 0, 1], [2, 3, 4]
    d, t, n, p, f = kv.to(DEV), _int(tables), _int(lens), _int(parents), _int(fresh)

    def step():
        ct, cn = fork_kv_blocks(d, t, n, p, f)
        return ct, cn, *compact_kv_blocks(d, torch.cat((t, ct)), torch.cat((n, cn)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        d.copy_(kv)
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        host = kv.clone()
        ct, cn = kvpages.fork(host, tables, lens, parents, fresh)
        nt, remap, live = kvpages.compact(host, tables + ct, lens + cn)
        for got, want in zip(outs, (ct, cn, nt, remap, [live])):
            _same(got, want)
        assert torch.equal(d.cpu(), host)
