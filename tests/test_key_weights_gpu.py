"""GPU parity of attention that adds up what every key receives, and of eviction by it, against the float64 oracle.

Tolerances. Weights (fp32): with S the largest sum |q_d k_d| scale of a row, a score is off by at most 128 roundings of its
128 products' running sum and four more (scale, its log2 form, the fma, the exponent's argument): 132 2^-24 S. A probability
takes its own score's and the row's lse's, and the row's sum of n terms and the exponentials round n + 8 times:
2 132 2^-24 S + (n + 8) 2^-24, relative. A weight that adds up c of them and what it held rounds c + 1 times more. Outputs
(bf16): every probability is rounded to bf16 beside its value (2^-8 of sum p |v|), the output once (2^-8), plus the fp32
terms. Eviction is exact."""

from __future__ import annotations

import pytest
import torch

from oracle import fp4
from oracle import key_weights as ref
from tests._util import paged_pool, randn
from voxcpm2_arabic_dialects_turbo_amd.kernels.kv_evict import evict_kv_tokens
from voxcpm2_arabic_dialects_turbo_amd.ops import decode_attention, varlen_attention
from voxcpm2_arabic_dialects_turbo_amd.ops_weights import decode_attention_weights, varlen_attention_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
SCALE = D ** -0.5
U = 2.0 ** -24


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _p_tolerance(size, n):
    """Relative, of one row block's probabilities: size [H, rows, keys]."""
    return 264 * U * float(size.max()) + (n + 8) * U if size.numel() else 0.0


class Want:
    """The oracle's outputs and weights of a call, and how far from them the kernels' may be."""

    def __init__(self, weights):
        self.w, self.tol = weights.double(), torch.zeros_like(weights, dtype=torch.float64)
        self.o, self.otol = [], []

    def sequence(self, q, k, v, counts, row, new, scale=SCALE, more=0.0):
        o, p, pv, size = ref.attend(q, k, v, scale, counts)
        rel = _p_tolerance(size, k.shape[0]) + more
        self.o.append(o)
        self.otol.append((2 ** -8 + 2 * rel) * pv + 2 ** -8 * (o.abs() + 2 ** -8 * pv) + 1e-30)
        if row is not None and 0 <= row < self.w.shape[0] and q.shape[0]:
            m, group = k.shape[0], q.shape[1] // k.shape[1]
            before = self.w[row].clone()
            ref.add(self.w[row], p, new)
            before[:, max(m - new, 0):] = 0  # (a new token's weight does not add to what its place held)
            got = self.w[row][:, :m].abs() + before[:, :m].abs()
            self.tol[row][:, :m] = (rel + (q.shape[0] * group + 2) * U) * got + 1e-35

    def check(self, o, weights):
        want, tol = torch.cat(self.o), torch.cat(self.otol)
        o, weights = o.cpu().double(), weights.cpu().double()
        assert o.isfinite().all()
        off = (o - want).abs() - tol
        assert (off <= 0).all(), f"output over its tolerance by {off.max():.3g}"
        off = (weights - self.w).abs() - self.tol
        bad = ~(off <= 0) & ~(weights.isnan() & self.w.isnan())
        assert not bad.any(), f"{int(bad.sum())} weights off, first at {bad.nonzero()[0].tolist()}: by {off[bad].max():.3g}"


def _received(gen, rows, hk, width):
    return torch.rand(rows, hk, width, generator=gen) * 3


# ----------------------------------------------------------------------------------------------------------------------
# decode


def _decode_case(seed, lens, h, hk, bs, rows=None, store=False, extra_cols=0, spare=2, drop=()):
    """Runs one decode call and checks it. rows: None or the rows' numbers; drop: (sequence, column) entries set to -1."""
    gen = torch.Generator().manual_seed(seed)
    B = len(lens)
    kc, vc, tables = paged_pool(gen, lens, sum(-(-n // bs) for n in lens) + spare, bs, hk, extra_cols=extra_cols)
    for b, c in drop:
        tables[b, c] = -1
    width = tables.shape[1] * bs + 64
    n_rows = B if rows is None else max([*rows, 0]) + 2
    w = _received(gen, n_rows, hk, width)
    q = randn(gen, B, h, D)
    key, value = randn(gen, B, hk, D), randn(gen, B, hk, D)
    # what no context reaches may hold anything: NaN in the caches and in the weights of new tokens
    flat_k, flat_v = kc.view(-1, hk, D), vc.view(-1, hk, D)
    live = torch.zeros(kc.shape[0] * bs, dtype=torch.bool)
    slots = []
    for b, n in enumerate(lens):
        at = [int(tables[b, j // bs]) * bs + j % bs if tables[b, j // bs] >= 0 else -1 for j in range(n)]
        live[[s for s in at if s >= 0]] = True
        slots.append(at[-1] if at else -1)
        r = b if rows is None else rows[b]
        if n and 0 <= r < n_rows:
            w[r, :, n - 1] = float("nan")
    flat_k[~live], flat_v[~live] = float("nan"), float("inf")
    args = [t.to(DEV) for t in (q, kc, vc)]
    wd = w.to(DEV)
    kw = dict(weight_rows=None if rows is None else _i32(rows))
    if store:
        kw.update(key=key.to(DEV), value=value.to(DEV), slot_mapping=_i32(slots))
    o = decode_attention_weights(*args, _i32(lens), tables.to(DEV), SCALE, wd, **kw)
    if store:
        for b, s in enumerate(slots):
            if s >= 0:
                flat_k[s], flat_v[s] = key[b], value[b]
        assert torch.equal(args[1].cpu().view(torch.int16), kc.view(torch.int16))
        assert torch.equal(args[2].cpu().view(torch.int16), vc.view(torch.int16))
    want = Want(w)
    for b, n in enumerate(lens):
        r = b if rows is None else rows[b]
        if n == 0:
            want.o.append(torch.zeros(1, h, D, dtype=torch.float64))
            want.otol.append(torch.zeros(1, h, D, dtype=torch.float64))
            continue
        k, ok = ref.keys_of(kc, tables[b], n)
        v, _ = ref.keys_of(vc, tables[b], n)
        want.sequence(q[b:b + 1], k, v, ok, r, 1)
    want.check(o, wd)
    return args, wd, o


@pytest.mark.parametrize("store", [False, True])
@pytest.mark.parametrize("h,hk,bs", [(16, 2, 256), (8, 1, 256), (4, 2, 64), (16, 1, 128), (6, 2, 96), (3, 1, 32), (2, 2, 256)])
def test_decode_lengths(h, hk, bs, store):
    """Lengths around the 16-token steps and the blocks, empty rows among them, in rows of any order."""
    lens = [1, 0, 15, 16, 17, 31, 33, 0, 95, 97, 255, 256, 257, 300, 511, 513, 0]
    gen = torch.Generator().manual_seed(h)
    rows = torch.randperm(len(lens) + 5, generator=gen)[:len(lens)].tolist()
    _decode_case(10 * h + hk + store, lens, h, hk, bs, rows, store)


@pytest.mark.parametrize("lens,h,hk", [([1], 16, 2), ([420], 16, 2), ([4099], 8, 1), ([33000], 16, 2), ([2, 9000, 5], 16, 2),
                                       ([40 + 13 * (i % 50) for i in range(150)], 16, 2), ([5] * 65, 4, 2),
                                       ([1 + i % 70 for i in range(700)], 8, 1)])
def test_decode_batches(lens, h, hk):
    """One short and one long sequence, batches past one lane a sequence (64) and past one launch (512)."""
    _decode_case(len(lens), lens, h, hk, 256)


def test_decode_rows_that_are_none_keep_none():
    """Rows -1 and past the last, and a wide table whose columns behind the contexts name nothing."""
    _decode_case(3, [40, 70, 300, 20, 600], 16, 2, 64, [3, -1, 1, 99, 0], extra_cols=7)


def test_decode_blocks_that_are_none_take_no_weight():
    """A block in the middle, and every block of a sequence: its output is zeros, its tokens get nothing."""
    _decode_case(4, [300, 200, 130], 16, 2, 64, drop=[(0, 1), (0, 2), (1, 0), (1, 1), (1, 2), (1, 3), (2, 2)])


def test_decode_output_is_that_of_decode_attention():
    for lens in ([420], [100 + 31 * i for i in range(40)], [256 + 11 * (i % 160) for i in range(150)]):
        (q, kc, vc), w, o = _decode_case(5, lens, 16, 2, 256)
        kc, vc = (torch.nan_to_num(x, 0.0, 0.0) for x in (kc, vc))
        gen = torch.Generator().manual_seed(5)
        _, _, tables = paged_pool(gen, lens, sum(-(-n // 256) for n in lens) + 2, 256, 2)
        assert torch.equal(o, decode_attention(q, kc, vc, _i32(lens), tables.to(DEV), SCALE))


@pytest.mark.parametrize("rides", [False, True])
def test_decode_rows_of_any_layout(rides):
    """Strided and expanded queries and new rows, and ones that 16-byte loads cannot take."""
    gen = torch.Generator().manual_seed(6)
    lens, hk, h = [70, 1, 300], 2, 16
    kc, vc, tables = paged_pool(gen, lens, 8, 64, hk)
    qkv = randn(gen, 3, (h + 2 * hk) * D + (8 if rides else 4))
    off = 0 if rides else 4
    q = randn(gen, 1, h, D).expand(3, h, D)
    key = qkv[:, off + h * D:off + (h + hk) * D].view(3, hk, D)
    value = qkv[:, off + (h + hk) * D:off + (h + 2 * hk) * D].view(3, hk, D)
    slots = [int(tables[b, (n - 1) // 64]) * 64 + (n - 1) % 64 for b, n in enumerate(lens)]
    qd, base = q[:1].to(DEV).expand(3, h, D), qkv.to(DEV)
    kd = base[:, off + h * D:off + (h + hk) * D].view(3, hk, D)
    vd = base[:, off + (h + hk) * D:off + (h + 2 * hk) * D].view(3, hk, D)
    w = _received(gen, 3, hk, tables.shape[1] * 64)
    wd, kcd, vcd = w.to(DEV), kc.to(DEV), vc.to(DEV)
    o = decode_attention_weights(qd, kcd, vcd, _i32(lens), tables.to(DEV).long(), SCALE, wd, key=kd, value=vd,
                                 slot_mapping=_i32(slots).long())
    kc.view(-1, hk, D)[slots], vc.view(-1, hk, D)[slots] = key, value
    assert torch.equal(kcd.cpu(), kc) and torch.equal(vcd.cpu(), vc)
    want = Want(w)
    for b, n in enumerate(lens):
        want.sequence(q[b:b + 1], ref.keys_of(kc, tables[b], n)[0], ref.keys_of(vc, tables[b], n)[0], None, b, 1)
    want.check(o, wd)


def test_decode_is_the_same_every_time():
    (q, kc, vc), w, o = _decode_case(7, [1500, 3, 700, 256], 16, 2, 256)
    gen = torch.Generator().manual_seed(7)
    _, _, tables = paged_pool(gen, [1500, 3, 700, 256], 13, 256, 2)
    first = torch.zeros_like(w)
    for _ in range(4):
        again = torch.zeros_like(w)
        o2 = decode_attention_weights(q, kc, vc, _i32([1500, 3, 700, 256]), tables.to(DEV), SCALE, again)
        first = again if not first.any() else first
        assert torch.equal(o2, o) and torch.equal(first, again)


# ----------------------------------------------------------------------------------------------------------------------
# chunks


def _varlen_case(seed, seqs, h, hk, bs=None, rows=None, extra_cols=0, drop=(), max_k=None, poison=True):
    """seqs: (queries, keys) of each; bs: cache blocks, None: packed rows."""
    gen = torch.Generator().manual_seed(seed)
    B, lens = len(seqs), [m for _, m in seqs]
    T, cu_q, cu_k = sum(n for n, _ in seqs), [0], [0]
    for n, m in seqs:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    q = randn(gen, T, h, D)
    max_k = max(lens) if max_k is None else max_k
    n_rows = B if rows is None else max([*rows, 0]) + 2
    width = (max(max_k, 1) + 255) // 256 * 256 + 256 * (extra_cols + 1)
    w = _received(gen, n_rows, hk, width)
    kw = dict(cu_seqlens_q=_i32(cu_q), cu_seqlens_k=_i32(cu_k), max_seqlen_q=max(n for n, _ in seqs), max_seqlen_k=max_k,
              softmax_scale=SCALE)
    for b, (n, m) in enumerate(seqs):  # a new token's place may hold anything
        r = b if rows is None else rows[b]
        if n and 0 <= r < n_rows:
            w[r, :, max(m - n, 0):m] = float("nan")
    if bs is None:
        k, v = randn(gen, cu_k[-1], hk, D), randn(gen, cu_k[-1], hk, D)
        keys = [(k[cu_k[b]:cu_k[b + 1]], v[cu_k[b]:cu_k[b + 1]], None) for b in range(B)]
        kd, vd = k.to(DEV), v.to(DEV)
    else:
        kc, vc, tables = paged_pool(gen, lens, sum(-(-n // bs) for n in lens) + 2, bs, hk, extra_cols=extra_cols)
        for b, c in drop:
            tables[b, c] = -1
        if poison:
            live = torch.zeros(kc.shape[0] * bs, dtype=torch.bool)
            for b, n in enumerate(lens):
                at = [int(tables[b, j // bs]) * bs + j % bs for j in range(n) if tables[b, j // bs] >= 0]
                live[at] = True
            kc.view(-1, hk, D)[~live], vc.view(-1, hk, D)[~live] = float("nan"), float("nan")
        keys = [(*(ref.keys_of(c, tables[b], n)[0] for c in (kc, vc)), ref.keys_of(kc, tables[b], n)[1])
                for b, n in enumerate(lens)]
        kd = vd = None
        kw.update(block_table=tables.to(DEV), k_cache=kc.to(DEV), v_cache=vc.to(DEV))
    wd = w.to(DEV)
    o = varlen_attention_weights(q.to(DEV), kd, vd, wd, None if rows is None else _i32(rows), **kw)
    want = Want(w)
    for b, (n, m) in enumerate(seqs):
        want.sequence(q[cu_q[b]:cu_q[b + 1]], *keys[b], b if rows is None else rows[b], n)
    want.check(o, wd)
    return q, kd, vd, kw, o


HEADS = [(16, 2), (8, 1), (4, 4), (8, 8), (32, 4), (16, 1), (32, 1), (64, 1)]


@pytest.mark.parametrize("h,hk", HEADS)
def test_packed_prompts(h, hk):
    """Prompts around the 32-, 64- and 128-row tiles, an empty one among them."""
    _varlen_case(h, [(n, n) for n in (1, 2, 0, 7, 31, 33, 64, 65, 129, 200)], h, hk)


@pytest.mark.parametrize("h,hk", HEADS)
@pytest.mark.parametrize("bs", [64, 256, 192])
def test_chunks_over_cached_prefixes(h, hk, bs):
    """Chunks over prefixes of none to several blocks, one-query rows, a sequence without queries, one with fewer keys than
    queries (its first rows see no key), and rows of any order, one of them none."""
    seqs = [(5, 55), (1, 1), (1, 300), (0, 130), (33, 33), (64, 257), (17, 11), (100, 420), (3, 64)]
    gen = torch.Generator().manual_seed(h + bs)
    rows = torch.randperm(len(seqs) + 3, generator=gen)[:len(seqs)].tolist()
    rows[1] = -1
    _varlen_case(h + hk + bs, seqs, h, hk, bs, rows, extra_cols=2)


@pytest.mark.parametrize("seqs,bs", [([(900, 900), (237, 237)], None), ([(700, 2300), (1, 1801)], 256), ([(1, 1)], 64),
                                     ([(1, 2)], None), ([(44, 94)] * 44, 256), ([(1100, 1100)] * 3 + [(513, 700)], 64)])
def test_chunk_sizes(seqs, bs):
    _varlen_case(len(seqs), seqs, 16, 2, bs)


def test_chunk_blocks_that_are_none_take_no_weight():
    _varlen_case(11, [(40, 300), (30, 200), (5, 130)], 16, 2, 64,
                 drop=[(0, 1), (0, 2), (1, 0), (1, 1), (1, 2), (1, 3), (2, 2)], rows=[2, 0, 1])


def test_chunk_wide_tables():
    """More columns than a wave has lanes."""
    _varlen_case(12, [(20, 64 * 70 + 5), (3, 9)], 8, 1, 64)


def test_chunk_output_is_that_of_varlen_attention():
    """To the rounding of either (the two may walk the keys in different orders)."""
    q, k, v, kw, o = _varlen_case(13, [(300, 300), (70, 70)], 16, 2)
    want = varlen_attention(q.to(DEV), k, v, cu_seqlens_q=kw["cu_seqlens_q"], cu_seqlens_k=kw["cu_seqlens_k"],
                            max_seqlen_q=300, softmax_scale=SCALE, causal=True)
    assert (o.float() - want.float()).abs().max() <= 2 ** -6 * want.float().abs().max()


def test_chunk_rows_of_any_layout():
    """Queries and packed keys as views of one projection, into a strided output; int64 index tensors."""
    gen = torch.Generator().manual_seed(14)
    h, hk, seqs = 16, 2, [(70, 70), (9, 9)]
    T = 79
    x = randn(gen, T, (h + 2 * hk) * D)
    q, k, v = x[:, :h * D].view(T, h, D), x[:, h * D:(h + hk) * D].view(T, hk, D), x[:, (h + hk) * D:].view(T, hk, D)
    xd = x.to(DEV)
    w = _received(gen, 2, hk, 128)
    wd = w.to(DEV)
    out = torch.zeros(T, h * D + 64, dtype=torch.bfloat16, device=DEV)[:, :h * D].view(T, h, D)
    cu = torch.tensor([0, 70, 79], device=DEV)
    o = varlen_attention_weights(xd[:, :h * D].view(T, h, D), xd[:, h * D:(h + hk) * D].view(T, hk, D),
                                 xd[:, (h + hk) * D:].view(T, hk, D), wd, torch.tensor([1, 0], device=DEV), cu_seqlens_q=cu,
                                 cu_seqlens_k=cu, max_seqlen_q=70, max_seqlen_k=70, softmax_scale=SCALE, out=out)
    assert o is out
    want = Want(w)
    for b, (a, e) in enumerate([(0, 70), (70, 79)]):
        want.sequence(q[a:e], k[a:e], v[a:e], None, 1 - b, e - a)
    want.check(o, wd)


def test_weights_of_a_chunk_are_those_of_its_tokens_one_by_one():
    """A prompt in one call, in two chunks, and token by token through the cache: the same weights, to rounding."""
    gen = torch.Generator().manual_seed(15)
    h, hk, bs, n = 16, 2, 64, 150
    kc, vc, tables = paged_pool(gen, [n], 4, bs, hk)
    q = randn(gen, n, h, D)
    qd, kcd, vcd, td = q.to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV)
    width = tables.shape[1] * bs

    def chunks(*ends):
        w, a = torch.full((1, hk, width), float("nan"), device=DEV), 0
        for e in ends:
            varlen_attention_weights(qd[a:e], None, None, w, cu_seqlens_q=_i32([0, e - a]), cu_seqlens_k=_i32([0, e]),
                                     max_seqlen_q=e - a, max_seqlen_k=e, softmax_scale=SCALE, block_table=td, k_cache=kcd,
                                     v_cache=vcd)
            a = e
        return w[..., :n].double().cpu()

    whole = chunks(n)
    steps = torch.full((1, hk, width), float("nan"), device=DEV)
    for e in range(1, n + 1):
        decode_attention_weights(qd[e - 1:e], kcd, vcd, _i32([e]), td, SCALE, steps)
    want = Want(torch.zeros(1, hk, width))
    want.sequence(q, ref.keys_of(kc, tables[0], n)[0], ref.keys_of(vc, tables[0], n)[0], None, 0, n)
    tol = want.tol[..., :n]
    for got in (whole, chunks(64, n), chunks(1, 65, 100, n), steps[..., :n].double().cpu()):
        assert ((got - want.w[..., :n]).abs() <= tol).all()
    assert (whole.sum(-1) - n * h / hk).abs().max() <= tol.sum(-1).max()


# ----------------------------------------------------------------------------------------------------------------------
# eviction


def _kv(gen, layers, blocks, bs, hk, kind):
    if kind == "fp4":
        return torch.randint(0, 256, (layers, 2, blocks, bs, hk, 68), generator=gen, dtype=torch.uint8)
    return torch.randn(layers, 2, blocks, bs, hk, 64 if kind == "narrow" else 128, generator=gen).to(torch.bfloat16)


def _tables(gen, lens, blocks, bs, cols):
    perm, at, out = torch.randperm(blocks, generator=gen).tolist(), 0, []
    for n in lens:
        need = min(-(-n // bs), cols)
        out.append(perm[at:at + need] + [-1] * (cols - need))
        at += need
    assert at <= blocks
    return out, perm[at:]


def _evict_case(kv, weights, tables, lens, budget, sinks=0, recent=0, rows=None, new_blocks=None):
    kd, wd = kv.to(DEV), weights.to(DEV)
    t, n = evict_kv_tokens(kd, wd, _i32(tables), _i32(lens), budget, recent=recent, sinks=sinks,
                           weight_rows=None if rows is None else _i32(rows),
                           new_blocks=None if new_blocks is None else _i32(new_blocks))
    want_t, want_n = ref.evict(kv, weights, tables, lens, budget, sinks, recent, rows, new_blocks)
    assert t.tolist() == want_t and n.tolist() == want_n
    as_int = torch.int16 if kv.dtype == torch.bfloat16 else torch.uint8
    assert torch.equal(wd.cpu().view(torch.int32), weights.view(torch.int32))
    assert torch.equal(kd.cpu().view(as_int), kv.view(as_int))


@pytest.mark.parametrize("kind", ["bf16", "fp4", "narrow"])
@pytest.mark.parametrize("bs,hk", [(256, 2), (64, 1), (64, 3)])
@pytest.mark.parametrize("budget,sinks,recent", [(100, 4, 30), (64, 0, 0), (257, 3, 254), (1, 0, 0), (1, 1, 0), (300, 0, 299)])
def test_evict(kind, bs, hk, budget, sinks, recent):
    """Lengths around the budget, empty ones, one past the tables' reach; weights with many ties."""
    gen = torch.Generator().manual_seed(bs + hk + budget)
    lens, cols = [budget - 1, budget, budget + 1, 0, 2 * budget + 7, 700, 9999], -(-800 // bs)
    tables, _ = _tables(gen, [min(n, 800) for n in lens], sum(min(-(-min(n, 800) // bs), cols) for n in lens) + 3, bs, cols)
    weights = torch.floor(torch.rand(2, 9, hk, cols * bs + 8, generator=gen) ** 3 * 40) / 8
    rows = torch.randperm(9, generator=gen)[:7].tolist()
    kv = _kv(gen, 2, max(max(r) for r in tables) + 2, bs, hk, kind)
    _evict_case(kv, weights, tables, lens, budget, sinks, recent, rows)


def test_evict_by_any_weights():
    """Infinities, NaN of both signs, both zeros, negative and subnormal numbers, all equal, in order either way."""
    gen = torch.Generator().manual_seed(20)
    n, bs = 400, 64
    inf, nan = float("inf"), float("nan")
    special = torch.tensor([inf, -inf, nan, -nan, 0.0, -0.0, 1e-40, -1e-40, 2e-40, 1.0, -1.0, 3.4e38, -3.4e38])
    rows = [special[torch.randint(0, 13, (448,), generator=gen)], torch.zeros(448), torch.arange(448.0),
            -torch.arange(448.0), torch.randn(448, generator=gen), torch.where(torch.rand(448, generator=gen) < 0.5, 0.0, -0.0),
            torch.full((448,), nan), 1 + torch.randint(0, 3, (448,), generator=gen) * 2.0 ** -23]
    weights = torch.stack(rows)[None, :, None].contiguous()
    lens = [n] * len(rows)
    tables, _ = _tables(gen, lens, 60, bs, 7)
    for budget, sinks, recent in ((100, 0, 0), (200, 5, 64), (399, 0, 1)):
        _evict_case(_kv(gen, 1, 60, bs, 1, "bf16"), weights.clone(), tables, lens, budget, sinks, recent)


@pytest.mark.parametrize("n,budget", [(33000, 8000), (2049, 2047), (8193, 1), (5000, 4096)])
def test_evict_long(n, budget):
    gen = torch.Generator().manual_seed(n)
    cols = -(-n // 256)
    tables, _ = _tables(gen, [n], cols + 1, 256, cols)
    weights = torch.floor(torch.rand(1, 1, 1, cols * 256, generator=gen) * 4096)
    _evict_case(_kv(gen, 1, cols + 1, 256, 1, "bf16"), weights, tables, [n], budget, 0, budget // 8)


def test_evict_leaves_rows_that_are_none():
    """Sequences whose row is outside the weights stay; tokens in blocks that are none, or whose new block is, do not move."""
    gen = torch.Generator().manual_seed(22)
    tables, lens = [[3, 0, 7], [1, 2, 5], [4, -1, 6], [8, 99, 9]], [180, 180, 180, 180]
    weights = torch.rand(2, 6, 2, 192, generator=gen)
    _evict_case(_kv(gen, 2, 10, 64, 2, "bf16"), weights, tables, lens, 100, 2, 20, [4, -1, 0, 2])
    _evict_case(_kv(gen, 2, 10, 64, 2, "bf16"), weights, tables, lens, 100, 2, 20, [7, 1, 6, -5])


@pytest.mark.parametrize("kind", ["bf16", "fp4"])
def test_evict_into_new_blocks(kind):
    """Two takes of one text share its blocks: each keeps its own choice in new blocks, the shared ones stay; a third, alone
    in its blocks, gets a new first block only."""
    gen = torch.Generator().manual_seed(23)
    tables = [[3, 0, 7, 2], [3, 0, 7, 5], [1, 4, 6, 8], [10, 9, -1, -1]]
    lens, new = [250, 256, 230, 90], [[11, 12, -1, -1], [13, 14, 19, -1], [15, -1, -1, -1], [16, 17, 18, -1]]
    for budget in (100, 64, 128):
        weights = torch.rand(2, 4, 2, 256, generator=gen)
        _evict_case(_kv(gen, 2, 20, 64, 2, kind), weights, tables, lens, budget, 2, 20, None, new)


def test_evict_nothing():
    kv, w = torch.zeros(1, 2, 4, 64, 1, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(1, 4, 1, 256, device=DEV)
    t, n = evict_kv_tokens(kv, w, _i32([[1, 2]])[:0], _i32([]), 10)
    assert t.shape == (0, 2) and n.shape == (0,)


# ----------------------------------------------------------------------------------------------------------------------
# steps that are mostly one-query rows


@pytest.mark.parametrize("h,hk,bs", [(16, 2, 256), (8, 1, 64), (4, 4, 64), (32, 2, 64)])
def test_chunk_mostly_one_query_rows(h, hk, bs):
    """On the decode kernels where they take the heads; sequences without queries and prompts among them, rows of any order."""
    seqs = [(1, 5 + 37 * i) for i in range(20)] + [(90, 90), (0, 50), (130, 400)] + [(1, 1), (1, 256)]
    gen = torch.Generator().manual_seed(h)
    rows = torch.randperm(len(seqs) + 3, generator=gen)[:len(seqs)].tolist()
    rows[3], rows[20] = -1, -1
    _varlen_case(30 + h, seqs, h, hk, bs, rows, extra_cols=1)


@pytest.mark.parametrize("bs", [64, None])
def test_chunk_more_sequences_than_a_launch_lays_out(bs):
    """More than 512 sequences, long ones behind the first 512."""
    _varlen_case(31, [(1 + i % 3, 1 + i % 3 + (i % 40 if bs else 0)) for i in range(700)] + [(100, 100), (1, 1)], 8, 1, bs)
    _varlen_case(32, [(1, 1 + (i % 70 if bs else 0)) for i in range(600)], 8, 1, bs)


def test_chunk_in_parts_of_its_rows():
    """Long prompts whose query rows are summed in several parts, over caches and packed, one past eight parts of 512 rows."""
    _varlen_case(33, [(700, 700), (65, 800), (64, 64)], 16, 2, 64)
    _varlen_case(34, [(600, 600), (130, 130)], 64, 1)
    _varlen_case(35, [(1300, 1300)], 8, 1)
    _varlen_case(36, [(2100, 2100)], 2, 2)


def test_evict_with_tables_wider_than_a_workgroup_holds():
    """Blocks of 16 tokens: 600 columns, with and without new blocks; a block size that is no power of two."""
    gen = torch.Generator().manual_seed(41)
    for bs, n, budget in ((16, 9500, 700), (48, 3000, 1111)):
        cols = -(-n // bs) + 5
        need = -(-n // bs)
        tables, rest = _tables(gen, [n, 40], need + 3 + -(-budget // bs) + 4, bs, cols)
        weights = torch.rand(1, 2, 2, cols * bs, generator=gen)
        kv = _kv(gen, 1, need + 3 + -(-budget // bs) + 4, bs, 2, "narrow")
        _evict_case(kv.clone(), weights.clone(), tables, [n, 40], budget, 3, 100)
        new = [rest[:-(-budget // bs)] + [-1] * (cols - -(-budget // bs)), [-1] * cols]
        _evict_case(kv, weights, tables, [n, 40], budget, 3, 100, None, new)


@pytest.mark.parametrize("bs", [64, None])
def test_chunk_lengths_past_what_the_call_says(bs):
    """Queries past max_seqlen_q and keys past max_seqlen_k are left out: the weights are those of the others, the places of
    keys that nothing saw as they were, and the memory around the scratch is not written."""
    gen = torch.Generator().manual_seed(51)
    h, hk, seqs, max_q, max_k = 16, 2, [(900, 900), (40, 40), (300, 500 if bs else 300)], 128, 400
    cu_q, cu_k = [0], [0]
    for n, m in seqs:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    q = randn(gen, cu_q[-1], h, D)
    w = _received(gen, 3, hk, 1024)
    wd = w.to(DEV)
    kw = dict(cu_seqlens_q=_i32(cu_q), cu_seqlens_k=_i32(cu_k), max_seqlen_q=max_q, max_seqlen_k=max_k, softmax_scale=SCALE)
    if bs:
        lens = [m for _, m in seqs]
        kc, vc, tables = paged_pool(gen, lens, 40, bs, hk)
        keys = [tuple(ref.keys_of(c, tables[b], m)[0] for c in (kc, vc)) for b, m in enumerate(lens)]
        kd = vd = None
        kw.update(block_table=tables.to(DEV), k_cache=kc.to(DEV), v_cache=vc.to(DEV))
    else:
        k, v = randn(gen, cu_k[-1], hk, D), randn(gen, cu_k[-1], hk, D)
        keys = [(k[cu_k[b]:cu_k[b + 1]], v[cu_k[b]:cu_k[b + 1]]) for b in range(3)]
        kd, vd = k.to(DEV), v.to(DEV)
    o = varlen_attention_weights(q.to(DEV), kd, vd, wd, **kw).cpu().double()
    want = Want(w)
    for b, (n, m) in enumerate(seqs):
        took, seen = min(n, max_q), m - n + min(n, max_q)
        before = want.w[b].clone()
        want.sequence(q[cu_q[b]:cu_q[b] + took], keys[b][0][:seen], keys[b][1][:seen], None, b, took)
        want.w[b][:, min(seen, max_k):] = before[:, min(seen, max_k):]
        assert ((o[cu_q[b]:cu_q[b] + took] - want.o[-1]).abs() <= want.otol[-1]).all()
    off = (wd.cpu().double() - want.w).abs() - want.tol
    assert (off <= 0).all()


def test_chunk_of_a_group_of_128():
    _varlen_case(52, [(70, 70), (3, 200), (1, 1)], 128, 1, 64)


def test_bounds_past_32_bits():
    """Budgets and numbers of queries that no sequence reaches, however large: nothing is dropped, nothing is left out."""
    gen = torch.Generator().manual_seed(53)
    for budget in (500, 2 ** 31, 2 ** 33 + 5):
        kv, w = _kv(gen, 1, 8, 64, 2, "bf16"), torch.rand(1, 2, 2, 256, generator=gen)
        _evict_case(kv, w, [[1, 2, 3, 0], [5, 6, -1, -1]], [256, 100], budget, 3, 90)
    _, k, v, kw, _ = _varlen_case(54, [(70, 70), (9, 9)], 16, 2)
    q, w = randn(gen, 79, 16, D).to(DEV), [torch.zeros(2, 2, 256, device=DEV) for _ in range(2)]
    for x, n in zip(w, (70, 2 ** 33 + 1)):
        o = varlen_attention_weights(q, k, v, x, **{**kw, "max_seqlen_q": n})
    assert torch.equal(*w) and w[0].any() and o.isfinite().all()


def test_caches_past_4_gib():
    """Planes of 4.7 GiB: blocks at both ends, in decode steps, chunks and evictions; and a long prefix."""
    gen = torch.Generator().manual_seed(55)
    n, bs, h, hk, cols = 36000, 256, 16, 2, 5
    lens, blocks = [1100, 300], [n - 1, 7, n - 2, 33000, 0, n - 3, 34001]
    small = _kv(gen, 1, 7, bs, hk, "bf16")  # (the blocks in this order)
    big = torch.empty(1, 2, n, bs, hk, D, dtype=torch.bfloat16, device=DEV)
    for i, at in enumerate(blocks):
        big[:, :, at] = small[:, :, i].to(DEV)
    near = torch.tensor([[0, 1, 2, 3, 4], [5, 6, -1, -1, -1]], dtype=torch.int32)
    far = torch.tensor([[blocks[i] if i >= 0 else -1 for i in row] for row in near.tolist()], dtype=torch.int32, device=DEV)
    q, w = randn(gen, 2, h, D), _received(gen, 2, hk, cols * bs)
    for chunk in (False, True):
        wd, want = w.to(DEV), Want(w)
        if chunk:
            qs = randn(gen, 60, h, D)
            o = varlen_attention_weights(qs.to(DEV), None, None, wd, cu_seqlens_q=_i32([0, 40, 60]), cu_seqlens_k=_i32([0, 1100, 1400]),
                                         max_seqlen_q=40, max_seqlen_k=1100, softmax_scale=SCALE, block_table=far,
                                         k_cache=big[0, 0], v_cache=big[0, 1])
            rows = [qs[:40], qs[40:]]
        else:
            o = decode_attention_weights(q.to(DEV), big[0, 0], big[0, 1], _i32(lens), far, SCALE, wd)
            rows = [q[:1], q[1:]]
        for b in range(2):
            k, v = (ref.keys_of(small[0, x], near[b], lens[b])[0] for x in (0, 1))
            want.sequence(rows[b], k, v, None, b, rows[b].shape[0])
        want.check(o, wd)
    weights = torch.rand(1, 2, hk, cols * bs, generator=gen)
    wd = weights.to(DEV)
    t, left = evict_kv_tokens(big, wd, far, _i32(lens), 260, recent=20, sinks=3)
    want_t, want_n = ref.evict(small, weights, near.tolist(), lens, 260, 3, 20, None, None)
    assert left.tolist() == want_n and t.tolist() == [[blocks[i] if i >= 0 else -1 for i in row] for row in want_t]
    assert torch.equal(wd.cpu(), weights)
    for i, at in enumerate(blocks):
        assert torch.equal(big[:, :, at].cpu(), small[:, :, i])


def test_chunk_behind_a_long_prefix():
    _varlen_case(56, [(40, 33000), (3, 9), (1, 20000)], 16, 2, 256)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_reaches_who_sees_it(bad):
    """A new token's key: the outputs of the queries before it and the weights of another sequence. Its value: no weight."""
    gen = torch.Generator().manual_seed(57)
    q, k, v = randn(gen, 130, 16, D).to(DEV), randn(gen, 130, 2, D).to(DEV), randn(gen, 130, 2, D).to(DEV)
    kw = dict(cu_seqlens_q=_i32([0, 100, 130]), cu_seqlens_k=_i32([0, 100, 130]), max_seqlen_q=100, max_seqlen_k=100,
              softmax_scale=SCALE)

    def run(k, v):
        w = torch.zeros(2, 2, 128, device=DEV)
        return varlen_attention_weights(q, k, v, w, **kw), w

    o, w = run(k, v)
    k2, v2 = k.clone(), v.clone()
    k2[99], v2[99] = bad, bad
    o2, w2 = run(k2, v)
    assert torch.equal(o2[:99], o[:99]) and torch.equal(o2[100:], o[100:]) and torch.equal(w2[1], w[1])
    assert w2[0, :, :100].isnan().all() and not w2[0, :, 100:].any() and o2[99].isnan().all()
    o3, w3 = run(k, v2)
    assert torch.equal(w3, w) and torch.equal(o3[100:], o[100:])


# ----------------------------------------------------------------------------------------------------------------------
# seeded random calls


def _draw(gen, lo, hi):
    return int(torch.randint(lo, hi + 1, (1,), generator=gen))


def _rows(gen, n):
    if _draw(gen, 0, 1):
        return None
    rows = torch.randperm(n + 4, generator=gen)[:n].tolist()
    return [-1 if _draw(gen, 0, 9) == 0 else r for r in rows]


@pytest.mark.parametrize("seed", range(16))
def test_random_decodes(seed):
    gen = torch.Generator().manual_seed(1000 + seed)
    h, hk = [(16, 2), (8, 1), (16, 1), (4, 2), (10, 2), (7, 1)][seed % 6]
    top = [40, 400, 1500][seed % 3]
    lens = [_draw(gen, 0, top) if _draw(gen, 0, 6) else 0 for _ in range(_draw(gen, 1, [180, 40, 12][seed % 3]))]
    _decode_case(1000 + seed, lens, h, hk, [256, 64, 32, 160][_draw(gen, 0, 3)], _rows(gen, len(lens)),
                 bool(_draw(gen, 0, 1)) and any(lens), extra_cols=_draw(gen, 0, 2))


@pytest.mark.parametrize("seed", range(32))
def test_random_chunks(seed):
    """Few rows and many, short keys and long: every form of the two launches."""
    gen = torch.Generator().manual_seed(2000 + seed)
    h, hk = [(16, 2), (8, 1), (16, 1), (4, 4), (32, 4), (64, 1)][_draw(gen, 0, 5)]
    packed, top = bool(_draw(gen, 0, 2) == 0), [20, 150, 700][seed % 3]
    seqs = []
    for _ in range(_draw(gen, 1, [90, 24, 5][seed % 3])):
        n = [0, 1, 1, _draw(gen, 1, top), _draw(gen, 1, top)][_draw(gen, 0, 4)]
        prefix = 0 if packed and _draw(gen, 0, 3) else _draw(gen, 0, [60, 500, 1500][_draw(gen, 0, 2)])
        seqs.append((n, max(n + prefix - (_draw(gen, 0, 9) == 0) * 3, 0)))
    if not any(n for n, _ in seqs):
        seqs.append((3, 5))
    _varlen_case(2000 + seed, seqs, h, hk, None if packed else [64, 256, 192][_draw(gen, 0, 2)], _rows(gen, len(seqs)),
                 extra_cols=_draw(gen, 0, 2))


@pytest.mark.parametrize("seed", range(16))
def test_random_evictions(seed):
    gen = torch.Generator().manual_seed(3000 + seed)
    kind, hk, bs = ["bf16", "fp4", "narrow"][seed % 3], _draw(gen, 1, 3), [16, 64, 96, 256][_draw(gen, 0, 3)]
    reach = _draw(gen, 1, [200, 1500, 3000][_draw(gen, 0, 2)])
    cols = -(-reach // bs)
    if kind == "fp4" and bs % 64:
        bs, cols = 64, -(-reach // 64)
    lens = [_draw(gen, 0, reach) for _ in range(_draw(gen, 1, 6))]
    budget = _draw(gen, 1, reach)
    sinks = _draw(gen, 0, budget)
    recent = _draw(gen, 0, budget - sinks)
    need, spare = sum(-(-n // bs) for n in lens), len(lens) * -(-budget // bs)
    tables, rest = _tables(gen, lens, need + spare + 2, bs, cols)
    new = None
    if _draw(gen, 0, 1):
        per = -(-budget // bs)
        new = [[rest[b * per + c] if c < per and _draw(gen, 0, 2) else -1 for c in range(cols)] for b in range(len(lens))]
    rows = _rows(gen, len(lens))
    weights = torch.rand(2, len(lens) + 4, hk, cols * bs + _draw(gen, 0, 9), generator=gen)
    if _draw(gen, 0, 1):
        weights = torch.floor(weights * 8)
    _evict_case(_kv(gen, 2, need + spare + 2, bs, hk, kind), weights, tables, lens, budget, sinks, recent, rows, new)


# ----------------------------------------------------------------------------------------------------------------------
# decode over 4-bit caches


def _decode_fp4_case(seed, lens, h, hk, bs, rows=None, store=False, plan=None):
    """As _decode_case. A score is off by at most 2^-13 of its magnitude (the scaled MFMA's sum) and by what the query's two
    fp8 parts leave, 2^-18 of the row's largest magnitude a channel; a probability takes its own score's error x and its
    row's: e^2x - 1 <= 2 x (1 + 2 x) of it."""
    gen = torch.Generator().manual_seed(seed)
    B, need = len(lens), sum(-(-n // bs) for n in lens) + 2
    _, _, tables = paged_pool(gen, lens, need, bs, 1, 1, 1)
    planes, live, slots = [], torch.zeros(need * bs, dtype=torch.bool), []
    for b, n in enumerate(lens):
        at = [int(tables[b, j // bs]) * bs + j % bs for j in range(n)]
        live[at] = True
        slots.append(at[-1] if at else -1)
    for _ in range(2):  # what no context reaches is not a number
        scales = torch.randint(123, 128, (need * bs, hk, 4), generator=gen, dtype=torch.uint8)
        scales[~live] = 255
        planes.append(fp4.plane(torch.randint(0, 256, (need, bs, hk, 64), generator=gen, dtype=torch.uint8),
                                scales.view(need, bs, hk, 4)))
    n_rows = B if rows is None else max([*rows, 0]) + 2
    w = _received(gen, n_rows, hk, tables.shape[1] * bs + 5)
    q, key, value = randn(gen, B, h, D), randn(gen, B, hk, D), randn(gen, B, hk, D)
    for b, n in enumerate(lens):
        r = b if rows is None else rows[b]
        if n and 0 <= r < n_rows:
            w[r, :, n - 1] = float("nan")
    kd, vd, wd = planes[0].to(DEV), planes[1].to(DEV), w.to(DEV)
    kw = dict(key=key.to(DEV), value=value.to(DEV), slot_mapping=_i32(slots)) if store else {}
    o = decode_attention_weights(q.to(DEV), kd, vd, _i32(lens), tables.to(DEV), SCALE, wd, plan=plan,
                                 weight_rows=None if rows is None else _i32(rows), **kw)
    if store:
        fp4.store(key, value, planes[0], planes[1], torch.tensor(slots, dtype=torch.int32))
        assert torch.equal(kd.cpu(), planes[0]) and torch.equal(vd.cpu(), planes[1])
    kv, vv = (fp4.cache_values(c) for c in planes)
    want = Want(w)
    for b, n in enumerate(lens):
        if n == 0:
            want.o.append(torch.zeros(1, h, D, dtype=torch.float64))
            want.otol.append(torch.zeros(1, h, D, dtype=torch.float64))
            continue
        k, v = ref.keys_of(kv, tables[b], n)[0], ref.keys_of(vv, tables[b], n)[0]
        size = (q[b].double().abs().view(hk, -1, D) @ k.abs().permute(1, 2, 0)).max()
        x = SCALE * float(2.0 ** -13 * size + 2.0 ** -18 * q[b].abs().max() * k.abs().sum(-1).max())
        want.sequence(q[b:b + 1], k, v, None, b if rows is None else rows[b], 1, more=2 * x * (1 + 2 * x))
    want.check(o, wd)


@pytest.mark.parametrize("store", [False, True])
@pytest.mark.parametrize("h,hk,bs", [(16, 2, 256), (8, 1, 64), (16, 1, 128), (6, 2, 192), (3, 1, 64), (2, 2, 256)])
def test_decode_fp4_lengths(h, hk, bs, store):
    """Lengths around the steps, the chunks of two and the blocks, padded rows, rows in any order and none."""
    lens = [1, 2, 0, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, bs - 1, bs, bs + 1, 0, 500, 3 * bs + 7]
    gen = torch.Generator().manual_seed(h)
    rows = torch.randperm(len(lens) + 3, generator=gen)[:len(lens)].tolist()
    rows[4] = -1
    _decode_fp4_case(60 + h + bs, lens, h, hk, bs, rows, store)
    _decode_fp4_case(61 + h + bs, lens, h, hk, bs, None, store, plan=("fp4", h, bs, store))


@pytest.mark.parametrize("lens,h,hk", [([420], 16, 2), ([33000], 16, 2), ([2, 9000, 5], 8, 1), ([40 + 7 * i for i in range(150)], 16, 2),
                                       ([20] * 600, 16, 1), ([20000] * 3 + [17000], 16, 2)])
def test_decode_fp4_batches(lens, h, hk):
    """Four waves a workgroup and eight, sequences in many ranges, more than a launch lays out."""
    _decode_fp4_case(len(lens), lens, h, hk, 256, None, len(lens) > 1)


def test_decode_fp4_blocks_that_are_none_take_no_weight():
    gen = torch.Generator().manual_seed(71)
    n, bs, h, hk = 500, 64, 16, 2
    planes = [fp4.plane(torch.randint(0, 256, (12, bs, hk, 64), generator=gen, dtype=torch.uint8),
                        torch.randint(123, 128, (12, bs, hk, 4), generator=gen, dtype=torch.uint8)) for _ in range(2)]
    table = torch.tensor([[3, -1, 5, 900, 7, 1, 0, 11]], dtype=torch.int32)
    q, w = randn(gen, 1, h, D), _received(gen, 1, hk, 512)
    before = w.clone().double()
    o = decode_attention_weights(q.to(DEV), planes[0].to(DEV), planes[1].to(DEV), _i32([n]), table.to(DEV), SCALE,
                                 wd := w.to(DEV))
    (k, ok), (v, _) = (ref.keys_of(fp4.cache_values(c), table[0], n) for c in planes)
    size = (q[0].double().abs().view(hk, -1, D) @ k.abs().permute(1, 2, 0)).max()
    x = SCALE * float(2.0 ** -13 * size + 2.0 ** -18 * q.abs().max() * k.abs().sum(-1).max())
    want = Want(w)
    want.sequence(q, k, v, ok, 0, 1, more=2 * x * (1 + 2 * x))
    want.check(o, wd)
    assert not ok[64:128].any() and torch.equal(wd[0, :, 64:128].cpu().double(), before[0, :, 64:128])


def _varlen_fp4_case(seed, seqs, h, hk, bs, rows=None, drop=(), plan=None):
    """As _varlen_case through block tables, the tolerances as _decode_fp4_case's."""
    gen = torch.Generator().manual_seed(seed)
    lens, T, cu_q, cu_k = [m for _, m in seqs], sum(n for n, _ in seqs), [0], [0]
    for n, m in seqs:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    need = sum(-(-n // bs) for n in lens) + 2
    _, _, tables = paged_pool(gen, lens, need, bs, 1, 1, 1)
    for b, c in drop:
        tables[b, c] = -1
    live = torch.zeros(need * bs, dtype=torch.bool)
    for b, n in enumerate(lens):
        live[[int(tables[b, j // bs]) * bs + j % bs for j in range(n) if tables[b, j // bs] >= 0]] = True
    planes = []
    for _ in range(2):
        scales = torch.randint(123, 128, (need * bs, hk, 4), generator=gen, dtype=torch.uint8)
        scales[~live] = 255
        planes.append(fp4.plane(torch.randint(0, 256, (need, bs, hk, 64), generator=gen, dtype=torch.uint8),
                                scales.view(need, bs, hk, 4)))
    n_rows = len(seqs) if rows is None else max([*rows, 0]) + 2
    w, q = _received(gen, n_rows, hk, tables.shape[1] * bs + 3), randn(gen, T, h, D)
    for b, (n, m) in enumerate(seqs):
        r = b if rows is None else rows[b]
        if n and 0 <= r < n_rows:
            w[r, :, max(m - n, 0):m] = float("nan")
    wd = w.to(DEV)
    o = varlen_attention_weights(q.to(DEV), None, None, wd, None if rows is None else _i32(rows), cu_seqlens_q=_i32(cu_q),
                                 cu_seqlens_k=_i32(cu_k), max_seqlen_q=max(n for n, _ in seqs), max_seqlen_k=max(lens),
                                 softmax_scale=SCALE, block_table=tables.to(DEV), k_cache=planes[0].to(DEV),
                                 v_cache=planes[1].to(DEV), plan=plan)
    kv, vv = (fp4.cache_values(c) for c in planes)
    want = Want(w)
    for b, (n, m) in enumerate(seqs):
        (k, ok), (v, _) = (ref.keys_of(c, tables[b], m) for c in (kv, vv))
        x, qb = 0.0, q[cu_q[b]:cu_q[b + 1]]
        if n and m:
            size = (qb.double().abs().view(n, hk, -1, D).transpose(0, 1).reshape(hk, -1, D) @ k.abs().permute(1, 2, 0)).max()
            x = SCALE * float(2.0 ** -13 * size + 2.0 ** -18 * qb.abs().max() * k.abs().sum(-1).max())
        want.sequence(qb, k, v, ok, b if rows is None else rows[b], n, more=2 * x * (1 + 2 * x))
    want.check(o, wd)


@pytest.mark.parametrize("h,hk", [(16, 2), (8, 1), (4, 4), (32, 4), (16, 1), (64, 1)])
@pytest.mark.parametrize("bs", [64, 256, 192])
def test_chunks_over_fp4_prefixes(h, hk, bs):
    """Chunks over prefixes of none to several blocks, a sequence without queries, one with fewer keys than queries, rows of
    any order, one of them none, blocks that are none."""
    seqs = [(5, 55), (1, 1), (1, 300), (0, 130), (33, 33), (64, 257), (17, 11), (100, 420), (3, 64)]
    gen = torch.Generator().manual_seed(h + bs)
    rows = torch.randperm(len(seqs) + 3, generator=gen)[:len(seqs)].tolist()
    rows[1] = -1
    _varlen_fp4_case(80 + h + hk + bs, seqs, h, hk, bs, rows, drop=[(7, 0)] if bs < 256 else [])


@pytest.mark.parametrize("seqs,h,hk", [
    ([(700, 2300), (1, 1801)], 16, 2), ([(44, 94)] * 44, 16, 2), ([(1100, 1100)] * 3 + [(513, 700)], 16, 2), ([(1, 1)], 8, 1),
    ([(1, 5 + 37 * i) for i in range(20)] + [(90, 90), (0, 50), (130, 400), (1, 1)], 16, 2),
    ([(1, 5 + 37 * i) for i in range(20)] + [(90, 90), (0, 50), (130, 400), (1, 1)], 8, 1),
    ([(1, 1 + i % 70) for i in range(600)], 8, 1), ([(40, 20000)], 16, 2), ([(1300, 1300)], 8, 1)])
def test_chunk_fp4_sizes(seqs, h, hk):
    _varlen_fp4_case(len(seqs) + h, seqs, h, hk, 256)
    _varlen_fp4_case(len(seqs) + h, seqs, h, hk, 64, plan=("fp4 chunk", len(seqs), h))


def test_chunk_fp4_groups_that_are_not_numbers():
    """A key's group without a number, at a cached token: NaN wherever a query sees it, and nowhere else."""
    gen = torch.Generator().manual_seed(91)
    codes = torch.randint(0, 256, (2, 4, 64, 2, 64), generator=gen, dtype=torch.uint8)
    scales = torch.randint(123, 128, (2, 4, 64, 2, 4), generator=gen, dtype=torch.uint8)
    scales[0, 0, 50, 1, 2] = 255  # token 50's key, kv head 1
    planes = [fp4.plane(c, s) for c, s in zip(codes, scales)]
    w = torch.zeros(1, 2, 256, device=DEV)
    o = varlen_attention_weights(randn(gen, 60, 16, D).to(DEV), None, None, w, cu_seqlens_q=_i32([0, 60]),
                                 cu_seqlens_k=_i32([0, 60]), max_seqlen_q=60, max_seqlen_k=60, softmax_scale=SCALE,
                                 block_table=_i32([[0, 1]]), k_cache=planes[0].to(DEV), v_cache=planes[1].to(DEV))
    assert w[0, 0, :60].isfinite().all() and o[:, :8].isfinite().all() and o[:50, 8:].isfinite().all()
    assert o[50:, 8:].isnan().all() and w[0, 1, :51].isnan().all()
