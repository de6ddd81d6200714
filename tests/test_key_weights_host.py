"""Key weights and eviction on the CPU: the oracle against closed forms, the host side (contexts, allocation, dispatch,
checks), and the refusals of the operators and of the C ABI (nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from oracle import attention, key_weights as ref
from voxcpm2_arabic_dialects_turbo_amd import _lib, checks, layers, ops_weights, runner
from voxcpm2_arabic_dialects_turbo_amd.context import get_context, reset_context, set_context
from voxcpm2_arabic_dialects_turbo_amd.kernels import kv_evict
from voxcpm2_arabic_dialects_turbo_amd.layers import Attention
from voxcpm2_arabic_dialects_turbo_amd.ops_weights import decode_attention_weights, varlen_attention_weights

BF16, I32 = torch.bfloat16, torch.int32


# ----------------------------------------------------------------------------------------------------------------------
# the oracle


def test_oracle_attention_is_the_oracles():
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 8, generator=gen, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    o, p, pv, size = ref.attend(q, k, v, 0.3)
    assert torch.allclose(o.reshape(5, -1), attention.attend(q, k, v, True, 0.3))
    assert torch.allclose(p.sum(-1), torch.ones(4, 5, dtype=torch.float64)) and (p[:, 0, 5:] == 0).all()
    assert (pv >= o.abs() - 1e-12).all()
    assert (size >= (torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(2, 1)) * 0.3).abs() - 1e-12).all()


def test_oracle_weights_known_answers():
    """Equal scores: token j of a prompt gets sum_{i >= j} 1 / (i + 1) from each head; a next token adds 1 / n to all."""
    q, k = torch.zeros(3, 4, 8), torch.zeros(4, 2, 8)
    row = torch.full((2, 6), float("nan"), dtype=torch.float64)
    ref.add(row, ref.attend(q, k[:3], k[:3], 1.0)[1], 3)
    want = 2 * torch.tensor([1 + 1 / 2 + 1 / 3, 1 / 2 + 1 / 3, 1 / 3], dtype=torch.float64)
    assert torch.allclose(row[:, :3], want.expand(2, 3)) and row[:, 3:].isnan().all()
    ref.add(row, ref.attend(q[:1], k, k, 1.0)[1], 1)
    assert torch.allclose(row[:, :4], torch.cat([want + 0.5, torch.tensor([0.5], dtype=torch.float64)]).expand(2, 4))


def test_oracle_keys_that_are_none_and_rows_without_keys():
    gen = torch.Generator().manual_seed(1)
    q, k = torch.randn(3, 2, 8, generator=gen), torch.randn(2, 1, 8, generator=gen)
    o, p, _, _ = ref.attend(q, k, k, 1.0)  # more queries than keys: the first sees none
    assert (o[0] == 0).all() and (p[:, 0] == 0).all() and torch.allclose(p[:, 1:].sum(-1), torch.ones(2, 2).double())
    k[0] = float("nan")
    o, p, _, _ = ref.attend(q, k, k, 1.0, torch.tensor([False, True]))
    assert (p[:, 2, 0] == 0).all() and (p[:, 2, 1] == 1).all() and (o[1] == 0).all()


def test_oracle_kept_known_answers():
    w = torch.tensor([9.0, 1, 5, 5, 2, 5, 0, 7])
    assert ref.kept(w, 8, 8, 0, 0) == list(range(8))
    assert ref.kept(w, 8, 4, 0, 0) == [0, 2, 3, 7]           # ties: the earliest
    assert ref.kept(w, 8, 4, 1, 2) == [0, 2, 6, 7]
    assert ref.kept(w, 8, 3, 1, 2) == [0, 6, 7]
    w[4] = float("nan")
    assert ref.kept(w, 8, 3, 0, 1) == [0, 4, 7]
    w[:] = torch.tensor([0.0, -0.0, 0, -0.0, 0, 0, 0, 0])
    assert ref.kept(w, 8, 3, 0, 0) == [0, 1, 2]


def test_oracle_evict_moves_heads_apart():
    kv = torch.arange(2 * 3 * 4 * 2 * 2).view(1, 2, 3, 4, 2, 2).float()
    w = torch.tensor([[[[1.0, 5, 2, 4, 3, 0, 0, 0], [5.0, 1, 4, 2, 3, 9, 9, 9]]]])
    old = kv.clone()
    tables, lens = ref.evict(kv, w, [[2, 0]], [5], 3)
    assert tables == [[2, -1]] and lens == [3]
    assert w[0, 0, 0].tolist() == [5, 4, 3, 4, 3, 0, 0, 0] and w[0, 0, 1].tolist() == [5, 4, 3, 2, 3, 9, 9, 9]
    for g, stay in ((0, [(2, 1), (2, 3), (0, 0)]), (1, [(2, 0), (2, 2), (0, 0)])):
        for j, (b, i) in enumerate(stay):
            assert torch.equal(kv[0, :, 2, j, g], old[0, :, b, i, g])
    assert torch.equal(kv[0, :, 2, 3], old[0, :, 2, 3]) and torch.equal(kv[0, :, :2], old[0, :, :2])


# ----------------------------------------------------------------------------------------------------------------------
# host side


def _task(table, n, cached):
    return runner.RunnerTask(table, n, cached)


def test_contexts_carry_rows_and_positions_go_on_behind_the_text():
    tasks = [_task([3], 20, 0), _task([1, 2], 300, 260)]
    try:
        plain = runner.prepare_prefill_context(tasks, 256, device="cpu")
        assert get_context().weight_rows is None
        pos = runner.prepare_prefill_context(tasks, 256, device="cpu", weight_rows=[5, -1], evicted=[0, 1000])
        ctx = get_context()
        assert ctx.weight_rows.tolist() == [5, -1] and ctx.weight_rows.dtype == I32
        assert torch.equal(pos[:20], plain[:20]) and torch.equal(pos[20:], plain[20:] + 1000)
        assert ctx.slot_mapping[-1] == 2 * 256 + 299 % 256 and ctx.block_tables.tolist() == [[3, -1], [1, 2]]
        pos = runner.prepare_decode_context(tasks, 256, device="cpu", weight_rows=[0, 4], evicted=[7, 0])
        ctx = get_context()
        assert pos.tolist() == [19 + 7, 299] and ctx.slot_mapping.tolist() == [3 * 256 + 19, 2 * 256 + 299 % 256]
        assert ctx.context_lens.tolist() == [20, 300] and ctx.weight_rows.tolist() == [0, 4]
        for fn in (runner.prepare_prefill_context, runner.prepare_decode_context):
            with pytest.raises(ValueError, match="one value per sequence"):
                fn(tasks, 256, device="cpu", weight_rows=[1])
            with pytest.raises(ValueError, match="one value per sequence"):
                fn(tasks, 256, device="cpu", evicted=[1, 2, 3])
    finally:
        reset_context()


def test_decode_graph_buffers_hold_the_rows():
    bufs = runner.DecodeGraphBuffers(4, 2, device="cpu", key_weights=True)
    try:
        bufs.bind(3)
        assert get_context().weight_rows.tolist() == [-1, -1, -1]
        runner.prepare_decode_context([_task([3], 20, 19), _task([1], 9, 8)], 256, device="cpu", weight_rows=[6, 2])
        bufs.load()
        assert bufs.weight_rows.tolist() == [6, 2, -1, -1]
        runner.prepare_decode_context([_task([3], 21, 20)], 256, device="cpu")
        bufs.load()
        assert bufs.weight_rows.tolist() == [-1] * 4
        runner.DecodeGraphBuffers(4, 2, device="cpu").bind(2)
        assert get_context().weight_rows is None
    finally:
        reset_context()


def test_allocate_key_weights():
    mods = [Attention(16, 128, 0.1, 2) for _ in range(3)]
    assert all(m.key_weights is None for m in mods)
    w = runner.allocate_key_weights(mods, 5, 512, device="cpu")
    assert w.shape == (3, 5, 2, 512) and w.dtype == torch.float32 and not w.any()
    assert all(m.key_weights.data_ptr() == w[i].data_ptr() for i, m in enumerate(mods))
    for bad in ((0, 512), (5, 0)):
        with pytest.raises(ValueError, match="positive"):
            runner.allocate_key_weights(mods, *bad, device="cpu")
    with pytest.raises(ValueError, match="one number of kv heads"):
        runner.allocate_key_weights([*mods, Attention(8, 128, 0.1, 1)], 5, 512, device="cpu")
    model = torch.nn.ModuleList([*mods, Attention(16, 128, 0.1, 4, is_causal=False)])
    assert runner.allocate_key_weights(model, 1, 256, device="cpu").shape == (3, 1, 2, 256)


@pytest.fixture
def calls(monkeypatch):
    """Attention.forward's operators, recorded."""
    seen = []
    for name in ("decode_attention_weights", "varlen_attention_weights", "store_kvcache", "decode_attention",
                 "prefill_attention_store"):
        def fn(q, *a, _name=name, **kw):
            seen.append((_name, a, kw))
            return q
        monkeypatch.setattr(layers, name, fn)
    yield seen
    reset_context()


def _layer(fp4=False):
    layer = Attention(16, 128, 0.1, 2)
    shape, dtype = ((4, 256, 2, 68), torch.uint8) if fp4 else ((4, 256, 2, 128), BF16)
    layer.k_cache, layer.v_cache = torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)
    return layer


def _rows(n):
    return torch.zeros(n, 16, 128, dtype=BF16), torch.zeros(n, 2, 128, dtype=BF16), torch.zeros(n, 2, 128, dtype=BF16)


def test_attention_adds_where_the_layer_has_weights_and_the_step_rows(calls):
    i32 = lambda *x: torch.tensor(x, dtype=I32)  # noqa: E731
    layer, rows = _layer(), i32(1, 0)

    def step(prefill, tables, weight_rows):
        calls.clear()
        if prefill:
            set_context(True, i32(0, 2, 3), i32(0, 2, 3), 2, 2, i32(0, 1, 256), None, tables, weight_rows)
            layer(*_rows(3))
        else:
            set_context(False, slot_mapping=i32(0, 256), context_lens=i32(1, 1), block_tables=i32(0, 1).view(2, 1),
                        weight_rows=weight_rows)
            layer(*_rows(2))
        return [c[0] for c in calls]

    tables = i32(0, 1).view(2, 1)
    for r in (None, rows):  # a layer without weights
        assert step(True, None, r) == ["prefill_attention_store"] and step(False, tables, r) == ["decode_attention"]
    layer.key_weights = torch.zeros(2, 2, 256)
    assert step(True, None, None) == ["prefill_attention_store"] and step(False, tables, None) == ["decode_attention"]
    assert step(True, None, rows) == ["store_kvcache", "varlen_attention_weights"]
    assert calls[1][2]["block_table"] is None and calls[1][1][3] is rows
    assert step(True, tables, rows) == ["store_kvcache", "varlen_attention_weights"]
    assert calls[1][2]["block_table"] is tables and calls[1][2]["max_seqlen_k"] == 2
    assert step(False, tables, rows) == ["decode_attention_weights"]
    assert calls[0][1][-2] is layer.key_weights and calls[0][2]["slot_mapping"].tolist() == [0, 256]


def test_attention_over_4_bit_caches_adds_too(calls):
    i32 = lambda *x: torch.tensor(x, dtype=I32)  # noqa: E731
    layer = _layer(fp4=True)
    layer.key_weights = torch.zeros(1, 2, 256)
    set_context(True, i32(0, 3), i32(0, 3), 3, 3, i32(0, 1, 2), None, None, i32(0))
    layer(*_rows(3))
    assert [c[0] for c in calls] == ["store_kvcache", "varlen_attention_weights"]
    calls.clear()
    set_context(True, i32(0, 3), i32(0, 3), 3, 3, i32(0, 1, 2), None, i32(0).view(1, 1), i32(0))
    layer(*_rows(3))
    assert [c[0] for c in calls] == ["store_kvcache", "varlen_attention_weights"]
    assert calls[1][2]["k_cache"] is layer.k_cache and calls[1][2]["block_table"] is not None


def test_eviction_violations():
    i32 = lambda *x: torch.tensor(x, dtype=I32)  # noqa: E731
    tables, lens = torch.tensor([[3, 0, 7], [3, 0, 5], [1, -1, -1]]), i32(180, 150, 60)
    look = lambda **kw: checks.eviction_violations(tables, lens, 64, 100, **kw)  # noqa: E731
    assert look(new_blocks=torch.tensor([[8, 9, -1], [10, 11, -1], [-1, -1, -1]])) == []
    assert any("names" in v for v in look())
    assert any("names" in v for v in look(new_blocks=torch.tensor([[8, -1, -1], [10, 11, -1], [-1, -1, -1]])))
    assert any("new block 1" in v for v in look(new_blocks=torch.tensor([[8, 1, -1], [10, 11, -1], [-1, -1, -1]])))
    assert any("both" in v for v in look(new_blocks=torch.tensor([[8, 9, -1], [10, 9, -1], [-1, -1, -1]])))
    assert any("share row 2" in v for v in look(weight_rows=i32(2, 0, 2), new_blocks=tables * 0 - 1))
    # rows -1 are not brought down, and may be several
    assert look(weight_rows=i32(-1, -1, -1)) == []
    assert checks.eviction_violations(tables[:, 2:], i32(10, 10, 0), 64, 4) == []
    assert checks.eviction_violations(tables, lens, 64, 500) == []


# ----------------------------------------------------------------------------------------------------------------------
# refusals


def _decode(**kw):
    a = dict(q=torch.zeros(2, 16, 128, dtype=BF16), k_cache=torch.zeros(4, 64, 2, 128, dtype=BF16),
             v_cache=torch.zeros(4, 64, 2, 128, dtype=BF16), context_lens=torch.zeros(2, dtype=I32),
             block_tables=torch.zeros(2, 2, dtype=I32), softmax_scale=0.1, key_weights=torch.zeros(2, 2, 128))
    a.update(kw)
    return decode_attention_weights(**a)


@pytest.mark.parametrize("kw,error,match", [
    (dict(), ValueError, "same GPU"),  # (CPU tensors)
    (dict(q=torch.zeros(2, 16, 128)), TypeError, "bf16"),
    (dict(q=torch.zeros(2, 16 * 128, dtype=BF16)), TypeError, "bf16"),
    (dict(k_cache=torch.zeros(4, 64, 2, 68, dtype=torch.uint8)), TypeError, "bf16 caches"),
    (dict(k_cache=torch.zeros(4, 64, 2, 64, dtype=BF16)), ValueError, "contiguous"),
    (dict(v_cache=torch.zeros(4, 64, 2, 256, dtype=BF16)[..., :128]), ValueError, "contiguous"),
    (dict(q=torch.zeros(2, 32, 128, dtype=BF16)), ValueError, "H <= 16"),
    (dict(q=torch.zeros(2, 3, 128, dtype=BF16)), ValueError, "H <= 16"),
    (dict(softmax_scale=0.0), ValueError, "positive"),
    (dict(softmax_scale=-1.0), ValueError, "positive"),
    (dict(softmax_scale=float("nan")), ValueError, "positive"),
    (dict(context_lens=torch.zeros(3, dtype=I32)), ValueError, "context_lens"),
    (dict(block_tables=torch.zeros(1, 2, dtype=I32)), ValueError, "block_tables"),
])
def test_decode_refusals(kw, error, match):
    with pytest.raises(error, match=match):
        _decode(**kw)


@pytest.mark.parametrize("kw,error,match", [
    (dict(key_weights=torch.zeros(2, 2, 128, dtype=torch.float64)), TypeError, "fp32"),
    (dict(key_weights=torch.zeros(2, 1, 128)), ValueError, "contiguous"),
    (dict(key_weights=torch.zeros(2, 2, 256)[..., ::2]), ValueError, "contiguous"),
    (dict(key_weights=torch.zeros(4, 2)), ValueError, "contiguous"),
    (dict(key_weights=torch.zeros(2, 2, 127)), ValueError, "the keys may be 128"),
    (dict(key_weights=torch.zeros(1, 2, 128)), ValueError, "1 rows for 2"),
    (dict(weight_rows=torch.zeros(3, dtype=I32)), ValueError, "one row per sequence"),
    (dict(key_weights=torch.zeros(0, 2, 128), weight_rows=torch.zeros(2, dtype=I32)), ValueError, "no rows"),
    (dict(weight_rows=torch.zeros(2)), TypeError, "integer"),
])
def test_weights_refusals(kw, error, match):
    a = dict(key_weights=torch.zeros(2, 2, 128), weight_rows=None)
    a.update(kw)
    with pytest.raises(error, match=match):
        ops_weights._weights("f", a["key_weights"], a["weight_rows"], 2, 2, 128, -1)


def test_decode_rows_refusals(monkeypatch):
    monkeypatch.setattr(ops_weights, "_check_cuda", lambda *t: torch.device("cpu"))
    k = torch.zeros(2, 2, 128, dtype=BF16)
    slots = torch.zeros(2, dtype=I32)
    for kw in (dict(key=k), dict(value=k), dict(slot_mapping=slots), dict(key=k, value=k), dict(value=k, slot_mapping=slots)):
        with pytest.raises(ValueError, match="go together"):
            _decode(**kw)
    with pytest.raises(ValueError, match="must hold 2 rows"):
        _decode(key=k[:1], value=k[:1], slot_mapping=slots)
    with pytest.raises(ValueError, match="must hold 2 rows"):
        _decode(key=k, value=k, slot_mapping=slots[:1])
    with pytest.raises(TypeError, match="bf16"):
        _decode(key=k.float(), value=k, slot_mapping=slots)
    with pytest.raises(ValueError, match="N, 2, 128"):
        _decode(key=k[:, :1], value=k[:, :1], slot_mapping=slots)
    with pytest.raises(ValueError, match="heads must be contiguous"):
        _decode(key=torch.zeros(2, 4, 128, dtype=BF16)[:, ::2], value=k, slot_mapping=slots)
    with pytest.raises(ValueError, match="out must be"):
        _decode(out=torch.zeros(2, 16, 256, dtype=BF16)[..., :128])
    with pytest.raises(ValueError, match="out must be"):
        _decode(out=torch.zeros(3, 16, 128, dtype=BF16))


@pytest.mark.parametrize("kw,error,match", [
    (dict(q=torch.zeros(4, 16, 128)), TypeError, "bf16"),
    (dict(cu_seqlens_k=torch.zeros(2, dtype=I32)), ValueError, "as many entries"),
    (dict(softmax_scale=0), ValueError, "positive"),
    (dict(k=None), ValueError, "packed keys"),
    (dict(k=torch.zeros(4, 2, 64, dtype=BF16)), ValueError, "N, 2, 128"),
    (dict(k=torch.zeros(4, 2, 128)), TypeError, "bf16"),
    (dict(k=torch.zeros(4, 3, 128, dtype=BF16), v=torch.zeros(4, 3, 128, dtype=BF16)), ValueError, "not a multiple"),
    (dict(k=torch.zeros(4, 256, dtype=BF16)), ValueError, "must be"),
    (dict(block_table=torch.zeros(2, 1, dtype=I32)), ValueError, "without caches"),
    (dict(block_table=torch.zeros(2, 1, dtype=I32), k_cache=torch.zeros(4, 32, 2, 128, dtype=BF16)), ValueError,
     "multiple of 64"),
    (dict(block_table=torch.zeros(1, 1, dtype=I32), k_cache=torch.zeros(4, 64, 2, 128, dtype=BF16)), ValueError,
     "block_table must be"),
    (dict(block_table=torch.zeros(2, 1, dtype=I32), k_cache=torch.zeros(4, 64, 2, 68, dtype=torch.uint8),
          v_cache=torch.zeros(4, 64, 2, 128, dtype=BF16)), TypeError, "bf16 caches"),
    (dict(max_seqlen_k=129), ValueError, "the keys may be 129"),
    (dict(key_weights=torch.zeros(1, 2, 128)), ValueError, "1 rows for 2"),
    (dict(out=torch.zeros(4, 16, 128)), ValueError, "out must be"),
])
def test_varlen_refusals(monkeypatch, kw, error, match):
    monkeypatch.setattr(ops_weights, "_check_cuda", lambda *t: torch.device("cpu"))
    a = dict(q=torch.zeros(4, 16, 128, dtype=BF16), k=torch.zeros(4, 2, 128, dtype=BF16),
             v=torch.zeros(4, 2, 128, dtype=BF16), key_weights=torch.zeros(2, 2, 128), cu_seqlens_q=torch.zeros(3, dtype=I32),
             cu_seqlens_k=torch.zeros(3, dtype=I32), max_seqlen_q=3, max_seqlen_k=3, softmax_scale=0.1)
    a.update(kw)
    if "k_cache" in a:
        a.setdefault("v_cache", a["k_cache"])
    with pytest.raises(error, match=match):
        varlen_attention_weights(**a)


@pytest.mark.parametrize("kw,error,match", [
    (dict(kv=torch.zeros(2, 4, 64, 1, 128, dtype=BF16)), ValueError, "kv must be"),
    (dict(kv=torch.zeros(1, 2, 4, 64, 1, 128, dtype=BF16)[..., ::2]), ValueError, "contiguous"),
    (dict(kv=torch.zeros(1, 2, 4, 64, 1, 100, dtype=BF16)), ValueError, "multiple of 16 bytes"),
    (dict(kv=torch.zeros(1, 2, 1, 64, 1, 2056, dtype=BF16)), ValueError, "multiple of 16 bytes"),
    (dict(kv=torch.zeros(1, 2, 4, 64, 1, 64, dtype=torch.uint8)), ValueError, "4-bit"),
    (dict(key_weights=torch.zeros(1, 2, 1, 128, dtype=BF16)), TypeError, "fp32"),
    (dict(key_weights=torch.zeros(2, 2, 1, 128)), ValueError, "contiguous"),
    (dict(key_weights=torch.zeros(1, 2, 2, 128)), ValueError, "contiguous"),
    (dict(key_weights=torch.zeros(1, 2, 1, 127)), ValueError, "the tables reach 128"),
    (dict(key_weights=torch.zeros(1, 1, 1, 128)), ValueError, "1 rows for 2"),
    (dict(budget=0), ValueError, "budget"),
    (dict(budget=10, sinks=6, recent=5), ValueError, "budget"),
    (dict(sinks=-1), ValueError, "budget"),
    (dict(recent=-1), ValueError, "budget"),
    (dict(weight_rows=torch.zeros(1, dtype=I32)), ValueError, "one row per sequence"),
    (dict(new_blocks=torch.zeros(2, 1, dtype=I32)), ValueError, "new_blocks"),
    (dict(new_blocks=torch.zeros(1, 2, dtype=I32)), ValueError, "new_blocks"),
    (dict(block_tables=torch.zeros(1, 2, dtype=I32)), ValueError, "block_tables"),
    (dict(block_tables=torch.zeros(2, 0, dtype=I32)), ValueError, "empty"),
])
def test_evict_refusals(monkeypatch, kw, error, match):
    from voxcpm2_arabic_dialects_turbo_amd.kernels import kv_pages
    monkeypatch.setattr(kv_pages, "_check_cuda", lambda *t: torch.device("cpu"))
    a = dict(kv=torch.zeros(1, 2, 4, 64, 1, 128, dtype=BF16), key_weights=torch.zeros(1, 2, 1, 128),
             block_tables=torch.zeros(2, 2, dtype=I32), context_lens=torch.zeros(2, dtype=I32), budget=10)
    a.update(kw)
    with pytest.raises(error, match=match):
        kv_evict.evict_kv_tokens(**a)


def test_evict_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="same GPU"):
        kv_evict.evict_kv_tokens(torch.zeros(1, 2, 4, 64, 1, 128, dtype=BF16), torch.zeros(1, 2, 1, 128),
                                 torch.zeros(2, 2, dtype=I32), torch.zeros(2, dtype=I32), 10)


# The C entries with addresses that are never followed: each call is refused for the one argument that is wrong.
P = 1 << 20


def _einval(status, match):
    assert status == _lib.VOX_EINVAL and match in _lib.load().vox_last_error().decode(), _lib.load().vox_last_error()


DECODE_C = dict(q=P, qs=2048, key=None, value=None, ks=0, vs=0, slots=None, kc=P, vc=P, blocks=4, bs=64, bt=P, bts=2, mb=2,
                lens=P, batch=2, h=16, hk=2, d=128, scale=0.1, w=P, rows=None, n_rows=2, width=128, scores=P,
                scores_bytes=1 << 30, plan=0, ws=P, ws_bytes=1 << 30, out=P, stream=None)


@pytest.mark.parametrize("kw,match", [
    (dict(batch=-1), "batch < 0"), (dict(plan=3), "plan mode"), (dict(w=None), "key_weights"), (dict(w=P + 2), "key_weights"),
    (dict(n_rows=0), "empty key_weights"), (dict(width=0), "empty key_weights"), (dict(scale=0.0), "positive"),
    (dict(scale=float("inf")), "positive"), (dict(key=P), "go together"), (dict(slots=P), "go together"),
    (dict(key=P, value=P, slots=P, ks=128, vs=256), "strides"), (dict(key=P + 8, value=P, slots=P, ks=256, vs=256), "aligned"),
    (dict(scores=None), "scores"), (dict(scores=P + 4), "scores"), (dict(scores_bytes=2 * 8 * 16 * 16 * 4 - 1), "needed"),
    (dict(bs=48), "multiple of 32"), (dict(hk=4), "num_kv_heads"), (dict(d=64), "head_dim"), (dict(ws_bytes=10), "workspace"),
])
def test_c_decode_refusals(kw, match):
    _einval(_lib.load().vox_decode_attn_weights(*{**DECODE_C, **kw}.values()), match)


def test_c_scores_bytes():
    lib = _lib.load()
    assert lib.vox_decode_scores_bytes(2, 2, 64, 16) == 2 * 8 * 16 * 16 * 4
    assert lib.vox_decode_scores_bytes(600, 3, 32, 8) == 512 * 6 * 8 * 16 * 4  # (one launch's)
    assert lib.vox_decode_scores_bytes(512, 1 << 20, 1024, 16) == 512 * (1 << 26) * 16 * 16 * 4
    for bad in ((0, 2, 64, 16), (2, 0, 64, 16), (2, 2, 0, 16), (2, 2, 64, 0), (-1, 2, 64, 16)):
        assert lib.vox_decode_scores_bytes(*bad) == 0
    assert lib.vox_decode_attn_weights(*{**DECODE_C, "batch": 0, "q": None}.values()) == _lib.VOX_OK


PREFILL_C = dict(q=P, qs=2048, key=P, value=P, ks=256, vs=256, kc=None, vc=None, blocks=0, bs=0, bt=None, bts=0, mb=0, cq=P,
                 ck=P, batch=2, mq=4, mk=4, n=8, h=16, hk=2, d=128, scale=0.1, w=P, rows=None, n_rows=2, width=128,
                 scratch=P, scratch_bytes=1 << 30, scores=None, scores_bytes=0, plan=0, ws=None, ws_bytes=0, out=P, outs=2048,
                 stream=None)
PAGED = dict(key=None, value=None, ks=0, vs=0, kc=P, vc=P, blocks=4, bs=64, bt=P, bts=2, mb=2)


@pytest.mark.parametrize("kw,match", [
    (dict(batch=-1), "negative"), (dict(mq=-1), "negative"), (dict(mk=-1), "negative"), (dict(n=-1), "negative"),
    (dict(cq=None), "null"), (dict(out=None), "null"), (dict(scratch=None), "scratch"), (dict(scratch=P + 8), "scratch"),
    (dict(scratch_bytes=8 * 16 * 4 - 1), "needed"), (dict(qs=1 << 24), "2^24"), (dict(w=None), "key_weights"),
    (dict(scale=-0.1), "positive"), (dict(outs=100), "out row stride"), (dict(out=P + 2), "alignment"),
    (dict(batch=70000), "65535"), (dict(key=None), "null key"), (dict(h=24, qs=3200, outs=3200), "divide 128"), (dict(d=64), "head_dim"),
    (dict(PAGED, bs=32), "multiple of 64"), (dict(PAGED, bs=0), "multiple of 64"), (dict(PAGED, mb=1 << 25, bts=1 << 25), "too wide"),
    (dict(PAGED, kc=None), "without caches"), (dict(PAGED, bts=1), "bad block table"),
    (dict(mq=1 << 28), "too large"), (dict(mk=(1 << 30) + 1), "too large"), (dict(mk=1 << 30, batch=100), "too large"),
    (dict(PAGED, ws=P, ws_bytes=10), "workspace"), (dict(PAGED, ws=P, ws_bytes=1 << 30, plan=5), "plan mode"),
    (dict(PAGED, ws=P, ws_bytes=1 << 30), "scores"),
    (dict(PAGED, ws=P, ws_bytes=1 << 30, scores=P, scores_bytes=2 * 8 * 16 * 16 * 4 - 1), "needed"),
])
def test_c_prefill_refusals(kw, match):
    _einval(_lib.load().vox_prefill_attn_weights(*{**PREFILL_C, **kw}.values()), match)


FP4 = [(dict(bs=96), "multiple of 64"), (dict(d=64), "head_dim"), (dict(kc=None), "null pointer"), (dict(vc=P + 8), "aligned"),
       (dict(blocks=0), "empty cache"), (dict(blocks=1 << 26), "int32 slots"), (dict(scale=1e-45), "positive"),
       (dict(w=None), "key_weights"), (dict(batch=-1), "batch")]


@pytest.mark.parametrize("kw,match", FP4 + [(dict(scores=None), "scores"), (dict(plan=7), "plan mode"),
                                            (dict(key=P), "go together"), (dict(hk=3, h=3), "num_kv_heads")])
def test_c_decode_fp4_refusals(kw, match):
    _einval(_lib.load().vox_decode_attn_weights_fp4(*{**DECODE_C, **kw}.values()), match)


@pytest.mark.parametrize("kw,match", FP4 + [
    (dict(bt=None), "null pointer"), (dict(scratch_bytes=8 * 16 * 4 - 1), "needed"), (dict(mk=-1), "negative"),
    (dict(ws=P, ws_bytes=10), "workspace"), (dict(ws=P, ws_bytes=1 << 30), "scores"), (dict(outs=100), "out row stride")])
def test_c_prefill_fp4_refusals(kw, match):
    args = {**PREFILL_C, **PAGED, **kw}
    for name in ("key", "value", "ks", "vs"):
        del args[name]
    _einval(_lib.load().vox_prefill_attn_weights_fp4(*args.values()), match)


def test_c_prefill_of_nothing():
    for kw in (dict(batch=0), dict(mq=0), dict(n=0)):
        assert _lib.load().vox_prefill_attn_weights(*{**PREFILL_C, "q": None, **kw}.values()) == _lib.VOX_OK


EVICT_C = dict(kv=P, layers=1, blocks=4, bs=64, hk=1, head=256, scale=0, bt=P, bts=2, mb=2, lens=P, batch=2, w=P, rows=None,
               n_rows=2, width=128, budget=10, sinks=1, recent=2, into=None, into_s=0, moves=P, tables=P, out_lens=P,
               stream=None)


@pytest.mark.parametrize("kw,match", [
    (dict(batch=-1), "negative"), (dict(layers=-1), "negative"), (dict(kv=None), "null"), (dict(moves=None), "null"),
    (dict(tables=None), "null"), (dict(out_lens=None), "null"), (dict(w=None), "null"), (dict(blocks=0), "cache of"),
    (dict(bs=0), "cache of"), (dict(blocks=1 << 26), "cache of"), (dict(hk=0), "kv heads"), (dict(head=100), "multiples of 16"),
    (dict(head=0), "multiples of 16"), (dict(head=4112), "multiples of 16"), (dict(scale=8), "0 or 4"),
    (dict(kv=P + 8), "aligned"), (dict(moves=P + 4), "aligned"), (dict(bs=1, head=16, scale=4), "aligned"), (dict(bts=1), "bad block table"),
    (dict(mb=0), "bad block table"), (dict(into=P, into_s=1), "new blocks"), (dict(width=127), "the tables reach 128"),
    (dict(n_rows=0), "key_weights"), (dict(budget=0), "budget"), (dict(sinks=9), "budget"), (dict(recent=-1), "budget"),
    (dict(sinks=2**31 - 1, recent=2**31 - 1), "budget"), (dict(batch=70000), "65535"), (dict(layers=40000), "32767"),
])
def test_c_evict_refusals(kw, match):
    _einval(_lib.load().vox_evict_kv_tokens(*{**EVICT_C, **kw}.values()), match)


def test_c_evict_of_nothing():
    for kw in (dict(batch=0), dict(layers=0)):
        assert _lib.load().vox_evict_kv_tokens(*{**EVICT_C, "kv": None, **kw}.values()) == _lib.VOX_OK
