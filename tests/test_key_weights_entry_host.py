"""Calls around the key weights on the CPU: steps that the module takes, looks at a step from the host (nothing is launched)."""

from __future__ import annotations

import pytest
import torch

from tests.test_key_weights_host import P, _einval, _layer, _rows, calls  # noqa: F401
from voxcpm2_arabic_dialects_turbo_amd import _lib, checks, ops_weights
from voxcpm2_arabic_dialects_turbo_amd.context import get_context, set_context
from voxcpm2_arabic_dialects_turbo_amd.ops_weights import varlen_attention_weights

BF16, I32 = torch.bfloat16, torch.int32


def _i32(*x):
    return torch.tensor(x, dtype=I32)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("paged", [False, True])
def test_last_rows_say_which_tokens_are_new(calls, paged, fp4):  # noqa: F811
    """cu_seqlens_q swapped on the live context: the operator gets the step's own beside it."""
    layer = _layer(fp4)
    layer.key_weights = torch.zeros(2, 2, 256)
    cu, tables = _i32(0, 2, 5), _i32(0, 1).view(2, 1) if paged else None
    set_context(True, cu, cu, 3, 3, _i32(0, 1, 256, 257, 258), None, tables, _i32(0, 1))
    (q, _, _), (_, k, v) = _rows(2), _rows(5)
    ctx = get_context()
    ctx.cu_seqlens_q, ctx.max_seqlen_q = _i32(0, 1, 2), 1
    layer(q, k, v)
    assert [c[0] for c in calls] == ["store_kvcache", "varlen_attention_weights"]
    kw = calls[1][2]
    assert kw["cu_seqlens_new"] is cu and kw["cu_seqlens_q"].tolist() == [0, 1, 2] and kw["max_seqlen_q"] == 1
    assert calls[0][1][3].numel() == 5
    ctx.cu_seqlens_q, ctx.max_seqlen_q = cu, 3
    layer(_rows(5)[0], k, v)
    assert calls[-1][2]["cu_seqlens_new"] is None


def test_fewer_queries_than_rows_need_the_new_tokens(calls):  # noqa: F811
    """Nothing is stored or added where the context does not say which tokens are new."""
    layer = _layer()
    layer.key_weights = torch.zeros(2, 2, 256)
    set_context(True, _i32(0, 1, 2), _i32(0, 2, 5), 1, 3, _i32(0, 1, 256, 257, 258), None, None, _i32(0, 1))
    with pytest.raises(ValueError, match="2 queries for 5 new tokens"):
        layer(_rows(2)[0], *_rows(5)[1:])
    get_context().cu_seqlens_new = None
    with pytest.raises(ValueError, match="2 queries for 5 new tokens"):
        layer(_rows(2)[0], *_rows(5)[1:])
    assert calls == []


@pytest.mark.parametrize("fp4", [False, True])
def test_decode_steps_with_more_rows_than_queries_store_then_attend(calls, fp4):  # noqa: F811
    """As a layer without weights takes them."""
    layer = _layer(fp4)
    layer.key_weights = torch.zeros(3, 2, 256)
    for rows, want in ((5, ["store_kvcache", "decode_attention_weights"]), (3, ["decode_attention_weights"])):
        calls.clear()
        slots = torch.arange(rows, dtype=I32) * 256
        set_context(False, slot_mapping=slots, context_lens=_i32(1, 1, 1), block_tables=_i32(0, 1, 2).view(3, 1),
                    weight_rows=_i32(0, 1, 2))
        (q, _, _), (_, k, v) = _rows(3), _rows(rows)
        layer(q, k, v)
        assert [c[0] for c in calls] == want
        if rows == 5:  # (the recorded store drops its first argument)
            assert calls[0][1][0] is v and calls[0][1][3] is slots
            assert calls[1][2].get("key") is None and calls[1][2].get("slot_mapping") is None
        else:
            assert calls[0][2]["key"] is k and calls[0][2]["slot_mapping"] is slots


@pytest.mark.parametrize("prefill", [False, True])
def test_steps_whose_sequences_share_a_row_are_found(calls, monkeypatch, prefill):  # noqa: F811
    layer = _layer()
    layer.key_weights = torch.zeros(3, 2, 256)

    def step(*rows):
        calls.clear()
        slots = torch.arange(3, dtype=I32) * 256
        if prefill:
            set_context(True, _i32(0, 1, 2, 3), _i32(0, 1, 2, 3), 1, 1, slots, None, None, _i32(*rows))
        else:
            set_context(False, slot_mapping=slots, context_lens=_i32(1, 1, 1), block_tables=_i32(0, 1, 2).view(3, 1),
                        weight_rows=_i32(*rows))
        layer(*_rows(3))

    step(1, 0, 1)  # (not looked for by default)
    monkeypatch.setenv("VOX_CHECK_STORE", "1")
    for rows in ((0, 1, 2), (-1, 2, -1)):
        step(*rows)
        assert calls
    with pytest.raises(ValueError, match="sequences 0 and 2 share row 1"):
        step(1, 0, 1)
    assert calls == []


def test_weight_row_violations():
    assert checks.weight_row_violations(_i32(3, -1, 0, -1, 7)) == []
    assert checks.weight_row_violations(_i32(3, 3, 3)) == ["sequences 0 and 1 share row 3 of the weights",
                                                         "sequences 1 and 2 share row 3 of the weights"]
    assert len(checks.weight_row_violations(torch.zeros(50, dtype=torch.int64), limit=4)) == 4


def test_eviction_violations_finds_blocks_that_keep_their_hash():
    tables, lens = torch.tensor([[3, 0, 7], [6, 4, 5], [1, -1, -1]]), _i32(180, 150, 60)
    look = lambda hashed, **kw: checks.eviction_violations(tables, lens, 64, 100, hashed_blocks=hashed, **kw)  # noqa: E731
    assert look([]) == [] and look([1, 5, 7]) == []  # (blocks of a sequence within the budget, and those behind it)
    assert look({0}) == ["sequence 0 is brought down into block 0, which is still handed out by its hash"]
    assert look(torch.tensor([3, 4])) == [f"sequence {b} is brought down into block {v}, which is still handed out by its hash"
                                          for b, v in ((0, 3), (1, 4))]
    new = torch.tensor([[8, 9, -1], [-1, -1, -1], [-1, -1, -1]])
    assert look([3, 0], new_blocks=new) == []
    assert look([3, 0, 9], new_blocks=new) == ["sequence 0 is brought down into block 9, which is still handed out by its hash"]
    assert look([3, 4], weight_rows=_i32(-1, 0, 1)) == ["sequence 1 is brought down into block 4, which is still handed out by "
                                                       "its hash"]


def test_new_tokens_refusals(monkeypatch):
    monkeypatch.setattr(ops_weights, "_check_cuda", lambda *t: torch.device("cpu"))
    a = dict(q=torch.zeros(4, 16, 128, dtype=BF16), k=torch.zeros(4, 2, 128, dtype=BF16), v=torch.zeros(4, 2, 128, dtype=BF16),
             key_weights=torch.zeros(2, 2, 128), cu_seqlens_q=torch.zeros(3, dtype=I32), cu_seqlens_k=torch.zeros(3, dtype=I32),
             max_seqlen_q=3, max_seqlen_k=3, softmax_scale=0.1)
    with pytest.raises(ValueError, match="as many entries"):
        varlen_attention_weights(**a, cu_seqlens_new=torch.zeros(2, dtype=I32))
    with pytest.raises(TypeError, match="integer"):
        varlen_attention_weights(**a, cu_seqlens_new=torch.zeros(3))
    monkeypatch.undo()
    with pytest.raises(ValueError, match="same GPU"):
        varlen_attention_weights(**a, cu_seqlens_new=torch.zeros(3, dtype=I32))


CLEAR_C = dict(w=P, rows=None, n_rows=2, width=128, hk=2, cu_new=P, cu_k=P, batch=2, max_keys=128, max_tokens=128, stream=None)


@pytest.mark.parametrize("kw,match", [
    (dict(batch=-1), "negative"), (dict(max_keys=-1), "negative"), (dict(max_tokens=-1), "negative"), (dict(w=None), "key_weights"),
    (dict(w=P + 2), "key_weights"), (dict(n_rows=0), "empty key_weights"), (dict(width=0), "empty key_weights"),
    (dict(cu_new=None), "null"), (dict(cu_k=None), "null"), (dict(hk=0), "65535"), (dict(hk=70000), "65535"),
    (dict(batch=70000), "65535")])
def test_c_clear_refusals(kw, match):
    _einval(_lib.load().vox_clear_key_weights(*{**CLEAR_C, **kw}.values()), match)


def test_c_clear_of_nothing():
    for kw in (dict(batch=0), dict(max_keys=0), dict(max_tokens=0)):
        assert _lib.load().vox_clear_key_weights(*{**CLEAR_C, "w": None, **kw}.values()) == _lib.VOX_OK
