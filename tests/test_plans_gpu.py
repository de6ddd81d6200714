"""Planned calls over 4-bit caches against the calls they stand for, where a plan's calls differ in form, fail, or have other
calls between them. Tolerances: test_fp4_gpu.py's, or none (the same kernels in the same order)."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as ref
from tests._util import paged_pool, randn
from tests.test_fp4_gpu import BS, D, DEV, SCALE, _check, _cu, _decode_ref, _gen, _pool
from voxcpm2_arabic_dialects_turbo_amd import _lib, ops
from voxcpm2_arabic_dialects_turbo_amd.ops_fp4 import decode_attention_fp4, store_kvcache_fp4, varlen_attention_fp4

pytestmark = pytest.mark.gpu
H, HK = 16, 2


@pytest.fixture(autouse=True)
def _no_plans():
    ops.forget_plans()
    yield
    ops.forget_plans()


def _step(seed, lens):
    """Caches, tables, lengths and slots of a decode step whose sequences end at a new token."""
    gen = _gen(seed)
    kc, vc, tables = _pool(gen, lens, HK)
    slots = torch.tensor([ref.slot_of(tables[b], n - 1, BS) for b, n in enumerate(lens)], dtype=torch.int32)
    return gen, kc, vc, tables, slots


def _new_rows(gen, n, offset):
    """Key and value rows [n, HK, 128], `offset` elements behind a 16-byte border."""
    x = (4 * randn(gen, 2, n * HK * D + 8)).to(DEV)
    return tuple(r[offset:offset + n * HK * D].view(n, HK, D) for r in x)


LENS = [3000, 40, 700, 1, 16, 2222]  # (some cut over workgroups, so that a merge has partials to read)


@pytest.mark.parametrize("forms", [(None, 0), (0, None, 0), (1, 0), (0, 1, 0, None, 0), (None, 1, 0, 0)])
def test_calls_of_other_forms_under_one_plan(forms):
    """Layers of one step under one plan, without rows (None) and with them at an element offset: each is its store followed
    by its attention."""
    gen, kc, vc, tables, slots = _step(900 + len(forms), LENS)
    lens, bt, s = torch.tensor(LENS, dtype=torch.int32, device=DEV), tables.to(DEV), slots.to(DEV)
    for i, form in enumerate(forms):
        q = randn(gen, len(LENS), H, D)
        a, b = (kc.to(DEV), vc.to(DEV)), (kc.to(DEV), vc.to(DEV))
        kw = {}
        if form is not None:
            k, v = _new_rows(gen, len(LENS), form)
            kw = dict(key=k, value=v, slot_mapping=s)
            store_kvcache_fp4(k, v, *b, s)
        o = decode_attention_fp4(q.to(DEV), *a, lens, bt, SCALE, plan="one step", **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        _check(o, *_decode_ref(q, b[0].cpu(), b[1].cpu(), tables, LENS), f"layer {i} of {forms}")


@pytest.mark.parametrize("first,second", [(1, 0), (0, 1), (1, 1), (0, 0)])
def test_the_library_scans_anew_where_a_record_is_of_the_other_form(first, second):
    """vox_decode_attn_store_fp4 recorded with unaligned rows (stored by a call of their own), then reused with aligned ones,
    and the reverse: the caller cannot see which form a call took."""
    lib = _lib.load()
    gen, kc, vc, tables, slots = _step(950, LENS)
    n = len(LENS)
    lens, bt, s = torch.tensor(LENS, dtype=torch.int32, device=DEV), tables.to(DEV), slots.to(DEV)
    ws = torch.zeros(lib.vox_decode_workspace_bytes(n), dtype=torch.uint8, device=DEV)
    for plan, offset in ((_lib.PLAN_RECORD, first), (_lib.PLAN_REUSE, second)):
        q = randn(gen, n, H, D)
        k, v = _new_rows(gen, n, offset)
        a, b, qd = (kc.to(DEV), vc.to(DEV)), (kc.to(DEV), vc.to(DEV)), q.to(DEV)
        store_kvcache_fp4(k, v, *b, s)
        o = torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV)
        _lib.check(lib.vox_decode_attn_store_fp4(
            qd.data_ptr(), H * D, k.data_ptr(), v.data_ptr(), HK * D, HK * D, s.data_ptr(), a[0].data_ptr(), a[1].data_ptr(),
            a[0].shape[0], BS, bt.data_ptr(), bt.shape[1], bt.shape[1], lens.data_ptr(), n, H, HK, D, SCALE, plan,
            ws.data_ptr(), ws.numel(), o.data_ptr(), _lib.stream_handle(o.device)), "decode_attn_store_fp4")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        _check(o, *_decode_ref(q, b[0].cpu(), b[1].cpu(), tables, LENS), f"plan mode {plan}")


OTHER = [700, 3000, 2222, 500, 1, 40]  # (another step of as many sequences)


def _bf16_step(seed, lens):
    gen = _gen(seed)
    kc, vc, tables = paged_pool(gen, lens, sum(-(-n // BS) for n in lens) + 2)
    return gen, kc, vc, tables


def _call(fp4, step, lens, q, plan, scale=SCALE, out=None, varlen=False):
    """One query per sequence of a step, over bf16 or 4-bit caches, as a decode or as a varlen call."""
    kc, vc, bt = step[1].to(DEV), step[2].to(DEV), step[3].to(DEV)
    if not varlen:
        fn = decode_attention_fp4 if fp4 else ops.decode_attention
        return fn(q, kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV), bt, scale, plan=plan, out=out)
    kw = dict(cu_seqlens_q=_cu([1] * len(lens)), cu_seqlens_k=_cu(lens), max_seqlen_q=1, block_table=bt, softmax_scale=scale,
              causal=True, plan=plan, out=out)
    return varlen_attention_fp4(q, kc, vc, **kw) if fp4 else ops.varlen_attention(q, None, None, k_cache=kc, v_cache=vc, **kw)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("varlen", [False, True])
def test_a_plan_whose_first_call_was_refused(fp4, varlen):
    """The workspace holds the records of another step of as many sequences; the refused call has made none."""
    make = _step if fp4 else _bf16_step
    before, now = make(960, OTHER), make(961, LENS)
    q = randn(now[0], len(LENS), H, D).to(DEV)
    want = _call(fp4, now, LENS, q, None, varlen=varlen)
    _call(fp4, before, OTHER, q, "before", varlen=varlen)
    with pytest.raises(ValueError):
        _call(fp4, now, LENS, q, "now", scale=float("nan"), varlen=varlen)
    for _ in range(2):
        assert torch.equal(_call(fp4, now, LENS, q, "now", varlen=varlen), want)


@pytest.mark.parametrize("fp4", [False, True])
def test_a_plan_whose_first_call_took_the_prefill_kernel(fp4):
    """An output 8 bytes behind a 16-byte border is taken, by the kernel that makes no records."""
    make = _step if fp4 else _bf16_step
    before, now = make(970, OTHER), make(971, LENS)
    q = randn(now[0], len(LENS), H, D).to(DEV)
    want = _call(fp4, now, LENS, q, None, varlen=True)
    _call(fp4, before, OTHER, q, "before", varlen=True)
    out = torch.zeros(len(LENS) * H * D + 4, dtype=torch.bfloat16, device=DEV)[4:].view(len(LENS), H, D)
    _call(fp4, now, LENS, q, "now", out=out, varlen=True)
    for _ in range(2):
        assert torch.equal(_call(fp4, now, LENS, q, "now", varlen=True), want)
    # (the two kernels differ by the rounding of probabilities and outputs)
    assert (out.float() - want.float()).abs().max() < 2e-2


@pytest.mark.parametrize("fp4,varlen", [(True, False), (True, True), (False, False), (False, True)])
@pytest.mark.parametrize("others", [[700, 3000, 2222, 500, 1, 40], [900] * 150, [9, 20]])
@pytest.mark.parametrize("other_varlen", [False, True])
def test_unplanned_calls_between_planned_ones(fp4, varlen, others, other_varlen):
    """Unplanned bf16 calls of as many and of other numbers of sequences between the layers of a planned step."""
    step, between = (_step if fp4 else _bf16_step)(980, LENS), _bf16_step(981, others)
    q, p = randn(step[0], len(LENS), H, D).to(DEV), randn(between[0], len(others), H, D).to(DEV)
    want = _call(fp4, step, LENS, q, None, varlen=varlen)
    first = _call(False, between, others, p, None, varlen=other_varlen)
    for _ in range(3):
        assert torch.equal(_call(fp4, step, LENS, q, "step", varlen=varlen), want)
        assert torch.equal(_call(False, between, others, p, None, varlen=other_varlen), first)
    assert torch.equal(_call(fp4, step, LENS, q, "step", varlen=varlen), want)
    assert torch.equal(_call(fp4, step, LENS, q, "step", varlen=varlen), want)
