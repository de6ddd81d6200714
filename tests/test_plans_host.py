"""Which plan mode a call asks the library for, on the CPU with the library recorded: a plan is reused only where a call
before has recorded it, in the same form, and nothing has taken the workspace since."""

from __future__ import annotations

import pytest
import torch

from voxcpm2_arabic_dialects_turbo_amd import _lib, ops, ops_fp4

BF16, U8, I32 = torch.bfloat16, torch.uint8, torch.int32
NONE, RECORD, REUSE = _lib.PLAN_NONE, _lib.PLAN_RECORD, _lib.PLAN_REUSE
# where the plan mode stands among a function's arguments
PLAN_ARG = dict(vox_decode_attn=15, vox_decode_attn_store=20, vox_prefill_attn=26, vox_prefill_attn_store_paged=26,
                vox_decode_attn_fp4=15, vox_decode_attn_store_fp4=20, vox_prefill_attn_fp4=21)
H, HK, D, BS, B = 16, 2, 128, 64, 3


class _Library:
    """Takes every call, keeps the plan modes, answers `status`."""

    def __init__(self):
        self.modes, self.status = [], _lib.VOX_OK

    def __getattr__(self, name):
        def call(*args):
            if name == "vox_decode_workgroups":
                return 256
            if name.endswith("_bytes"):
                return 256
            if name == "vox_last_error":
                return b"refused"
            if name in PLAN_ARG:
                self.modes.append(args[PLAN_ARG[name]])
            return self.status
        return call


@pytest.fixture
def lib(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(_lib, "capture_id", lambda stream: 0)
    for module in (ops, ops_fp4):
        monkeypatch.setattr(module, "_check_cuda", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(ops, "_device_index", lambda dev: 0)
    monkeypatch.setattr(ops, "_WORKSPACE", {})
    monkeypatch.setattr(ops, "_PLANNED", {})
    return lib


def _cache(fp4):
    return torch.zeros(4, BS, HK, 68, dtype=U8) if fp4 else torch.zeros(4, BS, HK, D, dtype=BF16)


def _rows(n, aligned=True):
    """[n, HK, 128] rows, or such that start 2 bytes behind a 16-byte border."""
    off = 0 if aligned else 1
    return torch.zeros(n * HK * D + 8, dtype=BF16)[off:off + n * HK * D].view(n, HK, D)


def _decode(fp4, plan, rows=None, lens=None, batch=B, **kw):
    c, i = _cache(fp4), torch.zeros(batch, dtype=I32)
    fn = ops_fp4.decode_attention_fp4 if fp4 else ops.decode_attention
    if rows is not None:
        kw.update(key=rows, value=rows, slot_mapping=i)
    return fn(torch.zeros(batch, H, D, dtype=BF16), c, c, i, torch.zeros(batch, 2, dtype=I32), 0.1, plan=plan, **kw)


@pytest.mark.parametrize("fp4", [False, True])
def test_a_plan_recorded_without_rows_is_not_reused_with_them(lib, fp4):
    """A record holds the new tokens' slots, so each form records its own."""
    for rows in (None, None, _rows(B), _rows(B), None):
        _decode(fp4, "step", rows)
    assert lib.modes == [RECORD, REUSE, RECORD, REUSE, RECORD]


def test_rows_that_do_not_ride_do_not_share_the_riding_rows_plan(lib):
    """Rows that are not 16-byte aligned are stored by a call of their own: the attention's record has no slots."""
    for rows in (_rows(B, False), _rows(B, False), _rows(B), _rows(B), _rows(B, False), None):
        _decode(True, "step", rows)
    assert lib.modes == [RECORD, REUSE, RECORD, REUSE, RECORD, REUSE]


def test_one_row_for_every_sequence_rides(lib):
    for _ in range(2):
        _decode(True, "step", _rows(1).expand(B, HK, D))
    _decode(True, "step", _rows(B))
    assert lib.modes == [RECORD, REUSE, REUSE]


def _varlen(fp4, plan, out=None, max_q=1, block_size=BS, hk=HK):
    width = (68, U8) if fp4 else (D, BF16)
    c = torch.zeros(4, block_size, hk, width[0], dtype=width[1])
    cu, kw = torch.arange(B + 1, dtype=I32), dict(softmax_scale=0.1, causal=True, plan=plan, out=out, max_seqlen_q=max_q)
    q, bt = torch.zeros(B, H, D, dtype=BF16), torch.zeros(B, 2, dtype=I32)
    if fp4:
        return ops_fp4.varlen_attention_fp4(q, c, c, cu_seqlens_q=cu, cu_seqlens_k=cu, block_table=bt, **kw)
    return ops.varlen_attention(q, None, None, cu_seqlens_q=cu, cu_seqlens_k=cu, block_table=bt, k_cache=c, v_cache=c, **kw)


def _prefill_store(_, plan, out=None):
    c, cu, rows = _cache(False), torch.arange(B + 1, dtype=I32), _rows(B)
    return ops.prefill_attention_store(torch.zeros(B, H, D, dtype=BF16), rows, rows, c, c, cu[:B], cu_seqlens_q=cu,
                                       cu_seqlens_k=cu, max_seqlen_q=1, softmax_scale=0.1, plan=plan, out=out,
                                       block_table=torch.zeros(B, 2, dtype=I32))


CALLS = pytest.mark.parametrize("call,fp4", [(_decode, False), (_decode, True), (_varlen, False), (_varlen, True),
                                             (_prefill_store, False)])
VARLEN = pytest.mark.parametrize("call,fp4", [(_varlen, False), (_varlen, True), (_prefill_store, False)])


@CALLS
def test_a_refused_call_has_recorded_nothing(lib, call, fp4):
    """The next call with its plan records: the workspace may hold another step's records."""
    for status in (_lib.VOX_EINVAL, _lib.VOX_EHIP):
        call(fp4, "before")
        lib.status = status
        with pytest.raises((ValueError, _lib.VoxAttnError)):
            call(fp4, "step")
        lib.status = _lib.VOX_OK
        lib.modes.clear()
        call(fp4, "step")
        call(fp4, "step")
        assert lib.modes == [RECORD, REUSE]


@CALLS
def test_a_refused_reuse_keeps_the_record(lib, call, fp4):
    call(fp4, "step")
    lib.status = _lib.VOX_EINVAL
    with pytest.raises(ValueError):
        call(fp4, "step")
    lib.status = _lib.VOX_OK
    call(fp4, "step")
    assert lib.modes == [RECORD, REUSE, REUSE]


@VARLEN
def test_calls_whose_outputs_the_decode_kernels_cannot_write_record_nothing(lib, call, fp4):
    """An output 8 bytes behind a 16-byte border, or with rows an odd number of 8 bytes apart, is the prefill kernel's in every
    row: no plan, whatever the workspace holds, and none forgotten."""
    call(fp4, "before")
    for out in (torch.zeros(B * H * D + 4, dtype=BF16)[4:].view(B, H, D),
                torch.zeros(B, H * D + 4, dtype=BF16)[:, :H * D].view(B, H, D)):
        lib.modes.clear()
        call(fp4, "step", out=out)
        call(fp4, "before")
        assert lib.modes == [NONE, REUSE]
    lib.modes.clear()
    call(fp4, "step", out=torch.zeros(B, H, D, dtype=BF16))
    call(fp4, "step")
    assert lib.modes == [RECORD, REUSE]


def test_shapes_that_the_decode_kernels_do_not_take_record_nothing(lib):
    for kw in (dict(block_size=48), dict(hk=4)):
        lib.modes.clear()
        _varlen(False, "before")
        _varlen(False, "step", **kw)
        _varlen(False, "before")
        assert lib.modes == [RECORD, NONE, REUSE]
        ops.forget_plans()


@pytest.mark.parametrize("call,fp4", [(_decode, False), (_varlen, False), (_prefill_store, False)])
@pytest.mark.parametrize("planned,fp4_planned", [(_decode, False), (_decode, True), (_varlen, False), (_varlen, True),
                                                 (_prefill_store, False)])
def test_an_unplanned_call_on_the_shared_workspace_ends_the_plan(lib, call, fp4, planned, fp4_planned):
    """It writes its own step layout and partials where the records and layout of the plan are."""
    planned(fp4_planned, "step")
    call(fp4, None)
    planned(fp4_planned, "step")
    planned(fp4_planned, "step")
    assert lib.modes == [RECORD, NONE, RECORD, REUSE]


@pytest.mark.parametrize("call", [_decode, _varlen])
def test_an_unplanned_4_bit_call_has_scratch_of_its_own(lib, call):
    _decode(False, "step")
    call(True, None)
    _decode(False, "step")
    assert lib.modes == [RECORD, NONE, REUSE]
