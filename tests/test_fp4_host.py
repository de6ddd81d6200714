"""4-bit caches and the care of blocks on the CPU: the format's oracle against known answers, allocation, dispatch, and the
refusals of the operators and of the C ABI (nothing is launched)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import fp4, kvpages
from voxcpm2_arabic_dialects_turbo_amd import _lib, layers, ops, ops_fp4, runner
from voxcpm2_arabic_dialects_turbo_amd.context import reset_context, set_context
from voxcpm2_arabic_dialects_turbo_amd.kernels import kv_copy, kv_pages
from voxcpm2_arabic_dialects_turbo_amd.layers import Attention
from voxcpm2_arabic_dialects_turbo_amd.ops_fp4 import _ids, _table

BF16, U8, I32 = torch.bfloat16, torch.uint8, torch.int32


def test_oracle_known_answers():
    """The grid itself is held exactly; 7 is the largest that 6 stands for at its scale; ties go to the even code."""
    x = torch.zeros(1, 1, 128)
    x[0, 0, :9] = torch.tensor([6.0, -0.25, 0.75, 1.25, -1.75, 2.5, 3.5, 5.0, 0.26])
    x[0, 0, 32], x[0, 0, 64], x[0, 0, 96] = 7.0, 7.03125, 2.0 ** -140
    codes, scales = fp4.quantize(x)
    assert scales.tolist() == [[[127, 127, 128, 1]]]
    v = fp4.values(codes, scales)[0, 0]
    assert v[:9].tolist() == [6.0, 0.0, 1.0, 1.0, -2.0, 2.0, 4.0, 4.0, 0.5]
    assert v[32] == 6.0 and v[64] == 8.0 and v[96] == 0.0
    assert codes[0, 0, 0] == 0x87  # 6 in the low nibble, -0 in the high one
    x[0, 0, 33] = float("nan")
    codes, scales = fp4.quantize(x)
    assert scales[0, 0].tolist() == [127, 255, 128, 1] and fp4.values(codes, scales)[0, 0, 32:64].isnan().all()


def test_quantize_is_the_nearest_of_the_grid():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(4, 2, 128, generator=gen).to(BF16)
    codes, scales = fp4.quantize(x)
    v, s = fp4.values(codes, scales), torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    assert ((v - x.double()).abs() <= s * torch.where(x.double().abs() > 4 * s, 1.0, torch.where(
        x.double().abs() > 2 * s, 0.5, 0.25))).all()
    again = fp4.quantize(v)
    assert torch.equal(fp4.values(*again), v)


def test_parts_are_views_of_the_bytes():
    planes = torch.arange(2 * 3 * 64 * 2 * 68).remainder(251).to(U8).view(2, 3, 64, 2, 68)
    for plane in planes:
        codes, scales = ops_fp4.fp4_parts(plane)
        want = fp4.parts(plane)
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
        assert torch.equal(fp4.plane(*want), plane)
    scales.zero_()
    assert fp4.parts(planes[1])[1].sum() == 0 and fp4.parts(planes[0])[1].sum() > 0


def test_allocate_4_bit_caches():
    mods = [Attention(16, 128, 0.1, 2) for _ in range(3)]
    kv = runner.allocate_kv_cache(mods, 5, 256, dtype=torch.float4_e2m1fn_x2, device="cpu")
    assert kv.shape == (3, 2, 5, 256, 2, 68) and kv.dtype == U8
    assert mods[1].v_cache.data_ptr() == kv[1, 1].data_ptr() and ops_fp4.is_fp4_cache(mods[1].v_cache)
    assert kv.numel() == 5 * runner.kv_cache_block_bytes(mods, 256, torch.float4_e2m1fn_x2)
    other = [Attention(16, 128, 0.1, 2), Attention(8, 128, 0.1, 1)]
    assert runner.allocate_kv_cache(other, 2, 256, dtype=torch.float4_e2m1fn_x2, device="cpu") is None
    assert other[1].k_cache.shape == (2, 256, 1, 68)
    with pytest.raises(ValueError, match="head_dim"):
        runner.allocate_kv_cache([Attention(4, 64, 0.1, 2)], 2, 256, dtype=torch.float4_e2m1fn_x2, device="cpu")
    assert runner.kv_cache_block_bytes(mods, 256) == 3 * 2 * 256 * 2 * 128 * 2


def _record(monkeypatch, module, *names):
    calls = []
    for name in names:
        def fake(*args, _name=name, **kw):
            calls.append((_name, args, kw))
            return torch.zeros(args[0].shape, dtype=BF16)
        monkeypatch.setattr(module, name, fake)
    return calls


def test_attention_forward_takes_4_bit_caches(monkeypatch):
    """Decode steps store and attend in one call; prefills store, then attend over the caches where the context has block
    tables, else over the step's rows."""
    calls = _record(monkeypatch, layers, "decode_attention_fp4", "store_kvcache", "flash_attn_varlen_func",
                    "decode_attention", "prefill_attention_store")
    m = Attention(16, 128, 0.1, 2)
    runner.allocate_kv_cache([m], 4, 256, dtype=torch.float4_e2m1fn_x2, device="cpu")
    q, k = torch.zeros(3, 16, 128, dtype=BF16), torch.zeros(3, 2, 128, dtype=BF16)
    slots, lens, tables = (torch.zeros(s, dtype=I32) for s in ((3,), (3,), (3, 1)))
    try:
        set_context(False, slot_mapping=slots, context_lens=lens, block_tables=tables)
        assert m(q, k, k).shape == (3, 1, 16, 128)
        (name, args, kw), = calls
        assert name == "decode_attention_fp4" and args[1] is m.k_cache and kw["slot_mapping"] is slots and kw["plan"]
        for bt in (None, tables):
            calls.clear()
            set_context(True, lens, lens, 3, 3, slots, None, bt)
            m(q, k, k)
            assert [c[0] for c in calls] == ["store_kvcache", "flash_attn_varlen_func"]
            assert calls[1][1][1] is (k if bt is None else m.k_cache) and calls[1][2]["block_table"] is bt
    finally:
        reset_context()


def test_entry_points_hand_4_bit_caches_on(monkeypatch):
    calls = _record(monkeypatch, ops_fp4, "store_kvcache_fp4", "varlen_attention_fp4", "decode_attention_fp4")
    cache = torch.zeros(2, 64, 2, 68, dtype=U8)
    q, k = torch.zeros(4, 16, 128, dtype=BF16), torch.zeros(4, 2, 128, dtype=BF16)
    i = torch.zeros(3, dtype=I32)
    ops.store_kvcache(k, k, cache, cache, i)
    ops.flash_attn_varlen_func(q, cache, cache, i, i, 2, 2, block_table=torch.zeros(2, 1, dtype=I32), causal=True)
    ops.flash_attn_with_kvcache(q[:2, None], cache, cache, cache_seqlens=i[:2], block_table=torch.zeros(2, 1, dtype=I32))
    ops.flash_attn_with_kvcache(q.view(2, 2, 16, 128), cache, cache, cache_seqlens=i[:2],
                                block_table=torch.zeros(2, 1, dtype=I32))
    assert [c[0] for c in calls] == ["store_kvcache_fp4", "varlen_attention_fp4", "decode_attention_fp4",
                                     "varlen_attention_fp4"]


def _args(**over):
    a = dict(cache=torch.zeros(2, 64, 2, 68, dtype=U8), q=torch.zeros(3, 16, 128, dtype=BF16),
             k=torch.zeros(3, 2, 128, dtype=BF16), i=torch.zeros(3, dtype=I32), t=torch.zeros(3, 2, dtype=I32))
    a.update(over)
    return a


@pytest.mark.parametrize("over,error", [
    (dict(cache=torch.zeros(2, 64, 2, 64, dtype=U8)), ValueError),
    (dict(cache=torch.zeros(2, 64, 2, 68, dtype=torch.int8)), TypeError),
    (dict(cache=torch.zeros(2, 64, 2, 128, dtype=BF16)), TypeError),
    (dict(cache=torch.zeros(2, 64, 4, 68, dtype=U8)[:, :, ::2]), ValueError),
    (dict(k=torch.zeros(3, 2, 128)), TypeError),
    (dict(k=torch.zeros(3, 2, 64, dtype=BF16)), ValueError),
    (dict(k=torch.zeros(3, 1, 128, dtype=BF16)), ValueError),
    (dict(k=torch.zeros(3, 128, 2, dtype=BF16).transpose(1, 2)), ValueError),
    (dict(k=torch.zeros(3, 4, 128, dtype=BF16)[:, ::2]), ValueError),
    (dict(i=torch.zeros(4, dtype=I32)), ValueError),
    (dict(), ValueError),  # (on the CPU)
])
def test_store_refusals(over, error):
    a = _args(**over)
    with pytest.raises(error):
        ops_fp4.store_kvcache_fp4(a["k"], a["k"], a["cache"], a["cache"], a["i"])


@pytest.mark.parametrize("over,error", [
    (dict(cache=torch.zeros(2, 64, 2, 128, dtype=BF16)), TypeError),
    (dict(q=torch.zeros(3, 16, 128)), TypeError),
    (dict(q=torch.zeros(3, 16, 64, dtype=BF16)), ValueError),
    (dict(q=torch.zeros(3, 128, 16, dtype=BF16).transpose(1, 2)), ValueError),
    (dict(q=torch.zeros(3, 15, 128, dtype=BF16)), ValueError),
    (dict(i=torch.zeros(5, dtype=I32)), ValueError),
    (dict(t=torch.zeros(1, 2, dtype=I32)), ValueError),
    (dict(), ValueError),  # (on the CPU)
])
def test_attention_refusals(over, error):
    a = _args(**over)
    with pytest.raises(error):
        ops_fp4.decode_attention_fp4(a["q"], a["cache"], a["cache"], a["i"], a["t"], 0.1)
    cu = torch.zeros(a["i"].numel() + 1, dtype=I32) if "i" not in over else a["i"]
    with pytest.raises(error):
        ops_fp4.varlen_attention_fp4(a["q"], a["cache"], a["cache"], cu_seqlens_q=torch.zeros(4, dtype=I32),
                                     cu_seqlens_k=cu, max_seqlen_q=2, block_table=a["t"], softmax_scale=0.1)


@pytest.mark.parametrize("heads,hk", [(17, 1), (32, 2), (8, 4), (0, 1)])
def test_decode_refuses_other_head_layouts(heads, hk):
    a = _args(q=torch.zeros(3, heads, 128, dtype=BF16), cache=torch.zeros(2, 64, hk, 68, dtype=U8))
    with pytest.raises(ValueError, match="decode supports"):
        ops_fp4.decode_attention_fp4(a["q"], a["cache"], a["cache"], a["i"], a["t"], 0.1)


@pytest.mark.parametrize("shape,dtype", [((2, 4, 64, 1, 128), BF16), ((1, 3, 4, 64, 1, 128), BF16), ((1, 2, 4, 64, 1, 64), U8)])
def test_pages_refuse_other_caches(shape, dtype):
    kv, t, i = torch.zeros(shape, dtype=dtype), torch.zeros(2, 2, dtype=I32), torch.zeros(2, dtype=I32)
    with pytest.raises(ValueError):
        kv_pages.fork_kv_blocks(kv, t, i, i, i)
    with pytest.raises(ValueError):
        kv_pages.compact_kv_blocks(kv, t, i)


def test_pages_refuse_the_cpu_and_bad_tables():
    kv, i = torch.zeros(1, 2, 4, 64, 1, 128, dtype=BF16), torch.zeros(2, dtype=I32)
    with pytest.raises(ValueError, match="GPU"):
        kv_pages.compact_kv_blocks(kv, torch.zeros(2, 2, dtype=I32), i)
    with pytest.raises(ValueError, match="contiguous"):
        kv_pages.compact_kv_blocks(kv[:, :, ::2], torch.zeros(2, 2, dtype=I32), i)
    with pytest.raises(ValueError, match="on a GPU"):
        kv_copy.copy_kv_block_prefix(torch.zeros(1, 2, 4, 64, 1, 68, dtype=U8), [(0, 1, 5)])


def test_oracle_compaction_by_hand():
    kv = torch.arange(6.0).view(1, 1, 6, 1, 1, 1).expand(1, 2, 6, 1, 1, 1).clone()
    new, remap, live = kvpages.compact(kv, [[5, 0], [4, 5]], [2, 1])
    assert (new, remap, live) == ([[2, 0], [1, -1]], [0, -1, -1, -1, 1, 2], 3)
    assert kv[0, 0, remap[5], 0, 0, 0] == 5 and kv[0, 0, remap[4], 0, 0, 0] == 4


# ---------------------------------------------------------------------------------------------------------------------
# the C ABI


P = ctypes.c_void_p(256)  # never dereferenced: the checks fail first


def _err():
    return _lib.load().vox_last_error().decode()


def _call(name, args, over):
    a = dict(args, **over)
    return getattr(_lib.load(), name)(*a.values())


STORE = dict(key=P, value=P, ks=256, vs=256, kc=P, vc=P, blocks=4, bs=64, slots=P, n=3, hk=2, d=128, stream=None)
LOAD = dict(kc=P, vc=P, blocks=4, bs=64, slots=P, n=3, hk=2, d=128, key=P, value=P, stream=None)
DECODE = dict(q=P, qs=2048, kc=P, vc=P, blocks=4, bs=64, bt=P, bts=4, mb=4, lens=P, batch=2, h=16, hk=2, d=128, scale=0.1,
              plan=0, ws=P, wsb=1 << 30, out=P, stream=None)
STORES = dict(q=P, qs=2048, key=P, value=P, ks=256, vs=256, slots=P, kc=P, vc=P, blocks=4, bs=64, bt=P, bts=4, mb=4,
              lens=P, batch=2, h=16, hk=2, d=128, scale=0.1, plan=0, ws=P, wsb=1 << 30, out=P, stream=None)
VARLEN = dict(q=P, qs=2048, kc=P, vc=P, blocks=4, bs=64, bt=P, bts=4, mb=4, cq=P, ck=P, batch=2, mq=7, n=9, h=16, hk=2,
              d=128, scale=0.1, causal=1, out=P, os=2048, plan=0, ws=None, wsb=0, stream=None)
CACHE = [dict(kc=None), dict(vc=ctypes.c_void_p(8)), dict(bs=32), dict(bs=0), dict(blocks=0), dict(d=64), dict(hk=0),
         dict(blocks=1 << 40)]


@pytest.mark.parametrize("name,args,over", [
    *(("vox_store_kvcache_fp4", STORE, o) for o in CACHE + [dict(n=-1), dict(key=None), dict(slots=None), dict(ks=128)]),
    *(("vox_load_kvcache_fp4", LOAD, o) for o in CACHE + [dict(n=-1), dict(key=None), dict(value=ctypes.c_void_p(2))]),
    *(("vox_decode_attn_fp4", DECODE, o) for o in CACHE + [
        dict(batch=-1), dict(plan=3), dict(q=None), dict(h=17), dict(hk=4), dict(mb=0), dict(bts=2), dict(ws=None),
        dict(wsb=16), dict(scale=float("nan")), dict(out=ctypes.c_void_p(8)), dict(qs=2052), dict(mb=1 << 25, bts=1 << 25)]),
    *(("vox_decode_attn_store_fp4", STORES, o) for o in CACHE + [
        dict(key=None), dict(slots=None), dict(ks=10), dict(ws=None), dict(h=17), dict(plan=-1)]),
    *(("vox_prefill_attn_fp4", VARLEN, o) for o in CACHE + [
        dict(batch=-1), dict(n=-1), dict(mq=-1), dict(q=None), dict(bt=None), dict(cq=None), dict(out=None), dict(os=100),
        dict(os=2050), dict(h=15), dict(h=24), dict(batch=70000), dict(scale=float("inf")), dict(qs=2051),
        dict(mb=1 << 25, bts=1 << 25), dict(ws=P, wsb=16)]),
])
def test_c_abi_rejects_bad_arguments_before_launching(name, args, over):
    assert _call(name, args, over) == _lib.VOX_EINVAL
    assert _err()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-39, float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("name,args", [("vox_decode_attn_fp4", DECODE), ("vox_decode_attn_store_fp4", STORES),
                                       ("vox_prefill_attn_fp4", VARLEN)])
def test_c_abi_takes_positive_softmax_scales(name, args, scale):
    assert _call(name, args, dict(scale=scale)) == _lib.VOX_EINVAL
    assert "softmax_scale" in _err()


def test_ids_past_int32_are_outside_every_cache():
    ids = torch.tensor([[0, 5, 2 ** 32 + 5], [-1, -2 ** 40, 2 ** 31]])
    assert _ids(ids, "ids").tolist() == [0, 5, 2 ** 31 - 1, -1, -1, 2 ** 31 - 1]
    table, stride = _table(ids)
    assert table.tolist() == [[0, 5, 2 ** 31 - 1], [-1, -1, 2 ** 31 - 1]] and stride == 3 and table.dtype == torch.int32


@pytest.mark.parametrize("name,args,over", [("vox_store_kvcache_fp4", STORE, dict(n=0)), ("vox_load_kvcache_fp4", LOAD, dict(n=0)),
                                            ("vox_decode_attn_fp4", DECODE, dict(batch=0)),
                                            ("vox_prefill_attn_fp4", VARLEN, dict(n=0)),
                                            ("vox_prefill_attn_fp4", VARLEN, dict(mq=0))])
def test_c_abi_calls_with_nothing_to_do(name, args, over):
    assert _call(name, args, over) == _lib.VOX_OK


COPY = dict(kv=P, planes=4, blocks=9, bs=64, slot=512, scales=0, entries=P, n=2, stream=None)
FORK = dict(kv=P, planes=4, blocks=9, bs=64, slot=512, scales=0, bt=P, bts=4, mb=4, lens=P, batch=2, parents=P, new=P, n=2,
            tables=P, clens=P, stream=None)
COMPACT = dict(kv=P, planes=4, blocks=9, bs=64, slot=512, scales=0, bt=P, bts=4, mb=4, lens=P, batch=2, tables=P, remap=P,
               live=P, moves=P, stream=None)
PAGES = [dict(kv=None), dict(planes=0), dict(planes=70000), dict(blocks=0), dict(bs=0), dict(slot=0), dict(scales=-1),
         dict(kv=ctypes.c_void_p(8)), dict(bs=3, slot=2), dict(blocks=1 << 40), dict(bs=1 << 29)]


@pytest.mark.parametrize("name,args,over", [
    *(("vox_copy_kv_blocks", COPY, o) for o in PAGES + [dict(n=-1), dict(entries=None)]),
    *(("vox_fork_kv_blocks", FORK, o) for o in PAGES + [
        dict(n=-1), dict(batch=-1), dict(bt=None), dict(parents=None), dict(tables=None), dict(mb=0), dict(bts=3),
        dict(mb=1 << 25, bts=1 << 25)]),
    *(("vox_compact_kv_blocks", COMPACT, o) for o in PAGES + [
        dict(batch=-1), dict(bt=None), dict(remap=None), dict(live=None), dict(moves=None), dict(mb=0), dict(bts=3),
        dict(blocks=(1 << 19) + 1), dict(blocks=(1 << 18) + 1)]),
])
def test_c_abi_pages_reject_bad_arguments_before_launching(name, args, over):
    assert _call(name, args, over) == _lib.VOX_EINVAL
    assert _err()
