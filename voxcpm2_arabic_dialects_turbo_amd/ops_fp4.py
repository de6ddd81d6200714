"""The attention operators over KV caches held in 4 bits: rows quantised into the cache, read back, and attended over.

A 4-bit cache is a uint8 tensor [num_blocks, block_size, HK, 68], contiguous, for keys and one for values: per token and
kv head 128 channels in the OCP MXFP4 format, 64 bytes of codes and 4 scales (0.27 of bf16's bytes). Every 32 channels
share a power of two; a value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 times it, with a sign. The last two dimensions do not
say where the bytes are: a block's bytes are its codes [block_size][HK][64], then its scales [block_size][HK][4]
(``fp4_parts`` gives both as views). ``runner.allocate_kv_cache(..., dtype=torch.float4_e2m1fn_x2)`` makes such caches,
and ``Attention.forward``, ``store_kvcache``, ``flash_attn_varlen_func`` and ``flash_attn_with_kvcache`` take them.

The attention is over the values that the cache holds, in bf16 arithmetic with fp32 sums as over a bf16 cache; new tokens
count as they were stored. Like the operators of ``ops``, these run on torch's current stream of the tensors' device,
allocate with torch, never synchronize and can be captured into HIP graphs. head_dim 128, block_size a multiple of 64.

No reference counterpart: the reference's caches are bf16.
"""

from __future__ import annotations

import contextlib

import torch

from . import _lib
from .ops import (HEAD_DIM, MAX_DECODE_HEADS, _SCOPE, _as_i32, _check_cuda, _flat, _plan_mode, _plan_recorded,
                  _takes_decode_rows, decode_workspace)

ROW_BYTES = 68  # of a token's head: 64 of codes, 4 of scales

_SAME_DEVICE = contextlib.nullcontext()
# without the check that torch is initialised, where this torch has it (0.1 us against 0.3): the calls have GPU tensors
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _on(dev: torch.device):
    """The context a launch on ``dev`` needs: none where it is the current device."""
    return _SAME_DEVICE if dev.index is None or dev.index == _current_device() else torch.cuda.device(dev)


def is_fp4_cache(cache: torch.Tensor) -> bool:
    """Whether ``cache`` is a 4-bit plane [num_blocks, block_size, HK, 68]."""
    return cache.dtype == torch.uint8 and cache.dim() == 4 and cache.shape[3] == ROW_BYTES


def fp4_parts(cache: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes [num_blocks, block_size, HK, 64] and the scales [num_blocks, block_size, HK, 4] of a 4-bit plane, as views
    of its memory."""
    blocks, bs, hk = _cache_shape(cache, cache)
    per = bs * hk * ROW_BYTES
    at = cache.storage_offset()
    return (cache.as_strided((blocks, bs, hk, 64), (per, hk * 64, 64, 1), at),
            cache.as_strided((blocks, bs, hk, 4), (per, hk * 4, 4, 1), at + bs * hk * 64))


def _cache_shape(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int]:
    """(num_blocks, block_size, HK) of a pair of 4-bit planes."""
    shape = k_cache.shape
    if len(shape) == 4 and shape[3] == ROW_BYTES and v_cache.shape == shape and k_cache.dtype == v_cache.dtype == torch.uint8 \
            and k_cache.is_contiguous() and v_cache.is_contiguous():
        return shape[0], shape[1], shape[2]
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise TypeError(f"4-bit caches are uint8, got {k_cache.dtype} and {v_cache.dtype}")
    if len(shape) != 4 or shape[3] != ROW_BYTES or v_cache.shape != shape:
        raise ValueError(f"4-bit caches must both be [num_blocks, block_size, HK, {ROW_BYTES}], got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    raise ValueError("4-bit caches must be contiguous")


def _rows(fn: str, key: torch.Tensor, value: torch.Tensor, hk: int) -> tuple[int, int, int]:
    """Key and value rows [N, hk, 128] bf16 with heads contiguous; token rows may be strided. N and the row strides."""
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise TypeError(f"{fn}: key and value must be bf16, got {key.dtype} and {value.dtype}")
    shape = key.shape
    if len(shape) != 3 or shape[1] != hk or shape[2] != HEAD_DIM or shape != value.shape:
        raise ValueError(f"{fn}: key and value must be [N, {hk}, {HEAD_DIM}], got {tuple(key.shape)} and "
                         f"{tuple(value.shape)}")
    ks, vs = key.stride(), value.stride()
    for s in (ks, vs):
        if s[2] != 1 or (s[1] != HEAD_DIM and hk > 1):
            raise ValueError(f"{fn}: key and value heads must be contiguous, got strides {s}")
    n = shape[0]
    if n == 1:  # (a single row's stride means nothing)
        return 1, hk * HEAD_DIM, hk * HEAD_DIM
    return n, ks[0], vs[0]


def _row_stride(t: torch.Tensor) -> int:
    """Elements between token rows (a single row's stride means nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def _ids(t: torch.Tensor, name: str) -> torch.Tensor:
    """Slots or block ids as a flat int32 tensor; those that int32 does not hold become ids outside every cache."""
    t = _flat(t)
    return _as_i32(t.clamp(-1, 2 ** 31 - 1) if t.dtype == torch.int64 else t, name)


def _table(block_tables: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A block table as int32 with contiguous rows, and the elements between them."""
    if block_tables.dtype == torch.int32:
        stride, width = block_tables.stride(), block_tables.shape[1]
        if stride[1] == 1 and stride[0] >= width:
            return block_tables, stride[0]
    bt = _ids(block_tables, "block_tables").view(block_tables.shape)
    return bt, bt.shape[1]


def store_kvcache_fp4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor) -> None:
    """Quantises key[i] / value[i] ([N, HK, 128] bf16, token rows may be strided) into slot slot_mapping[i] of the 4-bit
    caches; slots outside them (-1: padding) store nothing. A group of 32 channels gets the least power of two (2^-126
    at least, 2^125 at most: finite rows stay finite) that leaves its largest magnitude at most 7 times it, and every value
    the nearest of the grid, ties to the even code, at most 6; a group that holds an infinity or NaN stands for NaN. A slot
    that occurs twice holds a mix of its rows."""
    blocks, bs, hk = _cache_shape(k_cache, v_cache)
    n, key_stride, value_stride = _rows("store_kvcache_fp4", key, value, hk)
    if slot_mapping.numel() != n:
        raise ValueError("store_kvcache_fp4: slot_mapping must hold one slot per token")
    if n == 0:
        return
    dev = _check_cuda(key, value, k_cache, v_cache, slot_mapping)
    if key_stride == 0 or value_stride == 0:  # one row for every token
        key, value = key.contiguous(), value.contiguous()
        key_stride = value_stride = hk * HEAD_DIM
    slots = _ids(slot_mapping, "slot_mapping")
    lib = _lib.load()
    with _on(dev):
        _lib.check(lib.vox_store_kvcache_fp4(key.data_ptr(), value.data_ptr(), key_stride, value_stride,
                                             k_cache.data_ptr(), v_cache.data_ptr(), blocks, bs, slots.data_ptr(), n,
                                             hk, HEAD_DIM, _lib.stream_handle(dev)), "store_kvcache_fp4")


def load_kvcache_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor
                     ) -> tuple[torch.Tensor, torch.Tensor]:
    """The key and value rows held at ``slots`` ([N], any order, repeats allowed) as bf16 [N, HK, 128]: exact, zeros for
    slots outside the cache."""
    blocks, bs, hk = _cache_shape(k_cache, v_cache)
    dev = _check_cuda(k_cache, v_cache, slots)
    at = _ids(slots, "slots")
    n = at.numel()
    key, value = torch.empty(2, n, hk, HEAD_DIM, dtype=torch.bfloat16, device=dev).unbind(0)
    if n:
        lib = _lib.load()
        with _on(dev):
            _lib.check(lib.vox_load_kvcache_fp4(k_cache.data_ptr(), v_cache.data_ptr(), blocks, bs, at.data_ptr(), n, hk,
                                                HEAD_DIM, key.data_ptr(), value.data_ptr(), _lib.stream_handle(dev)),
                       "load_kvcache_fp4")
    return key, value


def _workspace(lib, dev: torch.device, batch: int, plan, *shape) -> tuple[torch.Tensor, int, object]:
    """The scratch of a decode call over ``batch`` sequences, then its plan mode and key as ``_plan_mode`` gives them. Without a
    plan the scratch is the call's own (in a captured graph, the graph's); with one it is the device's decode workspace, which
    keeps the records."""
    if plan is None:
        return torch.empty(lib.vox_decode_workspace_bytes(batch), dtype=torch.uint8, device=dev), _lib.PLAN_NONE, None
    return decode_workspace(dev), *_plan_mode(dev, plan, *shape)


def decode_attention_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, context_lens: torch.Tensor,
                         block_tables: torch.Tensor, softmax_scale: float, out: torch.Tensor | None = None,
                         key: torch.Tensor | None = None, value: torch.Tensor | None = None,
                         slot_mapping: torch.Tensor | None = None, plan=None) -> torch.Tensor:
    """``ops.decode_attention`` over 4-bit caches: q [B, H, 128] bf16 (sequence rows may be strided), one query per
    sequence over its first context_lens[b] cached tokens; o [B, H, 128] bf16, zeros where context_lens[b] is 0. Up to 16
    query heads over 1 or 2 kv heads.

    With key / value ([B, HK, 128]) and slot_mapping ([B]) the step's rows are stored in the same call: the result (and the
    caches afterwards) are those of ``store_kvcache_fp4`` followed by this attention, as long as no sequence's slot lies
    inside another sequence's context. ``softmax_scale`` is positive. ``plan``: as decode_attention's; planned calls of one
    device share a workspace with each other and with unplanned calls over bf16 caches, and must not overlap those."""
    blocks, bs, hk = _cache_shape(k_cache, v_cache)
    if q.dim() != 3 or q.dtype != torch.bfloat16:
        raise TypeError(f"decode_attention_fp4: q must be bf16 [B, H, {HEAD_DIM}], got {q.dtype} {tuple(q.shape)}")
    B, H, D = q.shape
    qs = q.stride()
    if D != HEAD_DIM or qs[2] != 1 or (qs[1] != D and H > 1):
        raise ValueError(f"q must be [B, H, {HEAD_DIM}] with contiguous heads, got {tuple(q.shape)} {q.stride()}")
    if hk not in (1, 2) or H == 0 or H % hk or H > MAX_DECODE_HEADS:
        raise ValueError(f"decode supports H <= {MAX_DECODE_HEADS} query heads over 1 or 2 KV heads, got {H}/{hk}")
    if context_lens.numel() != B or block_tables.dim() != 2 or block_tables.shape[0] < B:
        raise ValueError("context_lens must be [B] and block_tables [B, max_blocks]")
    dev = _check_cuda(q, k_cache, v_cache, context_lens, block_tables)
    if out is None:
        out = torch.empty(B, H, D, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out must be a contiguous bf16 [{B}, {H}, {D}] on {dev}")
    if key is not None:
        if value is None or slot_mapping is None:
            raise ValueError("decode_attention_fp4: key, value and slot_mapping go together")
        _check_cuda(q, key, value, slot_mapping)
        rows, key_stride, value_stride = _rows("decode_attention_fp4", key, value, hk)
        if rows != B or slot_mapping.numel() != B:
            raise ValueError(f"decode_attention_fp4: key, value and slot_mapping must hold {B} rows")
        slots = _ids(slot_mapping, "slot_mapping")
        if key_stride == 0 or value_stride == 0:
            key, value = key.contiguous(), value.contiguous()
            key_stride = value_stride = hk * D
    elif value is not None or slot_mapping is not None:
        raise ValueError("decode_attention_fp4: key, value and slot_mapping go together")
    if B == 0:
        return out
    if qs[0] == 0:
        q = q.contiguous()
    bt, bt_stride = _table(block_tables)
    lens = _as_i32(_flat(context_lens), "context_lens")
    mb = bt.shape[1]
    lib = _lib.load()
    with _on(dev):
        # a record holds the slots of rows that ride (the library stores others by a call of their own)
        rides = plan is not None and key is not None and (key.data_ptr() | value.data_ptr()) % 16 == 0 \
            and (key_stride | value_stride) % 8 == 0
        ws, mode, recorded = _workspace(lib, dev, B, plan, "decode_fp4", rides, B, mb, bt_stride, H, hk, bs)
        if key is None:
            _lib.check(lib.vox_decode_attn_fp4(q.data_ptr(), _row_stride(q), k_cache.data_ptr(), v_cache.data_ptr(), blocks,
                                               bs, bt.data_ptr(), bt_stride, mb, lens.data_ptr(), B, H, hk, D,
                                               float(softmax_scale), mode, ws.data_ptr(), ws.numel(), out.data_ptr(),
                                               _lib.stream_handle(dev)), "decode_attn_fp4")
            _plan_recorded(dev, recorded)
            return out
        _lib.check(lib.vox_decode_attn_store_fp4(q.data_ptr(), _row_stride(q), key.data_ptr(), value.data_ptr(),
                                                 key_stride, value_stride, slots.data_ptr(),
                                                 k_cache.data_ptr(), v_cache.data_ptr(), blocks, bs, bt.data_ptr(),
                                                 bt_stride, mb, lens.data_ptr(), B, H, hk, D, float(softmax_scale), mode,
                                                 ws.data_ptr(), ws.numel(), out.data_ptr(), _lib.stream_handle(dev)),
                   "decode_attn_store_fp4")
        _plan_recorded(dev, recorded)
    return out


def varlen_attention_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, cu_seqlens_q: torch.Tensor,
                         cu_seqlens_k: torch.Tensor, max_seqlen_q: int, block_table: torch.Tensor, softmax_scale: float,
                         causal: bool = True, out: torch.Tensor | None = None, plan=None) -> torch.Tensor:
    """``ops.varlen_attention`` over 4-bit caches through a block table: q [T, H, 128] bf16 (token rows may be strided), the
    queries of sequence b the last of its cu_seqlens_k[b + 1] - cu_seqlens_k[b] cached tokens (bottom-right causal, or
    every key where ``causal`` is false); o [T, H, 128] bf16, zeros for a query that sees no key. H / HK divides 128.
    One-query sequences run on the decode kernels where the call is mostly those. ``softmax_scale`` and ``plan``: as
    decode_attention_fp4's."""
    blocks, bs, hk = _cache_shape(k_cache, v_cache)
    if q.dim() != 3 or q.dtype != torch.bfloat16:
        raise TypeError(f"varlen_attention_fp4: q must be bf16 [T, H, {HEAD_DIM}], got {q.dtype} {tuple(q.shape)}")
    T, H, D = q.shape
    qs = q.stride()
    if D != HEAD_DIM or qs[2] != 1 or (qs[1] != D and H > 1):
        raise ValueError(f"q must be [T, H, {HEAD_DIM}] with contiguous heads, got {tuple(q.shape)} {q.stride()}")
    if hk == 0 or H == 0 or H % hk:
        raise ValueError(f"num_heads {H} is not a multiple of num_kv_heads {hk}")
    B = cu_seqlens_q.numel() - 1
    if cu_seqlens_k.numel() != B + 1:
        raise ValueError("cu_seqlens_k must have as many entries as cu_seqlens_q")
    if block_table.dim() != 2 or block_table.shape[0] < B:
        raise ValueError("block_table must be [B, max_blocks]")
    dev = _check_cuda(q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, block_table)
    if out is None:
        out = torch.empty(T, H, D, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or out.stride(1) != D or out.device != dev:
        raise ValueError(f"out must be a bf16 [{T}, {H}, {D}] with contiguous heads on {dev}")
    if T == 0 or B <= 0 or max_seqlen_q <= 0:
        return out
    if qs[0] == 0:
        q = q.contiguous()
    cu_q, cu_k = _as_i32(cu_seqlens_q, "cu_seqlens_q"), _as_i32(cu_seqlens_k, "cu_seqlens_k")
    bt, bt_stride = _table(block_table)
    mb = bt.shape[1]
    lib = _lib.load()
    with _on(dev):
        ws, mode, recorded = None, _lib.PLAN_NONE, None
        if (max_seqlen_q == 1 or 4 * T <= B * max_seqlen_q) and _takes_decode_rows(H, hk, bs, mb, out, _row_stride(out)):
            if plan is None:
                plan = getattr(_SCOPE, "key", None)
            ws, mode, recorded = _workspace(lib, dev, B, plan, "varlen_fp4", B, mb, bt_stride, H, hk, bs, max_seqlen_q > 1)
        _lib.check(lib.vox_prefill_attn_fp4(q.data_ptr(), _row_stride(q), k_cache.data_ptr(), v_cache.data_ptr(), blocks, bs,
                                            bt.data_ptr(), bt_stride, mb, cu_q.data_ptr(), cu_k.data_ptr(), B,
                                            int(max_seqlen_q), T, H, hk, D, float(softmax_scale), 1 if causal else 0,
                                            out.data_ptr(), _row_stride(out), mode, None if ws is None else ws.data_ptr(),
                                            0 if ws is None else ws.numel(), _lib.stream_handle(dev)),
                   "prefill_attn_fp4")
        _plan_recorded(dev, recorded)
    return out
