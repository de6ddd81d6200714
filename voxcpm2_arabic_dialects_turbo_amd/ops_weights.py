"""Attention that also adds up what every cached token receives of it, for eviction by that (kernels.kv_evict).

``key_weights`` is fp32 [rows, HK, width], contiguous, one plane per layer: for the sequence whose row it is and each kv
head, every cached token's sum of probabilities over the kv head's query heads and all queries so far, at the token's
position. ``weight_rows`` (int [B]) says which row is whose, so that streams may come and go in any order; left out,
sequence b has row b, and a row outside [0, rows) (-1) keeps none. No two sequences of a call share a row. The width covers
what the block tables reach (packed keys: max_seqlen_k).

A token that is new in a call starts with what it gets there, whatever its place held; the others get theirs on top. So a
row needs no clearing between the sequences that have it in turn. ``runner.allocate_key_weights`` makes the planes, and
``Attention.forward`` adds to its layer's.

The attention itself is that of ``ops``, or over 4-bit caches of ``ops_fp4``. There a score is off by at most x =
softmax_scale (2^-13 sum |q||k| + 2^-18 max |q| sum |k|), the largest of its row: the scaled MFMA's sum, and what the query's two
8-bit parts leave. A probability is off by at most e^(2x) - 1 of it, beside the roundings in 32 bits. A chunk's are made from
scores in bf16 products over a sum from the scaled MFMA, so those of one query add up to 1 within e^x - 1 only; a decode step's
come from one arithmetic and add up to 1.

Like their operators these run on torch's current stream of the tensors' device, allocate with torch, never synchronize and
can be captured into HIP graphs. head_dim 128, softmax_scale positive. No reference counterpart.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import (HEAD_DIM, MAX_DECODE_HEADS, _as_i32, _check_cuda, _flat, _plan_recorded, _takes_decode_rows,
                  store_kvcache)
from .ops_fp4 import _cache_shape, _ids, _on, _row_stride, _table, _workspace, is_fp4_cache, store_kvcache_fp4


def _weights(fn: str, key_weights: torch.Tensor, weight_rows: torch.Tensor | None, batch: int, hk: int, reach: int,
             index: int) -> tuple[int, int, torch.Tensor | None]:
    """The rows and width of key_weights, and weight_rows as int32 [batch], None where sequence b has row b."""
    if key_weights.dtype != torch.float32:
        raise TypeError(f"{fn}: key_weights must be fp32, got {key_weights.dtype}")
    shape = key_weights.shape
    if len(shape) != 3 or shape[1] != hk or not key_weights.is_contiguous():
        raise ValueError(f"{fn}: key_weights must be contiguous [rows, {hk}, width], got {tuple(shape)}")
    rows, _, width = shape
    if width < reach:
        raise ValueError(f"{fn}: key_weights hold {width} tokens a row, the keys may be {reach}")
    if key_weights.get_device() != index or (weight_rows is not None and weight_rows.get_device() != index):
        raise ValueError(f"{fn}: key_weights and weight_rows must be on the other tensors' GPU")
    if weight_rows is None:
        if rows < batch:
            raise ValueError(f"{fn}: key_weights have {rows} rows for {batch} sequences")
        return rows, width, None
    if weight_rows.numel() != batch:
        raise ValueError(f"{fn}: weight_rows must hold one row per sequence")
    if rows == 0:
        raise ValueError(f"{fn}: key_weights have no rows")
    if weight_rows.dtype == torch.int32 and weight_rows.is_contiguous():
        return rows, width, weight_rows
    return rows, width, _ids(weight_rows, "weight_rows")


def _query(fn: str, q: torch.Tensor, out: torch.Tensor | None, dev: torch.device, contiguous: bool
           ) -> tuple[torch.Tensor, int, torch.Tensor]:
    """q with token rows apart from each other, the elements between them, and where the output goes."""
    n, H, D = q.shape
    s0, s1, s2 = q.stride()
    if D != HEAD_DIM or s2 != 1 or (s1 != D and H > 1):
        raise ValueError(f"{fn}: q must be [rows, H, {HEAD_DIM}] with contiguous heads, got {tuple(q.shape)} {q.stride()}")
    if out is None:
        out = torch.empty((n, H, D), dtype=torch.bfloat16, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1 or out.stride(1) != D \
            or (contiguous and not out.is_contiguous()):
        raise ValueError(f"{fn}: out must be a bf16 [{n}, {H}, {D}] with contiguous heads on {dev}")
    if n == 1:  # (a single row's stride means nothing)
        return q, H * D, out
    return (q, s0, out) if s0 >= H * D else (q.contiguous(), H * D, out)


def _caches(fn: str, k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int]:
    """(num_blocks, block_size, HK) of a pair of bf16 caches."""
    shape = k_cache.shape
    if k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise TypeError(f"{fn} takes bf16 caches or 4-bit ones, got {k_cache.dtype} and {v_cache.dtype}")
    if len(shape) != 4 or shape[3] != HEAD_DIM or v_cache.shape != shape or not (k_cache.is_contiguous()
                                                                                and v_cache.is_contiguous()):
        raise ValueError(f"{fn}: caches must be contiguous [num_blocks, block_size, HK, {HEAD_DIM}] of one shape")
    return shape[0], shape[1], shape[2]


def _new_rows(fn: str, key: torch.Tensor, value: torch.Tensor, hk: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Key and value rows [N, hk, 128] bf16 with contiguous heads, token rows apart from each other."""
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise TypeError(f"{fn}: key and value must be bf16, got {key.dtype} and {value.dtype}")
    if key.dim() != 3 or key.shape[1:] != (hk, HEAD_DIM) or value.shape != key.shape:
        raise ValueError(f"{fn}: key and value must be [N, {hk}, {HEAD_DIM}], got {tuple(key.shape)} and {tuple(value.shape)}")
    for t in (key, value):
        if t.stride(2) != 1 or (t.stride(1) != HEAD_DIM and hk > 1):
            raise ValueError(f"{fn}: key and value heads must be contiguous, got strides {t.stride()}")
    return tuple(t.contiguous() if t.shape[0] > 1 and t.stride(0) < hk * HEAD_DIM else t for t in (key, value))


def _scale(fn: str, softmax_scale: float) -> float:
    if not softmax_scale > 0:
        raise ValueError(f"{fn}: softmax_scale must be positive, got {softmax_scale}")
    return float(softmax_scale)


def decode_attention_weights(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, context_lens: torch.Tensor,
                             block_tables: torch.Tensor, softmax_scale: float, key_weights: torch.Tensor,
                             weight_rows: torch.Tensor | None = None, out: torch.Tensor | None = None,
                             key: torch.Tensor | None = None, value: torch.Tensor | None = None,
                             slot_mapping: torch.Tensor | None = None, plan=None) -> torch.Tensor:
    """``ops.decode_attention`` (one query per sequence over its first context_lens[b] cached tokens, with key / value /
    slot_mapping the step's rows stored in the same call), adding to ``key_weights`` what every key received: for token j
    and kv head g the sum of g's query heads' probabilities, on top of the weight for j < context_lens[b] - 1, in its place
    for the newest. Returns o [B, H, 128] bf16, zeros where context_lens[b] is 0 (whose row is left alone).

    The call takes scratch for the scores of every token that the tables reach, 4 H bytes a token. ``plan``: as
    decode_attention's; planned calls share the device's decode workspace and must not overlap other calls on it."""
    fn = "decode_attention_weights"
    if q.dim() != 3 or q.dtype != torch.bfloat16:
        raise TypeError(f"{fn}: q must be bf16 [B, H, {HEAD_DIM}], got {q.dtype} {tuple(q.shape)}")
    fp4 = is_fp4_cache(k_cache) and is_fp4_cache(v_cache)
    blocks, bs, hk = _cache_shape(k_cache, v_cache) if fp4 else _caches(fn, k_cache, v_cache)
    B, H, D = q.shape
    if hk not in (1, 2) or H == 0 or H % hk or H > MAX_DECODE_HEADS:
        raise ValueError(f"decode supports H <= {MAX_DECODE_HEADS} query heads over 1 or 2 KV heads, got {H}/{hk}")
    if context_lens.numel() != B or block_tables.dim() != 2 or block_tables.shape[0] < B:
        raise ValueError("context_lens must be [B] and block_tables [B, max_blocks]")
    scale = _scale(fn, softmax_scale)
    dev = _check_cuda(q, k_cache, v_cache, context_lens, block_tables)
    bt, bt_stride = _table(block_tables)
    mb = bt.shape[1]
    n_rows, width, rows = _weights(fn, key_weights, weight_rows, B, hk, mb * bs, q.get_device())
    q, q_stride, out = _query(fn, q, out, dev, True)
    ride = (None, None, 0, 0, None)
    if key is not None:
        if value is None or slot_mapping is None:
            raise ValueError(f"{fn}: key, value and slot_mapping go together")
        _check_cuda(q, key, value, slot_mapping)
        key, value = _new_rows(fn, key, value, hk)
        if key.shape[0] != B or slot_mapping.numel() != B:
            raise ValueError(f"{fn}: key, value and slot_mapping must hold {B} rows")
        slots, ks, vs = _ids(slot_mapping, "slot_mapping"), _row_stride(key), _row_stride(value)
        # (rows that 16-byte loads cannot take are stored by a call of their own)
        if (key.data_ptr() | value.data_ptr()) % 16 == 0 and (ks | vs) % 8 == 0:
            ride = (key.data_ptr(), value.data_ptr(), ks, vs, slots.data_ptr())
    elif value is not None or slot_mapping is not None:
        raise ValueError(f"{fn}: key, value and slot_mapping go together")
    if B == 0:
        return out
    lens = _as_i32(_flat(context_lens), "context_lens")
    lib = _lib.load()
    with _on(dev):
        if key is not None and ride[0] is None:
            (store_kvcache_fp4 if fp4 else store_kvcache)(key, value, k_cache, v_cache, slots)
        need = lib.vox_decode_scores_bytes(B, mb, bs, H)
        mode, recorded = _lib.PLAN_NONE, None
        if plan is None:  # all scratch in one piece: the call's own
            ws_bytes = lib.vox_decode_workspace_bytes(B)
            scratch = torch.empty((ws_bytes + need,), dtype=torch.uint8, device=dev)
            ws = scratch.data_ptr()
            scores = ws + ws_bytes
        else:
            scratch = torch.empty((need,), dtype=torch.uint8, device=dev)
            scores = scratch.data_ptr()
            kept, mode, recorded = _workspace(lib, dev, B, plan, "decode_weights", fp4, ride[0] is not None, B, mb,
                                              bt_stride, H, hk, bs)
            ws, ws_bytes = kept.data_ptr(), kept.numel()
        call = lib.vox_decode_attn_weights_fp4 if fp4 else lib.vox_decode_attn_weights
        _lib.check(call(
            q.data_ptr(), q_stride, *ride, k_cache.data_ptr(), v_cache.data_ptr(), blocks, bs, bt.data_ptr(), bt_stride, mb,
            lens.data_ptr(), B, H, hk, D, scale, key_weights.data_ptr(), None if rows is None else rows.data_ptr(), n_rows,
            width, scores, need, mode, ws, ws_bytes, out.data_ptr(), _lib.stream_handle(dev)), fn)
    if recorded is not None:
        _plan_recorded(dev, recorded)
    return out


def varlen_attention_weights(q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, key_weights: torch.Tensor,
                             weight_rows: torch.Tensor | None = None, *, cu_seqlens_q: torch.Tensor,
                             cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float,
                             block_table: torch.Tensor | None = None, k_cache: torch.Tensor | None = None,
                             v_cache: torch.Tensor | None = None, out: torch.Tensor | None = None, plan=None,
                             cu_seqlens_new: torch.Tensor | None = None) -> torch.Tensor:
    """``ops.varlen_attention`` (causal: sequence b's queries q [T, H, 128] are the last of its keys, from packed rows k / v
    [Tk, HK, 128] or, with block_table, from the caches), adding to ``key_weights`` what every key received: for token j and
    kv head g the sum of the probabilities of b's queries at g's query heads, in place of the weight for the step's own
    tokens, the last cu_seqlens_q[b + 1] - cu_seqlens_q[b], on top of it for the earlier ones. Returns o [T, H, 128] bf16,
    zeros for a query that sees no key. A sequence without queries keeps its weights.

    ``cu_seqlens_new`` (int [B + 1], as cu_seqlens_k): the step's own tokens, where there are fewer queries than those (a layer
    that takes the last row of each sequence): the last cu_seqlens_new[b + 1] - cu_seqlens_new[b] of sequence b's keys start with
    what the queries give them, with 0 where it has none.

    No sequence has more than max_seqlen_q queries or max_seqlen_k keys (further ones are left out). H / HK divides 128, and
    cache blocks are a multiple of 64 tokens. One-query sequences run on the decode kernels where a call is mostly those, as
    varlen_attention's do; ``plan``: as decode_attention_weights's, for these. A key that is not finite reaches the queries that
    see it alone; a value that is not reaches, as in varlen_attention, outputs of earlier queries of its tile too (never
    weights)."""
    fn = "varlen_attention_weights"
    if q.dim() != 3 or q.dtype != torch.bfloat16:
        raise TypeError(f"{fn}: q must be bf16 [T, H, {HEAD_DIM}], got {q.dtype} {tuple(q.shape)}")
    T, H, D = q.shape
    B = cu_seqlens_q.numel() - 1
    if cu_seqlens_k.numel() != B + 1:
        raise ValueError("cu_seqlens_k must have as many entries as cu_seqlens_q")
    scale = _scale(fn, softmax_scale)
    dev = _check_cuda(q, cu_seqlens_q, cu_seqlens_k)
    if block_table is not None:
        if k_cache is None or v_cache is None:
            raise ValueError(f"{fn}: block_table given without caches")
        fp4 = is_fp4_cache(k_cache) and is_fp4_cache(v_cache)
        blocks, bs, hk = _cache_shape(k_cache, v_cache) if fp4 else _caches(fn, k_cache, v_cache)
        if bs % 64:
            raise ValueError(f"{fn}: cache blocks must be a multiple of 64 tokens, got {bs}")
        if block_table.dim() != 2 or block_table.shape[0] < B:
            raise ValueError("block_table must be [B, max_blocks]")
        _check_cuda(q, k_cache, v_cache, block_table)
        bt, bt_stride = _table(block_table)
        reach = min(int(max_seqlen_k), bt.shape[1] * bs)
        keys = (k_cache.data_ptr(), v_cache.data_ptr(), blocks, bs, bt.data_ptr(), bt_stride, bt.shape[1])
        if not fp4:
            keys = (None, None, 0, 0, *keys)
    else:
        if k is None or v is None:
            raise ValueError(f"{fn}: packed keys and values required without a block table")
        _check_cuda(q, k, v)
        hk = k.shape[1] if k.dim() == 3 else 0
        k, v = _new_rows(fn, k, v, hk)
        reach = int(max_seqlen_k)
        fp4 = False
        keys = (k.data_ptr(), v.data_ptr(), _row_stride(k), _row_stride(v), None, None, 0, 0, None, 0, 0)
    if hk == 0 or H == 0 or H % hk:
        raise ValueError(f"num_heads {H} is not a multiple of num_kv_heads {hk}")
    n_rows, width, rows = _weights(fn, key_weights, weight_rows, max(B, 0), hk, reach, q.get_device())
    q, q_stride, out = _query(fn, q, out, dev, False)
    cu_q, cu_k = _as_i32(cu_seqlens_q, "cu_seqlens_q"), _as_i32(cu_seqlens_k, "cu_seqlens_k")
    lib = _lib.load()
    if cu_seqlens_new is not None:
        if cu_seqlens_new.numel() != B + 1:
            raise ValueError("cu_seqlens_new must have as many entries as cu_seqlens_q")
        _check_cuda(q, cu_seqlens_new)
        cu_new = _as_i32(_flat(cu_seqlens_new), "cu_seqlens_new")
        if B > 0 and reach > 0:
            with _on(dev):
                _lib.check(lib.vox_clear_key_weights(
                    key_weights.data_ptr(), None if rows is None else rows.data_ptr(), n_rows, width, hk, cu_new.data_ptr(),
                    cu_k.data_ptr(), B, 2 ** 31 - 1 if block_table is None else bt.shape[1] * bs, reach,
                    _lib.stream_handle(dev)), fn)
    max_seqlen_q = min(int(max_seqlen_q), T)
    if T == 0 or B <= 0 or max_seqlen_q <= 0:
        return out
    with _on(dev):
        need = lib.vox_prefill_weights_bytes(T, B, max_seqlen_q, reach, H, hk)
        scores_at = (need + 255) // 256 * 256
        ws, scores_bytes, mode, recorded = None, 0, _lib.PLAN_NONE, None
        if block_table is not None and (max_seqlen_q == 1 or 4 * T <= B * max_seqlen_q) \
                and _takes_decode_rows(H, hk, bs, bt.shape[1], out, _row_stride(out)):
            ws, mode, recorded = _workspace(lib, dev, B, plan, "varlen_weights", fp4, B, bt.shape[1], bt_stride, H, hk, bs)
            scores_bytes = lib.vox_decode_scores_bytes(B, bt.shape[1], bs, H)
        scratch = torch.empty((scores_at + scores_bytes,), dtype=torch.uint8, device=dev)
        at = scratch.data_ptr()
        call = lib.vox_prefill_attn_weights_fp4 if fp4 else lib.vox_prefill_attn_weights
        _lib.check(call(
            q.data_ptr(), q_stride, *keys, cu_q.data_ptr(), cu_k.data_ptr(), B, max_seqlen_q, reach, T, H, hk, D,
            scale, key_weights.data_ptr(), None if rows is None else rows.data_ptr(), n_rows, width, at, need,
            at + scores_at if scores_bytes else None, scores_bytes, mode, None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel(), out.data_ptr(), _row_stride(out), _lib.stream_handle(dev)), fn)
    _plan_recorded(dev, recorded)
    return out
