"""The operators of a KV cache held in 4 bits and of a paged cache's blocks, as measurable cases.

A 4-bit cache holds each key and value row in the MXFP4 format: 32 channels of one token and kv head share a power of
two (one e8m0 byte), and every value is one of the sixteen of e2m1 times it. A plane is uint8 [blocks, block_size, HK,
68]; inside a block's bytes the codes [block_size][HK][64] come first, then the scales [block_size][HK][4].

Kinds: ``store`` (rows quantised into their slots, and read back), ``decode`` (one query per sequence, alone or with the
step's own rows stored in the same call), ``varlen`` (new tokens over cached prefixes, with or without decode rows in
the same step), ``fork`` (sequences that share a parent's blocks and copy its last one), ``compact`` (live blocks moved
to the front of the pool). Blocks of 256 tokens, head_dim 128, 16 query heads over 2 kv heads, or 8 over 1 as each of
two tensor-parallel ranks has them."""

from __future__ import annotations

import random

import torch

own = False

D, BS = 128, 256
SCALE = D ** -0.5
GROUP = 32  # channels that share a scale
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DEV = "cuda"


def listed():
    return [
        # the rows of one generated frame of a few streams, in a captured batch whose last rows are padding
        {"name": "store_step", "kind": "store", "rows": 8, "pad": 2, "heads": 16, "kv_heads": 2, "blocks": 64},
        # the prompts that are admitted together
        {"name": "store_prompts", "kind": "store", "rows": 2823, "pad": 0, "heads": 16, "kv_heads": 2, "blocks": 64},
        # a library of voice prompts brought into the cache
        {"name": "store_library", "kind": "store", "rows": 60001, "pad": 0, "heads": 16, "kv_heads": 2, "blocks": 512},
        # one speaker being served alone
        {"name": "decode_1", "kind": "decode", "batch": 1, "lo": 420, "hi": 420, "heads": 16, "kv_heads": 2,
         "store": False},
        # an ordinary load on one of two tensor-parallel ranks
        {"name": "decode_40", "kind": "decode", "batch": 40, "lo": 200, "hi": 1500, "heads": 8, "kv_heads": 1,
         "store": False},
        # peak concurrency: the step's rows stored and attended over in one call
        {"name": "decode_150", "kind": "decode", "batch": 150, "lo": 256, "hi": 2048, "heads": 16, "kv_heads": 2,
         "store": True},
        # book-length contexts of a few streams
        {"name": "decode_long", "kind": "decode", "batch": 24, "lo": 20000, "hi": 32768, "heads": 16, "kv_heads": 2,
         "store": False},
        # a burst of short texts after a cached voice prompt
        {"name": "prefix_burst", "kind": "varlen", "batch": 44, "lo": 33, "hi": 59, "prefix_lo": 50, "prefix_hi": 50,
         "decodes": 0, "ctx_lo": 0, "ctx_hi": 0, "heads": 16, "kv_heads": 2},
        # chapters continued after long cached contexts: compute-bound
        {"name": "prefix_long", "kind": "varlen", "batch": 6, "lo": 1000, "hi": 2000, "prefix_lo": 1500,
         "prefix_hi": 2500, "decodes": 0, "ctx_lo": 0, "ctx_hi": 0, "heads": 16, "kv_heads": 2},
        # prompts admitted while other streams decode, in one step
        {"name": "mixed", "kind": "varlen", "batch": 6, "lo": 300, "hi": 600, "prefix_lo": 0, "prefix_hi": 0,
         "decodes": 120, "ctx_lo": 128, "ctx_hi": 1800, "heads": 16, "kv_heads": 2},
        # several takes of the same texts, each going on from what has been said so far
        {"name": "fork_takes", "kind": "fork", "layers": 28, "blocks": 160, "batch": 24, "takes": 32, "lo": 60,
         "hi": 1500},
        # the pool after a peak: live blocks moved to its front, the rest of it given back
        {"name": "compact_pool", "kind": "compact", "layers": 12, "blocks": 384, "batch": 70, "lo": 60, "hi": 1024},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["store", "decode", "decode", "decode", "varlen", "varlen", "varlen", "fork", "compact"])
    heads, kv_heads = rng.choice([(16, 2), (16, 2), (8, 1)])
    if kind == "store":
        rows = log(1, 60000)
        return {"kind": kind, "rows": rows, "pad": rng.randint(0, rows // 4), "heads": heads, "kv_heads": kv_heads,
                "blocks": -(-rows // BS) + rng.randint(1, 64)}
    if kind == "decode":
        batch = log(1, 300)
        hi = min(32768, log(4, 600000 // batch))
        return {"kind": kind, "batch": batch, "lo": rng.randint(1, hi), "hi": hi, "heads": heads,
                "kv_heads": kv_heads, "store": rng.random() < 0.5}
    if kind == "varlen":
        hi = log(2, 2000)
        batch = log(1, max(1, min(64, 6000 // hi)))
        prefix = rng.choice([0, log(8, 2200)])
        decodes = rng.choice([0, log(1, 120)]) if hi <= 600 else 0
        ctx = log(16, 1800)
        return {"kind": kind, "batch": batch, "lo": rng.randint(max(2, hi // 4), hi), "hi": hi,
                "prefix_lo": prefix // 2, "prefix_hi": prefix, "decodes": decodes, "ctx_lo": max(1, ctx // 4),
                "ctx_hi": ctx, "heads": heads, "kv_heads": kv_heads}
    hi = log(20, 2000)
    batch = log(1, min(70, 160 * BS // (hi + BS)))
    layers = log(1, 28)
    most = batch * -(-hi // BS)
    if kind == "fork":
        return {"kind": kind, "layers": layers, "blocks": most + 40, "batch": batch, "takes": log(1, 36),
                "lo": rng.randint(1, hi), "hi": hi}
    return {"kind": kind, "layers": min(layers, 20), "blocks": most + log(8, 160), "batch": batch,
            "lo": rng.randint(1, hi), "hi": hi}


# ----------------------------------------------------------------------------------------------------------------------
# inputs


def _lens(what, n, lo, hi):
    """n lengths uniform in [lo, hi], the same for every seed of a case (the work depends on them)."""
    rng = random.Random("%s %d %d %d" % (what, n, lo, hi))
    return [rng.randint(lo, hi) for _ in range(n)]


def _sequences(case):
    """(new tokens, all tokens) of each sequence."""
    if case["kind"] == "varlen":
        new = _lens("new", case["batch"], case["lo"], case["hi"])
        ctx = _lens("ctx", case["decodes"], case["ctx_lo"], case["ctx_hi"])
        old = _lens("prefix", case["batch"], case["prefix_lo"], case["prefix_hi"])
        return [(n, n + p) for n, p in zip(new, old)] + [(1, n) for n in ctx]
    return [(1, n) for n in _lens("ctx", case["batch"], case["lo"], case["hi"])]


def _tables(lens, pool, seed):
    """Block tables (-1 padded) from a shuffled pool, and the pool's blocks that no table names."""
    need = [-(-n // BS) for n in lens]
    perm = list(range(pool))
    random.Random(seed).shuffle(perm)
    rows, at = [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (max(need) - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV), perm[at:]


def _pool(lens):
    need = sum(-(-n // BS) for n in lens)
    return need + max(4, need // 16)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _step_rows(case, n, seed):
    """A qkv projection's rows and q / k / v as views of them; keys and values differ in size by channel."""
    h, hk = case["heads"], case["kv_heads"]
    gen = _gen(seed)
    x = torch.randn(n, (h + 2 * hk) * D, generator=gen, device=DEV)
    x[:, h * D:] *= torch.exp(0.5 * torch.randn(2 * hk * D, generator=gen, device=DEV))
    x = x.to(torch.bfloat16)
    return (x[:, :h * D].view(n, h, D), x[:, h * D:(h + hk) * D].view(n, hk, D), x[:, (h + hk) * D:].view(n, hk, D))


def _plane(blocks, hk, seed):
    """A 4-bit plane holding rows whose channels differ in size."""
    gen = _gen(seed)
    size = torch.exp(0.5 * torch.randn(hk * D, generator=gen, device=DEV)).view(hk, D)
    cache = torch.empty(blocks, BS, hk, 68, dtype=torch.uint8, device=DEV)
    codes, scales = _parts(cache)
    for a in range(0, blocks, 256):
        n = min(256, blocks - a)
        x = (torch.randn(n, BS, hk, D, generator=gen, device=DEV) * size).to(torch.bfloat16)
        codes[a:a + n], scales[a:a + n] = _quantised(x)
    return cache


def _parts(cache):
    """The codes [blocks, block_size, HK, 64] and scales [blocks, block_size, HK, 4] of a plane, as views."""
    blocks, bs, hk, _ = cache.shape
    per = bs * hk * 68
    flat = cache.view(-1)
    return (flat.as_strided((blocks, bs, hk, 64), (per, hk * 64, 64, 1)),
            flat.as_strided((blocks, bs, hk, 4), (per, hk * 4, 4, 1), flat.storage_offset() + bs * hk * 64))


def _inputs(case, seed):
    kind = case["kind"]
    if kind == "store":
        n = case["rows"]
        _, k, v = _step_rows(case, n, 5 * seed)
        at = torch.arange(n, dtype=torch.int32, device=DEV)
        if n < 64:  # a step's rows are anywhere
            slots = torch.randperm(case["blocks"] * BS, generator=_gen(5 * seed + 1), device=DEV)[:n].to(torch.int32)
        else:  # prompts fill blocks
            perm = torch.randperm(case["blocks"], generator=_gen(5 * seed + 1), device=DEV).to(torch.int32)
            slots = perm[at // BS] * BS + at % BS
        slots[n - case["pad"]:] = -1
        hk = case["kv_heads"]
        planes = torch.zeros(2, case["blocks"], BS, hk, 68, dtype=torch.uint8, device=DEV)
        return {"k": k, "v": v, "slots": slots, "k_cache": planes[0], "v_cache": planes[1]}
    if kind in ("decode", "varlen"):
        seqs = _sequences(case)
        lens = [n for _, n in seqs]
        pool = _pool(lens)
        tables, _ = _tables(lens, pool, 5 * seed)
        hk = case["kv_heads"]
        q, k, v = _step_rows(case, sum(n for n, _ in seqs), 5 * seed + 1)
        x = {"q": q, "k_cache": _plane(pool, hk, 5 * seed + 2), "v_cache": _plane(pool, hk, 5 * seed + 3),
             "tables": tables, "lens": torch.tensor(lens, dtype=torch.int32, device=DEV)}
        if kind == "varlen":
            cu = torch.tensor([[0, 0], *seqs], dtype=torch.int32, device=DEV).cumsum(0).to(torch.int32)
            x.update(cu_q=cu[:, 0].contiguous(), cu_k=cu[:, 1].contiguous(), max_q=max(n for n, _ in seqs),
                     max_k=max(lens))
        elif case["store"]:
            last = x["lens"].long() - 1
            slots = tables.gather(1, (last // BS)[:, None])[:, 0] * BS + (last % BS).to(torch.int32)
            x.update(k=k, v=v, slots=slots.to(torch.int32))
        return x
    lens = _lens("ctx", case["batch"], case["lo"], case["hi"])
    tables, rest = _tables(lens, case["blocks"], 5 * seed)
    kv = torch.randn(case["layers"], 2, case["blocks"], BS, 2, D, generator=_gen(5 * seed + 1), device=DEV,
                     dtype=torch.bfloat16)
    x = {"kv": kv, "tables": tables, "lens": torch.tensor(lens, dtype=torch.int32, device=DEV)}
    if kind == "fork":
        who = _lens("parent", case["takes"], 0, case["batch"] - 1)
        x.update(parents=torch.tensor(who, dtype=torch.int32, device=DEV),
                 new=torch.tensor(rest[:case["takes"]], dtype=torch.int32, device=DEV))
    return x


def prepare(case, seed):
    return dict(_inputs(case, seed), kind=case["kind"])


# ----------------------------------------------------------------------------------------------------------------------
# one pass


def run(state):
    if own:
        return _own(state)
    return {"store": _store, "decode": _decode, "varlen": _varlen, "fork": _fork, "compact": _compact}[state["kind"]](state)


def _own(s):
    from voxcpm2_arabic_dialects_turbo_amd.kernels.kv_pages import compact_kv_blocks, fork_kv_blocks
    from voxcpm2_arabic_dialects_turbo_amd.ops_fp4 import (decode_attention_fp4, load_kvcache_fp4, store_kvcache_fp4,
                                                           varlen_attention_fp4)

    kind = s["kind"]
    if kind == "store":
        store_kvcache_fp4(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return load_kvcache_fp4(s["k_cache"], s["v_cache"], s["slots"])
    if kind == "decode":
        if "slots" not in s:
            return decode_attention_fp4(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["tables"], SCALE)
        o = decode_attention_fp4(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["tables"], SCALE, key=s["k"],
                                 value=s["v"], slot_mapping=s["slots"])
        return o, *load_kvcache_fp4(s["k_cache"], s["v_cache"], s["slots"])
    if kind == "varlen":
        return varlen_attention_fp4(s["q"], s["k_cache"], s["v_cache"], cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"],
                                    max_seqlen_q=s["max_q"], block_table=s["tables"], softmax_scale=SCALE)
    if kind == "fork":
        return *fork_kv_blocks(s["kv"], s["tables"], s["lens"], s["parents"], s["new"]), s["kv"]
    return *compact_kv_blocks(s["kv"], s["tables"], s["lens"]), s["kv"]


def _quantised(x):
    """x [..., HK, 128] as MXFP4: codes [..., HK, 64] and scales [..., HK, 4], both uint8."""
    g = x.float().unflatten(-1, (D // GROUP, GROUP))
    amax = g.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    # the least power of two that leaves the largest value at most 7, half a step over the grid's 6
    b = (e + (m > 0.875) + (127 - 3)).clamp(1, 254)
    a = torch.ldexp(g.abs(), (127 - b)[..., None])
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (g < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(amax.isfinite(), b, 255).to(torch.uint8)


def _values(codes, scales):
    """The values that codes [..., 64] and scales [..., 4] stand for, fp32 [..., 128]."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    return torch.ldexp(grid[code].unflatten(-1, (D // GROUP, GROUP)), scales.int()[..., None] - 127).flatten(-2)


def _stored(s):
    """Quantises the step's rows into their slots (none for -1)."""
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    for rows, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        codes, scales = _parts(cache)
        codes[at // BS, at % BS], scales[at // BS, at % BS] = _quantised(rows[keep])


def _rows(cache, slots):
    """The values at slots, fp32 [..., HK, 128]; zeros where a slot is -1."""
    codes, scales = _parts(cache)
    at = slots.clamp(min=0).long()
    return _values(codes[at // BS, at % BS], scales[at // BS, at % BS]) * (slots >= 0)[..., None, None]


def _store(s):
    _stored(s)
    return tuple(_rows(c, s["slots"]).to(torch.bfloat16) for c in (s["k_cache"], s["v_cache"]))


def _padded(s, n):
    """Keys and values of every sequence's first n positions, fp32 [B, HK, n, 128]."""
    pos = torch.arange(n, device=DEV)
    slots = s["tables"][:, pos // BS].long() * BS + pos % BS
    slots = torch.where(pos < s["lens"][:, None], slots, -1)
    return tuple(_rows(c, slots).transpose(1, 2) for c in (s["k_cache"], s["v_cache"]))


def _attended(q, k, v, mask):
    """softmax(q k^T SCALE) v over the keys that mask leaves: q [B, HK, n, 128], mask broadcast to [B, HK, n, keys]."""
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * SCALE
    x = torch.where(mask, x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top.isinf(), 0.0, top))
    return torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _decode(s):
    if "slots" in s:
        _stored(s)
    b, h, _ = s["q"].shape
    n = s["tables"].shape[1] * BS
    k, v = _padded(s, n)
    mask = (torch.arange(n, device=DEV) < s["lens"][:, None])[:, None, None]
    o = _attended(s["q"].float().reshape(b, k.shape[1], -1, D), k, v, mask).reshape(b, h, D).to(torch.bfloat16)
    if "slots" not in s:
        return o
    return o, *(_rows(c, s["slots"]).to(torch.bfloat16) for c in (s["k_cache"], s["v_cache"]))


def _varlen(s):
    k, v = _padded(s, s["max_k"])
    t, h, _ = s["q"].shape
    b, hk, g = k.shape[0], k.shape[1], h // k.shape[1]
    new = s["cu_q"].diff()
    i = torch.arange(s["max_q"], device=DEV)
    row = (s["cu_q"][:-1, None] + i).clamp(max=t - 1)  # the padded place (sequence, i) of each query row
    q = s["q"].float()[row].view(b, -1, hk, g, D).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, D)
    seen = s["lens"][:, None] - new[:, None] + i + 1  # the keys that query i sees
    mask = (torch.arange(s["max_k"], device=DEV) < seen[..., None]).repeat(1, g, 1)[:, None]
    o = _attended(q, k, v, mask).view(b, hk, g, -1, D).permute(0, 3, 1, 2, 4).reshape(b, -1, h, D)
    return o[i < new[:, None]].to(torch.bfloat16)


def _fork(s):
    tables, lens = s["tables"][s["parents"].long()], s["lens"][s["parents"].long()]
    col = torch.arange(tables.shape[1], device=DEV)
    full, tail = lens // BS, lens % BS
    part = (col == full[:, None]) & (tail > 0)[:, None]
    child = torch.where(col < full[:, None], tables, torch.where(part, s["new"][:, None], -1)).to(torch.int32)
    src = tables.gather(1, full.clamp(max=tables.shape[1] - 1).long()[:, None])[:, 0]
    j = torch.arange(BS, device=DEV)
    i, j = (j < tail[:, None]).nonzero(as_tuple=True)
    s["kv"][:, :, s["new"][i].long(), j] = s["kv"][:, :, src[i].long(), j]
    return child, lens, s["kv"]


def _compact(s):
    tables, n = s["tables"], s["kv"].shape[2]
    used = torch.arange(tables.shape[1], device=DEV) < (-(-s["lens"] // BS))[:, None]
    live = torch.zeros(n, dtype=torch.bool, device=DEV)
    live[tables[used].long()] = True
    count = live.sum()
    at = torch.arange(n, device=DEV)
    src = (live & (at >= count)).nonzero()[:, 0]
    dst = (~live & (at < count)).nonzero()[:, 0]
    remap = torch.where(live, at, -1)
    remap[src] = dst
    s["kv"][:, :, dst] = s["kv"][:, :, src]
    out = torch.where(used, remap[tables.clamp(min=0).long()], -1).to(torch.int32)
    return out, remap.to(torch.int32), count.to(torch.int32).view(1), s["kv"]


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    kind = case["kind"]
    if kind == "store":
        hk, n = case["kv_heads"], case["rows"] - case["pad"]
        # the rows read, their codes and scales written; then read, and the values written
        return {"bytes": n * 2 * hk * (2 * D + 68) * 2 + case["rows"] * 4, "flops": n * 2 * hk * D}
    if kind in ("decode", "varlen"):
        h, hk, seqs = case["heads"], case["kv_heads"], _sequences(case)
        new, keys = sum(n for n, _ in seqs), sum(n for _, n in seqs)
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in seqs)
        rows = case["batch"] * 2 * hk * (4 * D + 2 * 68) if case.get("store") else 0
        return {"bytes": new * h * D * 4 + keys * 2 * hk * 68 + rows, "flops": 4 * D * h * pairs}
    lens = _lens("ctx", case["batch"], case["lo"], case["hi"])
    slot = case["layers"] * 2 * 2 * D * 2  # bytes of a token in every plane
    if kind == "fork":
        who = _lens("parent", case["takes"], 0, case["batch"] - 1)
        return {"bytes": 2 * slot * sum(lens[i] % BS for i in who) + 1, "flops": 0}
    live = sum(-(-n // BS) for n in lens)
    # a shuffled pool leaves live (1 - live / blocks) of its live blocks behind the first `live` ones, give or take
    return {"bytes": 2 * slot * BS * live * (case["blocks"] - live) / case["blocks"] + 1, "flops": 0}


# ----------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits


def _exact_quantised(x):
    """The values that x [n, HK, 128] is held as: the nearest of the grid times its group's power of two, ties to the
    even code."""
    x = x.double().view(x.shape[0], -1, GROUP)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp_min(1e-300)))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e)) - 2
    e = torch.where(top > 7 * torch.exp2(e), e + 1, e).clamp(-126, 127)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    off = ((x.abs() / torch.exp2(e)).clamp(max=6.0)[..., None] - grid).abs()
    odd = torch.arange(8, device=x.device) % 2
    code = torch.where(off == off.amin(-1, keepdim=True), 2 - odd, 0).argmax(-1)
    return (grid[code] * x.sign() * torch.exp2(e)).view(x.shape[0], -1, D)


def _exact_rows(cache, table, n):
    """The first n tokens of one sequence in 64 bits [n, HK, 128], byte by byte of its blocks."""
    hk = cache.shape[2]
    block = cache.reshape(cache.shape[0], -1)[table[:-(-n // BS)].long()]
    codes, scales = block[:, :BS * hk * 64].reshape(-1, hk, 64), block[:, BS * hk * 64:].reshape(-1, hk, 4)
    out = torch.empty(n, hk, D, dtype=torch.float64, device=cache.device)
    for half in (0, 1):
        c = (codes[:n] >> (4 * half)) & 15
        mag = (c & 7).double()  # 0 1 2 3 | 4 5 | 6 7: steps of a half, then of one, then of two
        mag = torch.where(mag < 4, mag / 2, torch.where(mag < 6, mag - 2, 2 * mag - 8))
        out[..., half::2] = torch.where(c >= 8, -mag, mag)
    return out * torch.exp2(scales[:n].double() - 127).repeat_interleave(GROUP, -1)


def _exact_attention(q, k, v, group):
    """Queries [n, H, 128], the last n positions of keys [m, HK, 128]."""
    n, m = q.shape[0], k.shape[0]
    k, v = k.repeat_interleave(group, 1).permute(1, 2, 0).contiguous(), v.repeat_interleave(group, 1).transpose(0, 1).contiguous()
    x = torch.matmul(q.double().transpose(0, 1).contiguous(), k) * SCALE
    late = torch.arange(m, device=q.device)[None] > torch.arange(n, device=q.device)[:, None] + (m - n)
    return torch.matmul(torch.softmax(x.masked_fill(late, float("-inf")), -1), v).transpose(0, 1)


def exact(case, seed):
    x, kind = _inputs(case, seed), case["kind"]
    if kind == "store":
        live = (x["slots"] >= 0)[:, None, None]
        return tuple(_exact_quantised(x[r]) * live for r in ("k", "v"))
    if kind in ("decode", "varlen"):
        out, at, stored = [], 0, ()
        if "slots" in x:
            stored = _exact_quantised(x["k"]), _exact_quantised(x["v"])
        for b, (new, n) in enumerate(_sequences(case)):
            k, v = (_exact_rows(x[c], x["tables"][b], n) for c in ("k_cache", "v_cache"))
            if stored:
                k[n - 1], v[n - 1] = stored[0][b], stored[1][b]
            for a in range(0, new, 256):  # queries in slices, for their scores' memory
                e = min(new, a + 256)
                m = n - new + e
                out.append(_exact_attention(x["q"][at + a:at + e], k[:m], v[:m], case["heads"] // case["kv_heads"]))
            at += new
        o = torch.cat(out)
        return (o, *stored) if stored else o
    kv, tables, lens = x["kv"], x["tables"].tolist(), x["lens"].tolist()
    if kind == "fork":
        for p, to in zip(x["parents"].tolist(), x["new"].tolist()):
            if tail := lens[p] % BS:
                kv[:, :, to, :tail] = kv[:, :, tables[p][lens[p] // BS], :tail].clone()
        return None, None, kv
    live = sorted(b for row, n in zip(tables, lens) for b in row[:-(-n // BS)])
    holes = sorted(set(range(len(live))) - set(live))
    for src, dst in zip([b for b in live if b >= len(live)], holes):
        kv[:, :, dst] = kv[:, :, src]
    return None, None, None, kv
