"""The operators of a KV cache that drops what is attended to least, as measurable cases.

Beside a paged cache, ``key_weights`` (fp32 [rows, kv_heads, width]; one row per sequence, in any order: ``weight_rows``)
holds for every cached token and kv head the attention weight that it has received so far: the sum of its probabilities
over the queries of the kv head's group. Attention adds each step's: a token of the step itself starts with what it gets
there, the cached ones get theirs on top. Eviction keeps the ``budget`` tokens of a sequence that matter: its first
``sinks`` and last ``recent`` ones and, per layer and kv head, those with the largest weight among the others (of equal
ones the earliest), moved in their order to the front of the sequence's own blocks, their weights with them.

Kinds: ``decode`` (one query per sequence, alone or with the step's rows stored in the same call), ``chunk`` (new tokens
over packed rows or over a paged cache, with or without decode rows in the same step), ``evict`` (every layer and kv head
of bf16 or 4-bit caches). Blocks of 256 tokens, head_dim 128; 16 query heads over 2 kv heads, 8 over 1 as each of two
tensor-parallel ranks has them, or 4 over 2."""

from __future__ import annotations

import random

import torch

own = False

D, BS = 128, 256
SCALE = D ** -0.5
DEV = "cuda"


def listed():
    return [
        # one speaker being served alone
        {"name": "decode_1", "kind": "decode", "batch": 1, "lo": 420, "hi": 420, "heads": 16, "kv_heads": 2,
         "store": False},
        # an ordinary load on one of two tensor-parallel ranks
        {"name": "decode_40", "kind": "decode", "batch": 40, "lo": 200, "hi": 1500, "heads": 8, "kv_heads": 1,
         "store": False},
        # peak concurrency: the step's rows stored and attended over in one call
        {"name": "decode_150", "kind": "decode", "batch": 150, "lo": 256, "hi": 2048, "heads": 16, "kv_heads": 2,
         "store": True},
        # book-length contexts of a few streams, the caches that eviction is for
        {"name": "decode_long", "kind": "decode", "batch": 24, "lo": 20000, "hi": 32768, "heads": 16, "kv_heads": 2,
         "store": False},
        # a burst of short texts after a cached voice prompt
        {"name": "chunk_burst", "kind": "chunk", "packed": False, "batch": 44, "lo": 33, "hi": 59, "prefix_lo": 50,
         "prefix_hi": 50, "decodes": 0, "ctx_lo": 0, "ctx_hi": 0, "heads": 16, "kv_heads": 2},
        # prompts admitted together: their own rows, nothing cached yet
        {"name": "chunk_prompts", "kind": "chunk", "packed": True, "batch": 5, "lo": 237, "hi": 900, "prefix_lo": 0,
         "prefix_hi": 0, "decodes": 0, "ctx_lo": 0, "ctx_hi": 0, "heads": 16, "kv_heads": 2},
        # chapters continued after long cached contexts: compute-bound
        {"name": "chunk_long", "kind": "chunk", "packed": False, "batch": 6, "lo": 1000, "hi": 2000, "prefix_lo": 1500,
         "prefix_hi": 2500, "decodes": 0, "ctx_lo": 0, "ctx_hi": 0, "heads": 16, "kv_heads": 2},
        # prompts admitted while other streams decode, in one step
        {"name": "chunk_mixed", "kind": "chunk", "packed": False, "batch": 6, "lo": 300, "hi": 600, "prefix_lo": 0,
         "prefix_hi": 0, "decodes": 120, "ctx_lo": 128, "ctx_hi": 1800, "heads": 16, "kv_heads": 2},
        # one stream that has filled its budget and a block beyond it
        {"name": "evict_1", "kind": "evict", "layers": 28, "batch": 1, "lo": 1280, "hi": 1280, "budget": 1024,
         "sinks": 4, "recent": 256, "heads": 16, "kv_heads": 2, "four_bit": False},
        # many streams brought down together; some are still within the budget
        {"name": "evict_48", "kind": "evict", "layers": 28, "batch": 48, "lo": 600, "hi": 2048, "budget": 768,
         "sinks": 4, "recent": 128, "heads": 16, "kv_heads": 2, "four_bit": False},
        # book-length contexts brought down to a quarter, once they have been read
        {"name": "evict_long", "kind": "evict", "layers": 12, "batch": 8, "lo": 20000, "hi": 32768, "budget": 8000,
         "sinks": 16, "recent": 1024, "heads": 16, "kv_heads": 2, "four_bit": False},
        # caches held in 4 bits, on one of two tensor-parallel ranks
        {"name": "evict_4bit", "kind": "evict", "layers": 28, "batch": 30, "lo": 700, "hi": 1500, "budget": 500,
         "sinks": 1, "recent": 63, "heads": 8, "kv_heads": 1, "four_bit": True},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["decode", "chunk", "evict"])
    heads, kv_heads = rng.choice([(16, 2), (16, 2), (8, 1), (4, 2)])
    if kind == "decode":
        batch = log(1, 300)
        hi = min(32768, log(4, 600000 // batch))
        return {"kind": kind, "batch": batch, "lo": rng.randint(1, hi), "hi": hi, "heads": heads,
                "kv_heads": kv_heads, "store": rng.random() < 0.5}
    if kind == "chunk":
        hi = log(2, 2000)
        batch = log(1, max(1, min(64, 6000 // hi)))
        packed = rng.random() < 0.4
        prefix = 0 if packed else rng.choice([0, log(8, 2200)])
        decodes = rng.choice([0, log(1, 120)]) if hi <= 600 and not packed else 0
        ctx = log(16, 1800)
        return {"kind": kind, "packed": packed, "batch": batch, "lo": rng.randint(max(2, hi // 4), hi), "hi": hi,
                "prefix_lo": prefix // 2, "prefix_hi": prefix, "decodes": decodes, "ctx_lo": max(1, ctx // 4),
                "ctx_hi": ctx, "heads": heads, "kv_heads": kv_heads}
    hi = log(20, 32768)
    layers = log(1, 28)
    batch = log(1, max(1, min(64, 2000000 // (layers * hi))))
    budget = log(max(2, hi // 16), hi)
    sinks = rng.randint(0, min(16, budget // 4))
    return {"kind": kind, "layers": layers, "batch": batch, "lo": rng.randint(max(1, hi // 4), hi), "hi": hi,
            "budget": budget, "sinks": sinks, "recent": rng.randint(0, (budget - sinks) // 2), "heads": heads,
            "kv_heads": kv_heads, "four_bit": rng.random() < 0.3}


# ----------------------------------------------------------------------------------------------------------------------
# inputs


def _lens(what, n, lo, hi):
    """n lengths uniform in [lo, hi], the same for every seed of a case (the work depends on them)."""
    rng = random.Random("%s %d %d %d" % (what, n, lo, hi))
    return [rng.randint(lo, hi) for _ in range(n)]


def _sequences(case):
    """(new tokens, all tokens) of each sequence."""
    if case["kind"] == "chunk":
        new = _lens("new", case["batch"], case["lo"], case["hi"])
        ctx = _lens("ctx", case["decodes"], case["ctx_lo"], case["ctx_hi"])
        old = _lens("prefix", case["batch"], case["prefix_lo"], case["prefix_hi"])
        return [(n, n + p) for n, p in zip(new, old)] + [(1, n) for n in ctx]
    return [(1, n) for n in _lens("ctx", case["batch"], case["lo"], case["hi"])]


def _tables(lens, pool, seed):
    """Block tables (-1 padded) from a shuffled pool."""
    need = [-(-n // BS) for n in lens]
    perm = list(range(pool))
    random.Random(seed).shuffle(perm)
    rows, at = [], 0
    for n in need:
        rows.append(perm[at:at + n] + [-1] * (max(need) - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


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


def _received(shape, seed):
    """Weights as they add up: a few large ones, most small; whole multiples of 1 / 4096, so that some are equal."""
    return torch.floor(torch.rand(shape, generator=_gen(seed), device=DEV) ** 4 * 16384) / 4096


def _inputs(case, seed):
    hk, seqs = case["kv_heads"], _sequences(case)
    lens = [n for _, n in seqs]
    pool = _pool(lens)
    tables = _tables(lens, pool, 5 * seed)
    width = tables.shape[1] * BS
    rows = len(lens) + 3  # a row per stream that may be served, those of this call among them
    x = {"lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "tables": tables,
         "rows": torch.randperm(rows, generator=_gen(5 * seed + 1), device=DEV)[:len(lens)].to(torch.int32)}
    if case["kind"] == "evict":
        shape = (case["layers"], 2, pool, BS, hk)
        if case["four_bit"]:
            kv = torch.randint(0, 256, (*shape, 68), generator=_gen(5 * seed + 2), device=DEV, dtype=torch.uint8)
        else:
            kv = torch.randn(*shape, D, generator=_gen(5 * seed + 2), device=DEV, dtype=torch.bfloat16)
        x.update(kv=kv, weights=_received((case["layers"], rows, hk, width), 5 * seed + 3), budget=case["budget"],
                 sinks=case["sinks"], recent=case["recent"])
        return x
    q, k, v = _step_rows(case, sum(n for n, _ in seqs), 5 * seed + 2)
    x.update(q=q, weights=_received((rows, hk, width), 5 * seed + 3))
    if case["kind"] == "chunk":
        cu = torch.tensor([[0, 0], *seqs], dtype=torch.int32, device=DEV).cumsum(0).to(torch.int32)
        x.update(cu_q=cu[:, 0].contiguous(), cu_k=cu[:, 1].contiguous(), max_q=max(n for n, _ in seqs), max_k=max(lens))
        if case["packed"]:
            x.update(k=k, v=v)
            return x
    gen = _gen(5 * seed + 4)
    for name in ("k_cache", "v_cache"):
        size = torch.exp(0.5 * torch.randn(hk, D, generator=gen, device=DEV)).to(torch.bfloat16)
        x[name] = torch.randn(pool, BS, hk, D, generator=gen, device=DEV, dtype=torch.bfloat16).mul_(size)
    if case["kind"] == "decode" and case["store"]:
        last = x["lens"].long() - 1
        slots = tables.gather(1, (last // BS)[:, None])[:, 0] * BS + (last % BS).to(torch.int32)
        x.update(k=k, v=v, slots=slots.to(torch.int32))
    return x


def prepare(case, seed):
    return dict(_inputs(case, seed), kind=case["kind"])


# ----------------------------------------------------------------------------------------------------------------------
# one pass


def run(state):
    if own:
        return _own(state)
    return {"decode": _decode, "chunk": _chunk, "evict": _evict}[state["kind"]](state)


def _own(s):
    from voxcpm2_arabic_dialects_turbo_amd.kernels.kv_evict import evict_kv_tokens
    from voxcpm2_arabic_dialects_turbo_amd.ops_weights import decode_attention_weights, varlen_attention_weights

    if s["kind"] == "decode":
        if "slots" not in s:
            o = decode_attention_weights(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["tables"], SCALE, s["weights"],
                                         weight_rows=s["rows"])
            return o, s["weights"]
        o = decode_attention_weights(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["tables"], SCALE, s["weights"],
                                     weight_rows=s["rows"], key=s["k"], value=s["v"], slot_mapping=s["slots"])
        return o, s["weights"], s["k_cache"], s["v_cache"]
    if s["kind"] == "chunk":
        o = varlen_attention_weights(s["q"], s.get("k"), s.get("v"), s["weights"], weight_rows=s["rows"],
                                     cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"], max_seqlen_q=s["max_q"],
                                     max_seqlen_k=s["max_k"], softmax_scale=SCALE,
                                     block_table=None if "k" in s else s["tables"], k_cache=s.get("k_cache"),
                                     v_cache=s.get("v_cache"))
        return o, s["weights"]
    tables, lens = evict_kv_tokens(s["kv"], s["weights"], s["tables"], s["lens"], s["budget"], recent=s["recent"],
                                   sinks=s["sinks"], weight_rows=s["rows"])
    return tables, lens, s["kv"], s["weights"]


def _cached(s, n):
    """Keys and values of every sequence's first n positions, fp32 [B, HK, n, 128], zeros past its context."""
    pos = torch.arange(n, device=DEV)
    live = pos < s["lens"][:, None]
    blk = torch.where(live, s["tables"][:, pos // BS], 0).long()
    return tuple((c[blk, pos % BS].float() * live[..., None, None]).transpose(1, 2) for c in (s["k_cache"], s["v_cache"]))


def _packed(s, n):
    """The same of packed rows."""
    pos = torch.arange(n, device=DEV)
    live = pos < s["lens"][:, None]
    row = torch.where(live, s["cu_k"][:-1, None] + pos, 0).long()
    return tuple((x[row].float() * live[..., None, None]).transpose(1, 2) for x in (s["k"], s["v"]))


def _attended(q, k, v, mask):
    """softmax(q k^T SCALE) v over the keys that mask leaves, and the probabilities: q [B, HK, n, 128], mask broadcast to
    [B, HK, n, keys]."""
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * SCALE
    x = torch.where(mask, x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top.isinf(), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return torch.matmul(p, v.contiguous()), p


def _add(s, got, new):
    """Adds got [B, HK, n] to the rows' weights; the last `new` ([B]) tokens of a sequence start with theirs."""
    n = got.shape[2]
    pos = torch.arange(n, device=DEV)
    lens, rows = s["lens"][:, None, None], s["rows"].long()
    old = s["weights"][rows, :, :n]
    out = torch.where(pos >= lens - new[:, None, None], got, old + got)
    s["weights"][rows, :, :n] = torch.where(pos < lens, out, old)


def _decode(s):
    if "slots" in s:
        at = s["slots"].long()
        s["k_cache"][at // BS, at % BS] = s["k"]
        s["v_cache"][at // BS, at % BS] = s["v"]
    b, h, _ = s["q"].shape
    n = s["tables"].shape[1] * BS
    k, v = _cached(s, n)
    mask = (torch.arange(n, device=DEV) < s["lens"][:, None])[:, None, None]
    o, p = _attended(s["q"].float().reshape(b, k.shape[1], -1, D), k, v, mask)
    _add(s, p.sum(2), torch.ones_like(s["lens"]))
    o = o.reshape(b, h, D).to(torch.bfloat16)
    return (o, s["weights"], s["k_cache"], s["v_cache"]) if "slots" in s else (o, s["weights"])


def _chunk(s):
    k, v = _packed(s, s["max_k"]) if "k" in s else _cached(s, s["max_k"])
    t, h, _ = s["q"].shape
    b, hk, g = k.shape[0], k.shape[1], h // k.shape[1]
    new = s["cu_q"].diff()
    i = torch.arange(s["max_q"], device=DEV)
    row = (s["cu_q"][:-1, None] + i).clamp(max=t - 1)  # the padded place (sequence, i) of each query row
    q = s["q"].float()[row].view(b, -1, hk, g, D).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, D)
    seen = s["lens"][:, None] - new[:, None] + i + 1  # the keys that query i sees
    mask = (torch.arange(s["max_k"], device=DEV) < seen[..., None]).repeat(1, g, 1)[:, None]
    o, p = _attended(q, k, v, mask)
    live = (i < new[:, None]).repeat(1, g)[:, None, :, None]
    _add(s, torch.where(live, p, 0.0).sum(2), new)
    o = o.view(b, hk, g, -1, D).permute(0, 3, 1, 2, 4).reshape(b, -1, h, D)
    return o[i < new[:, None]].to(torch.bfloat16), s["weights"]


def _evict(s):
    kv, tables, lens, rows = s["kv"], s["tables"], s["lens"], s["rows"].long()
    n = tables.shape[1] * BS
    most = min(s["budget"], n)
    pos = torch.arange(n, device=DEV)
    left = lens.clamp(max=s["budget"])
    w = s["weights"][:, rows, :, :n]  # [layers, B, HK, n]
    kept = (pos < s["sinks"]) | (pos >= lens[:, None] - s["recent"])
    rank = torch.where(kept[:, None], float("inf"), w).masked_fill((pos >= lens[:, None])[:, None], float("-inf"))
    src = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :most].sort(-1).values
    s["weights"][:, rows, :, :most] = w.gather(3, src)  # (a sequence within the budget keeps every place)
    to = torch.arange(most, device=DEV)
    layer, seq, head, j = (src != to).nonzero(as_tuple=True)
    i = src[layer, seq, head, j]
    a, z = tables[seq, i // BS].long(), tables[seq, j // BS].long()
    for x in _planes(kv):
        x[layer, :, z, j % BS, head] = x[layer, :, a, i % BS, head]
    used = torch.arange(tables.shape[1], device=DEV) < (-(-left // BS))[:, None]
    return torch.where(used, tables, -1), left, kv, s["weights"]


def _planes(kv):
    """The parts of a cache that hold a token's head in one run, as views [layers, 2, blocks, block_size, HK, bytes]: a 4-bit
    block has its codes first, then its scales."""
    if kv.dtype != torch.uint8:
        return (kv,)
    layers, two, blocks, bs, hk, width = kv.shape
    per = bs * hk * width
    outer = (two * blocks * per, blocks * per, per)
    return (kv.as_strided((layers, two, blocks, bs, hk, 64), (*outer, hk * 64, 64, 1)),
            kv.as_strided((layers, two, blocks, bs, hk, 4), (*outer, hk * 4, 4, 1), kv.storage_offset() + bs * hk * 64))


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    h, hk, seqs = case["heads"], case["kv_heads"], _sequences(case)
    if case["kind"] == "evict":
        over = [n for _, n in seqs if n > case["budget"]]
        # every weight read; the kept tokens behind the first ones read and written in both caches, with their weights
        moved = len(over) * (case["budget"] - case["sinks"])
        row = 68 if case["four_bit"] else 2 * D
        return {"bytes": case["layers"] * hk * (4 * sum(over) + moved * (4 * row + 4)) + 1, "flops": 0}
    new, keys = sum(n for n, _ in seqs), sum(n for _, n in seqs)
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in seqs)
    rows = new * 2 * hk * 4 * D if case.get("store") else 0
    # queries and outputs, keys and values once, the cached tokens' weights read and everyone's written
    return {"bytes": new * h * D * 4 + keys * hk * (4 * D + 4) + (keys - new) * hk * 4 + rows, "flops": 4 * D * h * pairs}


# ----------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits


def _exact_attention(q, k, v, group):
    """Queries [n, H, 128], the last n positions of keys [m, HK, 128]: outputs [n, H, 128], and what every key receives of
    them [HK, m]."""
    n, m, hk = q.shape[0], k.shape[0], k.shape[1]
    keys = k.repeat_interleave(group, 1).permute(1, 2, 0).contiguous()
    values = v.repeat_interleave(group, 1).transpose(0, 1).contiguous()
    x = torch.matmul(q.double().transpose(0, 1).contiguous(), keys) * SCALE
    late = torch.arange(m, device=q.device)[None] > torch.arange(n, device=q.device)[:, None] + (m - n)
    p = torch.softmax(x.masked_fill(late, float("-inf")), -1)
    return torch.matmul(p, values).transpose(0, 1), p.sum(1).view(hk, group, m).sum(1)


def _exact_evict(case, x):
    kv, weights, tables = x["kv"], x["weights"], x["tables"].tolist()
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    for row, n, blocks in zip(x["rows"].tolist(), x["lens"].tolist(), tables):
        if n <= budget:
            continue
        blocks = torch.tensor(blocks[:-(-n // BS)], device=DEV)
        mid = weights[:, row, :, sinks:n - recent].double()
        # the place of each of them among the others: how many are larger, or equal and earlier
        place = torch.empty_like(mid, dtype=torch.long)
        place.scatter_(2, torch.argsort(-mid, dim=2, stable=True), torch.arange(mid.shape[2], device=DEV).expand_as(mid).contiguous())
        keep = torch.ones(*mid.shape[:2], n, dtype=torch.bool, device=DEV)
        keep[..., sinks:n - recent] = place < budget - sinks - recent
        for layer in range(case["layers"]):
            for head in range(case["kv_heads"]):
                at = keep[layer, head].nonzero()[:, 0]
                weights[layer, row, head, :budget] = weights[layer, row, head, at].clone()
                for part in _planes(kv):
                    both = part[layer, :, blocks, :, head].flatten(1, 2)  # [2, tokens of the blocks, bytes]
                    both[:, :budget] = both[:, at].clone()
                    part[layer, :, blocks, :, head] = both.view(2, -1, BS, both.shape[2])
    return None, None, None if case["four_bit"] else kv, weights


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(case, x)
    out, at, group = [], 0, case["heads"] // case["kv_heads"]
    weights, store = x["weights"].double(), "slots" in x
    if store:
        for i, slot in enumerate(x["slots"].tolist()):
            x["k_cache"].view(-1, case["kv_heads"], D)[slot] = x["k"][i]
            x["v_cache"].view(-1, case["kv_heads"], D)[slot] = x["v"][i]
    for b, (new, n) in enumerate(_sequences(case)):
        if case["kind"] == "chunk" and case["packed"]:
            k, v = (x[c][at:at + n].double() for c in ("k", "v"))  # (as many keys as queries)
        else:
            blocks = x["tables"][b, :-(-n // BS)].long()
            k, v = (x[c][blocks].flatten(0, 1)[:n].double() for c in ("k_cache", "v_cache"))
        mine = weights[int(x["rows"][b])]
        mine[:, n - new:n] = 0
        for a in range(0, new, 256):  # queries in slices, for their scores' memory
            e = min(new, a + 256)
            m = n - new + e
            o, got = _exact_attention(x["q"][at + a:at + e], k[:m], v[:m], group)
            out.append(o)
            mine[:, :m] += got
        at += new
    o = torch.cat(out)
    return (o, weights, x["k_cache"], x["v_cache"]) if store else (o, weights)
