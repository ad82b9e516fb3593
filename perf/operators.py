"""Operators around the paged KV cache that is held in 8 bits, as a serving program runs them, for timing and for comparing outputs.

The cache holds K and V as e4m3 numbers `[blocks, block_size, kv_heads, head_dim]` and a power-of-two scale for each block and
kv head `[blocks, kv_heads]` of K and of V; a value stands for number x scale.  Four operators: the layout of a packed step built on
the GPU from request lengths, the append of new K/V rows, decode attention, packed prefill attention.  `prepare` makes what a
program holds before the call, `run` is one pass, `work` the bytes and operations that the pass cannot do without, `exact` the
outputs from the definition in 64 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

MODEL = "8x2x256x16"  # query heads, kv heads, head_dim, tokens per block: the model of this repository's benchmark
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
LARGEST = 448.0  # of e4m3
LOW, HIGH = -117, 119  # exponents a scale may have
MOST_KEYS = 60 * 20480  # keys of a drawn decode case


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # a full decode batch's block tables grown and its slots found on the device, one token per row: latency
        {"name": "layout_decode_256", "kind": "layout", "rows": 256, "cached": 4096, "new": 1, "width": 512, "bs": 16, "pad": 0},
        # admission of a burst of prompts in one packed step: the largest plan
        {"name": "layout_prompts_4096", "kind": "layout", "rows": 4096, "cached": 512, "new": 63, "width": 64, "bs": 16, "pad": 777},
        # one layer's append of a decode step: a token per row, most blocks partly filled
        {"name": "append_decode_256", "kind": "append", "rows": 256, "tokens": 256, "cached": 2048, "heads": MODEL, "dtype": "bfloat16", "pad": 0},
        # one layer's append of a large packed prefill step: five requests at different depths
        {"name": "append_prompts_16384", "kind": "append", "rows": 5, "tokens": 16384, "cached": 1000, "heads": MODEL, "dtype": "bfloat16", "pad": 0},
        # the same in fp32 activations, more and shorter heads, a padded bucket
        {"name": "append_777_fp32", "kind": "append", "rows": 7, "tokens": 777, "cached": 300, "heads": "32x8x128x16", "dtype": "float32", "pad": 23},
        # a handful of short requests in a padded decode batch: latency is all there is
        {"name": "decode_4_rows", "kind": "decode", "rows": 4, "lo": 64, "hi": 512, "wide": 1, "heads": MODEL, "dtype": "bfloat16", "empty": 1},
        # decode-heavy serving: a full batch at mixed depths
        {"name": "decode_256_rows", "kind": "decode", "rows": 256, "lo": 1024, "hi": 4096, "wide": 1, "heads": MODEL, "dtype": "bfloat16", "empty": 0},
        # long conversations: the largest decode batch
        {"name": "decode_64_long_rows", "kind": "decode", "rows": 64, "lo": 8192, "hi": 32768, "wide": 1, "heads": MODEL, "dtype": "bfloat16", "empty": 0},
        # eight kv heads of 128, blocks of 32 tokens, fp16 queries
        {"name": "decode_48_rows_heads_8", "kind": "decode", "rows": 48, "lo": 200, "hi": 3000, "wide": 1, "heads": "32x8x128x32", "dtype": "float16", "empty": 0},
        # verification of speculated tokens: five query tokens per row
        {"name": "verify_64x5", "kind": "decode", "rows": 64, "lo": 1024, "hi": 4096, "wide": 5, "heads": MODEL, "dtype": "bfloat16", "empty": 0},
        # chunked prefill: a 512-token chunk made up of three requests at different depths
        {"name": "prefill_chunk_512", "kind": "prefill", "rows": 3, "tokens": 512, "cached": 1024, "heads": MODEL, "dtype": "bfloat16", "pad": 0},
        # a long prompt in one chunk: the largest prefill
        {"name": "prefill_16384", "kind": "prefill", "rows": 1, "tokens": 16384, "cached": 0, "heads": MODEL, "dtype": "bfloat16", "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("layout", "append", "append", "decode", "decode", "decode", "prefill", "prefill"))
    heads = rng.choice((MODEL, MODEL, "32x8x128x16", "32x8x128x32", "16x2x64x16", "4x4x64x48", "24x2x128x64", "16x1x256x16"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    hq, hkv, d, bs = _heads({"heads": heads})
    width = hkv * d
    if kind == "layout":
        rows, new = _log(rng, 1, 4096), _log(rng, 1, 4096)
        new = max(1, min(new, 131072 // rows))
        bs, cached = rng.choice((16, 16, 32, 64)), rng.choice((0, _log(rng, 1, 4096)))
        return {"kind": kind, "rows": rows, "cached": cached, "new": new, "width": -(-(cached + 2 * new) // bs) + rng.randint(0, 40), "bs": bs,
                "pad": rng.choice((0, rng.randint(1, 900)))}
    if kind == "append":
        rows = _log(rng, 1, 512)
        tokens = max(rows, _log(rng, 1, 16384 if width <= 512 else 8192))
        return {"kind": kind, "rows": rows, "tokens": tokens, "cached": rng.choice((0, _log(rng, 1, 2048))), "heads": heads, "dtype": dtype,
                "pad": rng.choice((0, rng.randint(1, 99)))}
    if kind == "decode":
        hi, rows = _log(rng, 16, 32768), _log(rng, 1, 512)
        lo = max(1, hi // rng.choice((1, 2, 4, 8, 30)))
        wide = rng.choice((1, 1, 1, rng.randint(2, 9)))
        cost = max(1, width // 512) * (wide if wide > 4 else 1)
        rows = max(1, min(rows, MOST_KEYS // cost // hi))
        return {"kind": kind, "rows": rows, "lo": lo, "hi": hi, "wide": wide, "heads": heads, "dtype": dtype, "empty": rng.choice((0, 0, 1, 3))}
    tokens = _log(rng, 17, 8192 if heads == MODEL and dtype == "bfloat16" else 2048)
    return {"kind": kind, "rows": max(1, min(rng.randint(1, 8), tokens // 16)), "tokens": tokens,
            "cached": rng.choice((0, _log(rng, 16, 2048))), "heads": heads, "dtype": dtype, "pad": rng.choice((0, -tokens % 64, 5))}


# ------------------------------------------------------------------------------------------------ sizes

def _heads(case):
    """(query heads, kv heads, head_dim, tokens per block)"""
    return [int(n) for n in case["heads"].split("x")]


def _spread(lo, hi, n):
    """n lengths over [lo, hi], evenly."""
    return [int(round(lo + (hi - lo) * (i + 0.5) / n)) for i in range(n)]


def _chunks(case):
    """(new tokens, tokens already cached) of each row of a packed batch: ragged, every row at another depth."""
    n, tokens = case["rows"], case["tokens"]
    if tokens == n:  # a decode step
        return [(1, c) for c in _spread(case["cached"] // 2, case["cached"] * 2, n)]
    cuts = [i + (tokens - n) * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]
    return [(cuts[i + 1] - cuts[i], case["cached"] * (n - i) // n) for i in range(n)]


def _layout_rows(case):
    """(new tokens, cached tokens) of each row of a plan: up to twice the mean, one row in eight without new tokens unless it is a decode step."""
    n = case["rows"]
    if case["new"] == 1:
        return [(1, c) for c in _spread(case["cached"] // 2, case["cached"], n)]
    return [(0 if i % 8 == 5 else 1 + (i * 37) % (2 * case["new"] - 1), (i * 101) % (case["cached"] + 1)) for i in range(n)]


def work(case):
    """Every input read once and every output written once; products of the visible keys alone."""
    kind = case["kind"]
    if kind == "layout":
        rows, bs = _layout_rows(case), case["bs"]
        fresh = sum(-(-(n + c) // bs) - -(-c // bs) for n, c in rows)
        tokens = sum(n for n, _ in rows) + case["pad"]
        return {"bytes": 16 * len(rows) + 8 * fresh + 12 * tokens, "flops": 0}
    hq, hkv, d, bs = _heads(case)
    item = DTYPES[case["dtype"]].itemsize
    if kind == "append":
        rows = _chunks(case)
        tokens = sum(n for n, _ in rows)
        blocks = sum(-(-(n + c) // bs) - c // bs for n, c in rows)
        return {"bytes": 2 * tokens * hkv * d * (item + 1) + blocks * (4 + 16 * hkv) + 8 * tokens, "flops": 0}
    rows = _chunks(case) if kind == "prefill" else [(case["wide"], max(0, x - case["wide"])) for x in _spread(case["lo"], case["hi"], case["rows"])]
    tokens, live = sum(n for n, _ in rows), sum(n + c for n, c in rows)
    blocks = sum(-(-(n + c) // bs) for n, c in rows)
    return {"bytes": 2 * live * hkv * d + blocks * (4 + 8 * hkv) + tokens * hq * d * (item + 4) + 8 * tokens,
            "flops": 4 * hq * d * sum(n * c + n * (n + 1) // 2 for n, c in rows)}


# ------------------------------------------------------------------------------------------------ inputs

def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, dtype, *shape):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(dtype)


def _held(g, blocks, heads):
    """Filled blocks: N(0, 1) values, louder and quieter blocks among them, as e4m3 numbers and scales."""
    _, hkv, d, bs = heads
    x = torch.empty(blocks, bs, hkv, d, device="cuda").normal_(generator=g)
    x *= torch.randint(-2, 3, (blocks, 1, hkv, 1), generator=g, device="cuda").float().exp2()
    mantissa, power = torch.frexp(x.abs().amax((1, 3)))
    scale = torch.ldexp(torch.ones_like(mantissa), power - 9 + (mantissa > 0.875))
    return (x / scale[:, None, :, None]).to(torch.float8_e4m3fn), scale


def _tables(g, room, bs, extra=0):
    """Block tables with room for `room[b]` tokens in row b, scattered over a pool a little larger than that; unused entries 0."""
    need = [-(-r // bs) for r in room]
    pool = sum(need) + sum(need) // 8 + 8
    ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    mask = torch.arange(max(need) + extra, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    tables = torch.zeros(len(need), max(need) + extra, dtype=torch.int32, device="cuda")
    tables[mask] = ids[: sum(need)]
    return tables, pool, ids[sum(need):]


def _packed(rows, pad):
    """positions, token_row_ids [1, T], query_start_loc and lengths of a packed batch, padded with (position 0, row 0)."""
    positions = np.concatenate([np.arange(c, c + n) for n, c in rows] + [np.zeros(pad)]).astype(np.int32)
    owners = np.concatenate([np.full(n, i) for i, (n, _) in enumerate(rows)] + [np.zeros(pad)]).astype(np.int32)
    qsl = np.concatenate([[0], np.cumsum([n for n, _ in rows])]).astype(np.int32)
    return (torch.from_numpy(positions)[None].cuda(), torch.from_numpy(owners)[None].cuda(), torch.from_numpy(qsl).cuda(),
            _int([n + c for n, c in rows]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "layout":
        rows = _layout_rows(case)
        order = torch.randperm(len(rows), generator=g, device="cuda").cpu().tolist()
        rows = [rows[i] for i in order]
        bs = case["bs"]
        held = [-(-c // bs) for _, c in rows]
        need = [-(-(n + c) // bs) - h for (n, c), h in zip(rows, held)]
        ids = torch.randperm(sum(held) + sum(need) + 500, generator=g, device="cuda").to(torch.int32)
        tables = torch.zeros(len(rows), case["width"], dtype=torch.int32, device="cuda")
        mask = torch.arange(case["width"], device="cuda")[None] < torch.tensor(held, device="cuda")[:, None]
        tables[mask] = ids[: sum(held)]
        return {"case": case, "cached": _int([c for _, c in rows]), "new": _int([n for n, _ in rows]), "tables": tables,
                "free": ids[sum(held):].contiguous(), "head": _int([37]), "bucket": sum(n for n, _ in rows) + case["pad"]}
    heads, dtype = _heads(case), DTYPES[case["dtype"]]
    hq, hkv, d, bs = heads
    if kind == "decode":
        lens = _spread(case["lo"], case["hi"], case["rows"])
        lens = [lens[i] for i in torch.randperm(len(lens), generator=g, device="cuda").cpu().tolist()]
        tables, pool, _ = _tables(g, lens + [1] * case["empty"], bs)
        lens = lens + [0] * case["empty"]  # a batch padded to its bucket
        wide = case["wide"]
        (k, ks), (v, vs) = _held(g, pool, heads), _held(g, pool, heads)
        return {"case": case, "k": k, "v": v, "ks": ks, "vs": vs, "tables": tables, "lens": _int(lens),
                "q": _normal(g, dtype, len(lens), wide, hq, d) if wide > 1 else _normal(g, dtype, len(lens), hq, d),
                "pos": _int([[max(0, x - wide + t) for t in range(wide)] for x in lens]) if wide > 1 else None}
    rows = _chunks(case)
    tables, pool, _ = _tables(g, [n + c for n, c in rows], bs, extra=3)
    (k, ks), (v, vs) = _held(g, pool, heads), _held(g, pool, heads)
    positions, owners, qsl, lens = _packed(rows, case["pad"])
    tokens = positions.shape[1]
    state = {"case": case, "k": k, "v": v, "ks": ks, "vs": vs, "tables": tables, "lens": lens, "pos": positions, "owners": owners, "qsl": qsl}
    if kind == "append":
        return dict(state, new_k=_normal(g, dtype, 1, tokens, hkv, d) * 3, new_v=_normal(g, dtype, 1, tokens, hkv, d) * 3,
                    most=max(n for n, _ in rows))
    singles = sum(n == 1 for n, _ in rows)
    return dict(state, q=_normal(g, dtype, 1, tokens, hq, d), most=max(n for n, _ in rows), singles=singles,
                tiles=sum(-(-n // 64) for n, _ in rows if n > 1))


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state, kind)
    return {"layout": _plain_layout, "append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[kind](state)


_modules = None


def _own(s, kind):
    global _modules
    if _modules is None:
        from nano_vllm_jax_b200.kernels import paged_kv, quantized_kv
        _modules = paged_kv, quantized_kv
    paged, quantized = _modules
    case = s["case"]
    if kind == "layout":
        p = paged.build_packed_layout(s["cached"], s["new"], s["tables"], s["free"], s["head"], case["bs"], s["bucket"])
        return p.positions, p.token_row_ids, p.slot_mapping, p.query_start_loc, p.seq_lens, p.free_head, s["tables"]
    if kind == "append":
        return quantized.kv_append_quantized(s["new_k"], s["new_v"], s["k"], s["v"], s["ks"], s["vs"], s["pos"], s["tables"],
                                             query_start_loc=s["qsl"], token_row_ids=s["owners"])
    hq, hkv, d, bs = _heads(case)
    if kind == "decode":
        return quantized.paged_decode_attention_quantized(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"], d ** -0.5,
                                                          positions=s["pos"])
    return quantized.packed_paged_prefill_attention_quantized(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"], s["pos"],
                                                              s["qsl"], bs, d ** -0.5, hq // hkv, num_decode_rows=s["singles"],
                                                              query_tile_pairs=s["tiles"])


def _plain_layout(s):
    cached, new, tables, free, head = s["cached"].long(), s["new"].long(), s["tables"], s["free"], s["head"].long()
    bs, bucket, dev = s["case"]["bs"], s["bucket"], s["cached"].device
    held = (cached + bs - 1) // bs
    need = (cached + new + bs - 1) // bs - held
    qsl = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    first = head + need.cumsum(0) - need
    column = torch.arange(tables.shape[1], device=dev)[None] - held[:, None]
    fresh = (column >= 0) & (column < need[:, None])
    tables.copy_(torch.where(fresh, free[(first[:, None] + column).clamp(0, free.numel() - 1)], tables))
    token = torch.arange(bucket, device=dev)
    row = torch.searchsorted(qsl[1:].contiguous(), token, right=True)
    live = token < qsl[-1]
    row = torch.where(live, row, 0)
    position = torch.where(live, cached[row] + token - qsl[row], 0)
    slot = torch.where(live, tables[row, position // bs].long() * bs + position % bs, -1)
    i32 = torch.int32
    return (position.to(i32)[None], row.to(i32)[None], slot.to(i32)[None], qsl.to(i32), (cached + new).to(i32), (head + need.sum()).to(i32), tables)


def _power(largest):
    """Exponent of a block's scale for its largest finite magnitude: the least e with largest <= 448 * 2^e."""
    mantissa, power = torch.frexp(largest)
    return torch.where(largest > 0, power - 9 + (mantissa > 0.875), LOW).clamp(LOW, HIGH)


def _plain_append(s):
    hq, hkv, d, bs = _heads(s["case"])
    qsl, pos, tables = s["qsl"].long(), s["pos"][0].long(), s["tables"].long()
    start, count = pos[qsl[:-1]], qsl.diff()
    columns = (s["most"] + bs - 2) // bs + 1  # blocks that a row's new tokens may touch
    column = start[:, None] // bs + torch.arange(columns, device=pos.device)[None]
    place = column[:, :, None] * bs + torch.arange(bs, device=pos.device)  # positions of those blocks' tokens [rows, columns, bs]
    fresh = (place >= start[:, None, None]) & (place < (start + count)[:, None, None])
    touched = fresh.any(-1)
    ids = tables.gather(1, column.clamp(max=tables.shape[1] - 1))
    source = (qsl[:-1, None, None] + place - start[:, None, None]).clamp(0, pos.numel() - 1)
    begun = fresh[:, :, 0][..., None]  # the block's first token is among the new ones
    out = []
    for new, held, scale in ((s["new_k"][0], s["k"], s["ks"]), (s["new_v"][0], s["v"], s["vs"])):
        x = torch.where(fresh[..., None, None], new[source].float(), 0.0)  # [rows, columns, bs, hkv, d]
        old_scale = scale[ids]
        largest = torch.where(torch.isfinite(x), x.abs(), 0.0).amax((2, 4))
        wanted = torch.ldexp(torch.ones_like(largest), _power(largest))
        new_scale = torch.where(begun, wanted, torch.maximum(wanted, old_scale))
        fits = (x / new_scale[:, :, None, :, None]).clamp(-LARGEST, LARGEST)
        ratio = torch.where(begun, 1.0, old_scale / new_scale)
        kept = held[ids].float() * ratio[:, :, None, :, None]
        both = torch.where(fresh[..., None, None], fits, kept).to(torch.float8_e4m3fn)
        where = ids[touched]
        held.view(torch.uint8)[where] = both.view(torch.uint8)[touched]
        scale[where] = new_scale[touched]
        out += [held, scale]
    return out[0], out[2], out[1], out[3]


def _values(held, scale, ids):
    """fp32 values of the blocks of a table: [rows, kv heads, keys, head_dim]."""
    x = held[ids].float() * scale[ids][:, :, None, :, None]
    return x.flatten(1, 2).transpose(1, 2)


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v for q [rows, hkv, groups * tokens, d] over the keys that `seen` [rows, 1, queries, keys] lets through."""
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(q.shape[-1] ** -0.5).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight, v) / torch.where(total > 0, total, 1.0)


def _plain_decode(s):
    hq, hkv, d, bs = _heads(s["case"])
    wide, ids, lens = s["case"]["wide"], s["tables"].long(), s["lens"].long()
    rows, groups = lens.numel(), hq // hkv
    k, v = _values(s["k"], s["ks"], ids), _values(s["v"], s["vs"], ids)
    key = torch.arange(k.shape[2], device=k.device)
    live = key[None] < lens[:, None]
    v = torch.where(live[:, None, :, None], v, 0.0)
    seen = live[:, None, :]
    if wide > 1:
        seen = seen & (key[None, None] <= s["pos"].long()[:, :, None])
    q = s["q"].float().view(rows, wide, hkv, groups, d).permute(0, 2, 3, 1, 4).reshape(rows, hkv, groups * wide, d)
    out = _attend(q, k, v, seen.repeat(1, groups, 1)[:, None])
    out = out.view(rows, hkv, groups, wide, d).permute(0, 3, 1, 2, 4)
    return out.reshape(rows, wide, hq * d) if wide > 1 else out.reshape(rows, hq, d)


def _plain_prefill(s):
    hq, hkv, d, bs = _heads(s["case"])
    ids, lens, qsl, pos = s["tables"].long(), s["lens"].long(), s["qsl"].long(), s["pos"][0].long()
    rows, groups, most, tokens = lens.numel(), hq // hkv, s["most"], pos.numel()
    k, v = _values(s["k"], s["ks"], ids), _values(s["v"], s["vs"], ids)
    key, step = torch.arange(k.shape[2], device=k.device), torch.arange(most, device=k.device)
    live = key[None] < lens[:, None]
    v = torch.where(live[:, None, :, None], v, 0.0)
    index = (qsl[:-1, None] + step[None]).clamp(max=tokens - 1)  # [rows, most]
    seen = live[:, None, :] & (key[None, None] <= pos[index][:, :, None])
    q = s["q"][0][index].float().view(rows, most, hkv, groups, d).permute(0, 2, 3, 1, 4).reshape(rows, hkv, groups * most, d)
    out = _attend(q, k, v, seen.repeat(1, groups, 1)[:, None])
    out = out.view(rows, hkv, groups, most, d).permute(0, 3, 1, 2, 4).reshape(rows, most, hq * d)
    token = torch.arange(tokens, device=k.device)
    inside = token < qsl[-1]
    row = s["owners"][0].long()
    picked = out[row, (token - qsl[row]).clamp(0, most - 1)]
    return torch.where(inside[:, None], picked, 0.0)[None]


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def _nearest_e4m3(x):
    """The e4m3 number next to each x (ties to the even one), magnitudes over 448 held at 448."""
    size = np.abs(x)
    _, power = np.frexp(np.where(size > 0, size, 1.0))
    step = np.exp2(np.maximum(power - 1, -6) - 3.0)
    return np.sign(x) * np.minimum(np.rint(size / step) * step, LARGEST)


def exact(case, seed):
    if case["kind"] == "layout":
        return None
    s = prepare(case, seed)
    hq, hkv, d, bs = _heads(case)
    if case["kind"] == "append":
        return _exact_append(case, s)
    lens, tables = s["lens"].tolist(), s["tables"]
    if case["kind"] == "decode":
        wide = case["wide"]
        q = s["q"].double().view(len(lens), wide, hq, d)
        out = torch.zeros(len(lens), wide, hq, d, dtype=torch.float64, device=q.device)
        for b, n in enumerate(lens):
            if n > 0:
                limits = s["pos"][b].long() if wide > 1 else torch.tensor([n - 1], device=q.device)
                _exact_row(out[b], q[b], s, tables[b], n, limits, hkv, bs)
        return out.reshape(len(lens), wide, hq * d) if wide > 1 else out[:, 0]
    q = s["q"][0].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    cuts = s["qsl"].tolist()
    for b, n in enumerate(lens):
        for lo in range(cuts[b], cuts[b + 1], 1024):
            hi = min(lo + 1024, cuts[b + 1])
            _exact_row(out[lo:hi], q[lo:hi], s, tables[b], n, s["pos"][0, lo:hi].long(), hkv, bs)
    return out.reshape(1, q.shape[0], hq * d)


def _exact_row(out, q, s, table, n, limits, hkv, bs):
    """out[t] for the query tokens q [t, hq, d] of one row of n keys; token t sees the keys up to limits[t]."""
    blocks = table[: -(-n // bs)].long()
    groups = q.shape[1] // hkv
    hidden = torch.arange(n, device=q.device)[None] > limits[:, None]
    for h in range(hkv):
        k = (s["k"][blocks, :, h].double() * s["ks"][blocks, h].double()[:, None, None]).flatten(0, 1)[:n]
        v = (s["v"][blocks, :, h].double() * s["vs"][blocks, h].double()[:, None, None]).flatten(0, 1)[:n]
        for j in range(h * groups, (h + 1) * groups):
            score = ((q[:, j] @ k.T) / math.sqrt(q.shape[2])).masked_fill(hidden, -math.inf)
            out[:, j] = torch.softmax(score, -1) @ v


def _exact_append(case, s):
    hq, hkv, d, bs = _heads(case)
    tables = s["tables"].cpu().numpy()
    out = []
    for new, held, scale in ((s["new_k"], s["k"], s["ks"]), (s["new_v"], s["v"], s["vs"])):
        new, held, scale = (t.double().cpu().numpy() for t in (new[0], held, scale))
        at = 0
        for b, (n, c) in enumerate(_chunks(case)):
            first = c
            while first < c + n:
                last = min((first // bs + 1) * bs, c + n)
                block, lo = tables[b, first // bs], first % bs
                x = new[at + first - c: at + last - c]
                for h in range(hkv):
                    largest = np.abs(x[:, h]).max()
                    e = LOW
                    if largest > 0:
                        e = int(math.frexp(largest)[1]) - 10
                        while largest > LARGEST * 2.0 ** e:
                            e += 1
                    e = min(max(e, LOW), HIGH)
                    now = 2.0 ** e if lo == 0 else max(2.0 ** e, scale[block, h])
                    if lo > 0 and now > scale[block, h]:
                        held[block, :, h] = _nearest_e4m3(held[block, :, h] * (scale[block, h] / now))
                    held[block, lo: lo + len(x), h] = _nearest_e4m3(x[:, h] / now)
                    scale[block, h] = now
                first = last
            at += n
        out += [torch.from_numpy(held), torch.from_numpy(scale)]
    return out[0], out[2], out[1], out[3]
