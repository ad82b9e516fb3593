"""Operators of a paged cache whose decode attention reads selected blocks, as a serving program runs them, for timing and for comparing outputs.

Beside the pages K and V `[blocks, block_size, kv_heads, head_dim]` such a cache holds the bounds of every block's keys
`[blocks, kv_heads, 2, head_dim]`: the smallest and the largest number of each dimension.  Three operators: the append, which rotates
queries and keys by their positions on the way and keeps the bounds; the selection, which scores every block of a row by an upper
bound of query x key and takes the best; attention over the selected blocks.  A fourth kind of case runs them together through the
backend, as a decode step of one layer.  `prepare` makes what a program holds before the call, `run` is one pass, `work` the bytes
and operations that the pass cannot do without, `exact` the outputs from the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

MODEL = "8x2x256x16"  # query heads, kv heads, head_dim, tokens per block: the model of this repository's benchmark
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BASE = 1e7  # of the rotation's frequencies
MOST_BLOCKS = 32 * 4096 * 2  # blocks x kv heads that a drawn selection scores


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    bf16, f16, f32 = "bfloat16", "float16", "float32"
    return [
        # one layer's append of a full decode batch: a token per row, most blocks partly filled; queries and keys are views of one projection
        {"name": "append_decode_256", "kind": "append", "rows": 256, "tokens": 256, "cached": 2048, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "rot": 64, "pairs": False, "pad": 0},
        # one layer's append of a large packed prefill step: five requests at different depths
        {"name": "append_prompts_16384", "kind": "append", "rows": 5, "tokens": 16384, "cached": 1000, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "rot": 64, "pairs": False, "pad": 0},
        # fp32 activations and cache, more and shorter heads, every dimension rotated in neighbouring pairs, a padded bucket
        {"name": "append_777_fp32", "kind": "append", "rows": 7, "tokens": 777, "cached": 300, "heads": "32x8x128x16", "dtype": f32, "cache": f32,
         "rot": 128, "pairs": True, "pad": 23},
        # a handful of requests in a padded decode batch: latency is all there is
        {"name": "select_4_rows", "kind": "select", "rows": 4, "lo": 500, "hi": 4000, "wide": 1, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 32, "empty": 1},
        # a full decode batch at middle depths
        {"name": "select_256_rows", "kind": "select", "rows": 256, "lo": 2048, "hi": 8192, "wide": 1, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 64, "empty": 0},
        # long conversations: the most blocks to score
        {"name": "select_64_long_rows", "kind": "select", "rows": 64, "lo": 16384, "hi": 65536, "wide": 1, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 128, "empty": 0},
        # the same small decode batch's attention
        {"name": "attend_4_rows", "kind": "attend", "rows": 4, "lo": 500, "hi": 4000, "wide": 1, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 32, "empty": 1},
        # ... and the full one's: the most bytes of selected keys
        {"name": "attend_256_rows", "kind": "attend", "rows": 256, "lo": 2048, "hi": 8192, "wide": 1, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 64, "empty": 0},
        # eight kv heads of 128, blocks of 32 tokens, fp16
        {"name": "attend_48_rows_heads_8", "kind": "attend", "rows": 48, "lo": 1000, "hi": 9000, "wide": 1, "heads": "32x8x128x32", "dtype": f16,
         "cache": f16, "budget": 48, "empty": 0},
        # verification of speculated tokens: five query tokens per row, each with a selection of its own
        {"name": "attend_verify_32x5", "kind": "attend", "rows": 32, "lo": 1024, "hi": 4096, "wide": 5, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 64, "empty": 0},
        # one layer's decode step through the backend, append, selection and attention: few rows
        {"name": "step_8_rows", "kind": "step", "rows": 8, "lo": 2000, "hi": 16000, "wide": 1, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 64, "empty": 0},
        # ... and many
        {"name": "step_128_rows", "kind": "step", "rows": 128, "lo": 4096, "hi": 16384, "wide": 1, "heads": MODEL, "dtype": bf16, "cache": bf16,
         "budget": 64, "empty": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "append", "select", "select", "attend", "attend", "step"))
    heads = rng.choice((MODEL, MODEL, "32x8x128x16", "32x8x128x32", "16x2x64x16", "4x4x64x48", "24x2x128x64", "16x1x256x16", "6x3x96x16"))
    dtype, cache = rng.choice((("bfloat16", "bfloat16"),) * 3 + (("float16", "float16"), ("float32", "float32"), ("float32", "bfloat16")))
    hq, hkv, d, bs = _heads({"heads": heads})
    if kind == "append":
        rows = _log(rng, 1, 512)
        tokens = max(rows, _log(rng, 1, 16384 if hq * d <= 2048 and dtype != "float32" else 4096))
        return {"kind": kind, "rows": rows, "tokens": tokens, "cached": rng.choice((0, _log(rng, 1, 2048))), "heads": heads, "dtype": dtype,
                "cache": cache, "rot": rng.choice((d, d // 2, min(64, d), 16, 0)), "pairs": rng.choice((False, False, True)),
                "pad": 0 if tokens == rows else rng.choice((0, rng.randint(1, 99)))}
    hi, rows = _log(rng, 16, 65536 if kind == "select" else 16384), _log(rng, 1, 256)
    lo = max(1, hi // rng.choice((1, 2, 4, 8, 30)))
    wide = 1 if kind == "step" else rng.choice((1, 1, 1, rng.randint(2, 6)))
    budget = rng.choice((_log(rng, 4, 128), 64, 32))
    if kind == "select":  # (a row of more blocks than are selected: the others leave nothing to choose)
        hi = max(hi, 8 * bs)
        budget = max(FIRST + LAST, min(budget, -(-((lo + hi) // 2) // bs) - 1))
        rows = min(rows, MOST_BLOCKS // (wide * hkv * max(1, d // 128) * max(1, hq // hkv // 4) * -(-hi // bs)))
    else:
        dear = DTYPES[cache].itemsize // 2 * (2 if kind == "step" else 1)
        each = max(1, hi * hkv * d * dear // 512)  # bytes of a row's cache over 2 KiB
        rows = min(rows, 256 * 6000 // each, 256 * 64 * 16 * 512 // (min(budget * bs, hi) * wide * hkv * d * dear * max(1, hq // hkv // 4)))
    return {"kind": kind, "rows": max(1, rows), "lo": lo, "hi": hi, "wide": wide, "heads": heads, "dtype": dtype, "cache": cache, "budget": budget,
            "empty": rng.choice((0, 0, 1, 3))}


# ------------------------------------------------------------------------------------------------ sizes

FIRST, LAST = 1, 2  # blocks at a row's two ends that are always selected


def _heads(case):
    """(query heads, kv heads, head_dim, tokens per block)"""
    return [int(n) for n in case["heads"].split("x")]


def _spread(lo, hi, n):
    """n lengths over [lo, hi], evenly."""
    return [int(round(lo + (hi - lo) * (i + 0.5) / n)) for i in range(n)]


def _chunks(case):
    """(new tokens, tokens already cached) of each row of an append: ragged, every row at another depth."""
    n, tokens = case["rows"], case["tokens"]
    if tokens == n:  # a decode step
        return [(1, c) for c in _spread(case["cached"] // 2, case["cached"] * 2, n)]
    cuts = [i + (tokens - n) * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]
    return [(cuts[i + 1] - cuts[i], case["cached"] * (n - i) // n) for i in range(n)]


def _visible(case):
    """Keys that each query token sees, row by row."""
    wide = case["wide"]
    return [max(0, x - wide + t + 1) for x in _spread(case["lo"], case["hi"], case["rows"]) for t in range(wide)]


def work(case):
    """Every input read once and every output written once; products of the selected keys alone."""
    kind = case["kind"]
    hq, hkv, d, bs = _heads(case)
    item, held = DTYPES[case["dtype"]].itemsize, DTYPES[case["cache"]].itemsize
    bytes_, flops = 0, 0
    if kind in ("append", "step"):
        rows = _chunks(case) if kind == "append" else [(1, x - 1) for x in _spread(case["lo"], case["hi"], case["rows"])]
        tokens = sum(n for n, _ in rows)
        touched = sum(-(-(n + c) // bs) - c // bs for n, c in rows)
        begun = sum(-(-(n + c) // bs) - -(-c // bs) for n, c in rows)
        bytes_ += tokens * 2 * hkv * d * (item + held) + (2 * touched - begun) * hkv * 2 * d * held + 4 * tokens + 4 * touched
        if kind == "append":
            return {"bytes": bytes_ + tokens * 2 * hq * d * item, "flops": 3 * tokens * (hq + hkv) * case["rot"]}
    budget = case["budget"]
    if kind in ("select", "step"):
        wide = case["wide"]
        seen = [-(-n // bs) for n in _visible(case)]
        scored = [n for n in seen if n > budget]
        rows_of = [n for n in seen[wide - 1:: wide] if n > budget]  # a row's bounds are read once for all of its tokens
        bytes_ += sum(rows_of) * (hkv * 2 * d * held + 4) + len(seen) * (hq * d * item + 4 * hkv * budget + 4)
        flops += 4 * hq * d * sum(scored)
        if kind == "select":
            return {"bytes": bytes_, "flops": flops}
    wide = case["wide"]
    keys = [min(n, budget * bs) for n in _visible(case)]
    last = _visible(case)[wide - 1:: wide]
    read = sum(min(n, wide * budget * bs) for n in last)  # the tokens of a row select blocks of one cache
    tokens = len(keys)
    bytes_ += 2 * read * hkv * d * held + tokens * (hq * d * (item + 4) + 4 * hkv * budget)
    return {"bytes": bytes_, "flops": flops + 4 * hq * d * sum(keys)}


# ------------------------------------------------------------------------------------------------ inputs

def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, dtype, *shape):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=g).to(dtype)


def _gains(g, hkv, d):
    """Loud and quiet dimensions of the keys, as trained models have them."""
    return torch.empty(hkv, d, device="cuda").normal_(generator=g).mul_(0.5).exp_()


def _pages(g, pool, heads, dtype):
    """Filled blocks of K and V: the keys of a block have something in common, the dimensions differ in loudness."""
    _, hkv, d, bs = heads
    k = torch.empty(pool, bs, hkv, d, device="cuda").normal_(generator=g)
    k += torch.empty(pool, 1, hkv, d, device="cuda").normal_(generator=g).mul_(0.7)
    k *= _gains(g, hkv, d)
    return k.to(dtype), _normal(g, dtype, pool, bs, hkv, d)


def _bounds(k):
    return torch.stack((k.amin(1), k.amax(1)), 2).contiguous()


def _tables(g, room, bs, extra=0):
    """Block tables with room for `room[b]` tokens in row b, scattered over a pool a little larger than that; unused entries 0."""
    need = [-(-r // bs) for r in room]
    pool = sum(need) + sum(need) // 8 + 8
    ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    mask = torch.arange(max(need) + extra, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    tables = torch.zeros(len(need), max(need) + extra, dtype=torch.int32, device="cuda")
    tables[mask] = ids[: sum(need)]
    return tables, pool


def _projection(g, dtype, rows, cols, heads):
    """q, k, v as views of one projection's output."""
    hq, hkv, d, _ = heads
    x = _normal(g, dtype, rows, cols, (hq + 2 * hkv) * d)
    q, k, v = x.split((hq * d, hkv * d, hkv * d), -1)
    return q.unflatten(-1, (hq, d)), k.unflatten(-1, (hkv, d)), v.unflatten(-1, (hkv, d))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, heads, dtype, held = case["kind"], _heads(case), DTYPES[case["dtype"]], DTYPES[case["cache"]]
    hq, hkv, d, bs = heads
    if kind == "append":
        rows = _chunks(case)
        tables, pool = _tables(g, [n + c for n, c in rows], bs, extra=3)
        k, v = _pages(g, pool, heads, held)
        state = {"case": case, "tables": tables, "k": k, "v": v, "bounds": _bounds(k), "most": max(n for n, _ in rows)}
        half = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
        state["freq"] = (BASE ** (-2.0 * half / max(1, case["rot"]))).float()
        if case["tokens"] == case["rows"]:
            q, nk, nv = _projection(g, dtype, len(rows), 1, heads)
            return dict(state, q=q, new_k=nk, new_v=nv, pos=_int([[c] for _, c in rows]), owners=None, qsl=None)
        q, nk, nv = _projection(g, dtype, 1, case["tokens"] + case["pad"], heads)
        pos = [c + i for n, c in rows for i in range(n)] + [0] * case["pad"]
        owners = [r for r, (n, _) in enumerate(rows) for _ in range(n)] + [0] * case["pad"]
        cuts = [0]
        for n, _ in rows:
            cuts.append(cuts[-1] + n)
        return dict(state, q=q, new_k=nk, new_v=nv, pos=_int([pos]), owners=_int([owners]), qsl=_int(cuts))
    lens = _spread(case["lo"], case["hi"], case["rows"])
    lens = [lens[i] for i in torch.randperm(len(lens), generator=g, device="cuda").cpu().tolist()]
    tables, pool = _tables(g, lens + [1] * case["empty"], bs)
    lens = lens + [0] * case["empty"]  # a batch padded to its bucket
    rows, wide, budget = len(lens), case["wide"], case["budget"]
    state = {"case": case, "tables": tables, "lens": _int(lens)}
    state["pos"] = _int([[max(0, x - wide + t) for t in range(wide)] for x in lens]) if wide > 1 or kind == "step" else None
    state["q"] = _normal(g, dtype, rows, wide, hq, d) if wide > 1 or kind == "step" else _normal(g, dtype, rows, hq, d)
    if kind == "select":
        middle = torch.empty(pool, hkv, d, device="cuda").normal_(generator=g).mul_(0.7)
        reach = [torch.empty(pool, hkv, d, device="cuda").normal_(generator=g).mul_(0.4).add_(1.7).abs_() for _ in range(2)]
        gains = _gains(g, hkv, d)
        return dict(state, bounds=torch.stack(((middle - reach[0]) * gains, (middle + reach[1]) * gains), 2).to(held).contiguous())
    k, v = _pages(g, pool, heads, held)
    if kind == "step":
        _, nk, nv = _projection(g, held, rows, 1, heads)
        state.update(k=k[None], v=v[None], bounds=_bounds(k)[None], new_k=nk.contiguous(), new_v=nv.contiguous())
        if own:
            from nano_vllm_jax_b200 import backends, kv_cache
            state["backend"] = backends.B200Backend()
            state["store"] = kv_cache.SelectiveKVCacheStorage(state["k"], state["v"], state["bounds"], budget, FIRST, LAST)
        return state
    # a selection: the blocks at the ends and others at random, in ascending order, -1 behind them
    seen = torch.tensor(lens, device="cuda")[:, None] - wide + 1 + torch.arange(wide, device="cuda")[None]
    blocks = ((seen + bs - 1) // bs).clamp(min=0)[:, :, None, None]
    column = torch.arange(tables.shape[1], device="cuda")
    liking = torch.rand(rows, wide, hkv, tables.shape[1], generator=g, device="cuda")
    liking = torch.where((column < FIRST) | (column >= blocks - LAST), 2.0, liking).masked_fill(column >= blocks, -1.0)
    top = liking.topk(min(budget, tables.shape[1]), -1)
    chosen = top.indices.masked_fill(top.values < 0, 1 << 30).sort(-1).values
    chosen = torch.nn.functional.pad(chosen, (0, budget - chosen.shape[-1]), value=1 << 30)
    chosen = chosen.masked_fill(chosen == 1 << 30, -1).to(torch.int32)
    return dict(state, k=k, v=v, chosen=chosen if wide > 1 else chosen[:, 0].contiguous())


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state, kind)
    return {"append": _plain_append, "select": _plain_select, "attend": _plain_attend, "step": _plain_step}[kind](state)


_module = None


def _own(s, kind):
    global _module
    if _module is None:
        from nano_vllm_jax_b200.kernels import selective_kv
        _module = selective_kv
    case = s["case"]
    hq, hkv, d, bs = _heads(case)
    if kind == "append":
        q = _module.rope_kv_append(s["q"], s["new_k"], s["new_v"], s["k"], s["v"], s["pos"], s["tables"], s["freq"], k_bounds=s["bounds"],
                                   query_start_loc=s["qsl"], token_row_ids=s["owners"], interleaved=case["pairs"])
        return q, s["k"], s["v"], s["bounds"]
    if kind == "select":
        return _module.select_blocks(s["q"], s["bounds"], s["tables"], s["lens"], bs, case["budget"], positions=s["pos"], first=FIRST, last=LAST)
    if kind == "attend":
        return _module.paged_decode_attention_selected(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["chosen"], d ** -0.5, positions=s["pos"])
    backend = s["backend"]
    metadata = backend.build_attention_metadata(s["pos"], s["tables"], s["lens"], bs, False)
    _, out = backend.write_kv_and_attention(0, s["q"], s["new_k"], s["new_v"], s["store"], metadata, bs, d ** -0.5, hq // hkv, False)
    return out, s["k"], s["v"], s["bounds"]


def _rotate(x, angle, pairs):
    """x [.., heads, d] fp32 turned by angle [.., rot / 2] in 64 bits."""
    n = angle.shape[-1]
    c, s = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    if pairs:
        a, b = x[..., 0: 2 * n: 2], x[..., 1: 2 * n: 2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n: 2 * n]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _into_blocks(new_k, new_v, k, v, bounds, start, count, first_token, tables, most):
    """Rows of new tokens [tokens, hkv, d], `count` each from position `start` and token `first_token` on, into their blocks."""
    bs = k.shape[1]
    columns = (most + bs - 2) // bs + 1  # blocks that a row's new tokens may touch
    column = start[:, None] // bs + torch.arange(columns, device=k.device)[None]
    place = column[:, :, None] * bs + torch.arange(bs, device=k.device)  # positions of those blocks' tokens [rows, columns, bs]
    fresh = (place >= start[:, None, None]) & (place < (start + count)[:, None, None])
    touched = fresh.any(-1)
    where = tables.gather(1, column.clamp(max=tables.shape[1] - 1))[touched]
    source = (first_token[:, None, None] + place - start[:, None, None]).clamp(0, new_k.shape[0] - 1)[touched]
    fresh, begun = fresh[touched], fresh[touched][:, 0]
    stored = new_k.to(k.dtype)[source]
    mask = fresh[..., None, None]
    k[where] = torch.where(mask, stored, k[where])
    v[where] = torch.where(mask, new_v.to(v.dtype)[source], v[where])
    low = torch.where(mask, stored, math.inf).amin(1)
    high = torch.where(mask, stored, -math.inf).amax(1)
    old, begun = bounds[where], begun[:, None, None]
    low = torch.where(begun, low, torch.minimum(low, old[:, :, 0]))
    high = torch.where(begun, high, torch.maximum(high, old[:, :, 1]))
    bounds[where] = torch.stack((low, high), 2)


def _plain_append(s):
    case, pos = s["case"], s["pos"].long()
    angle = pos.double()[..., None] * s["freq"].double()
    q = _rotate(s["q"].float(), angle, case["pairs"]).to(s["q"].dtype)
    new_k = _rotate(s["new_k"].float(), angle, case["pairs"]).flatten(0, 1)
    flat = pos.flatten()
    if s["qsl"] is None:
        first_token, count = torch.arange(flat.numel(), device=flat.device), torch.ones_like(flat)
    else:
        first_token, count = s["qsl"].long()[:-1], s["qsl"].long().diff()
    _into_blocks(new_k, s["new_v"].flatten(0, 1), s["k"], s["v"], s["bounds"], flat[first_token], count, first_token, s["tables"].long(), s["most"])
    return q, s["k"], s["v"], s["bounds"]


def _seen(s):
    """Keys that each token sees [rows, wide]."""
    lens = s["lens"].long()
    if s["pos"] is None:
        return lens[:, None]
    return torch.minimum(lens[:, None], s["pos"].long() + 1).clamp(min=0)


def _select(q, bounds, tables, seen, bs, budget):
    """q [rows, wide, hq, d] -> columns [rows, wide, hkv, budget]; scores in 64 bits, so that the border is where it belongs."""
    rows, wide, hq, d = q.shape
    hkv, width = bounds.shape[1], tables.shape[1]
    blocks = ((seen + bs - 1) // bs)[:, :, None, None]
    column = torch.arange(width, device=q.device)
    rank = torch.empty(rows, wide, hkv, width, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 28) // (width * hkv * d * 2))
    for lo in range(0, rows, step):
        held = bounds[tables[lo: lo + step]].double()  # [some, width, hkv, 2, d]
        some = held.shape[0]
        x = q[lo: lo + step].double().view(some, wide, hkv, hq // hkv, d).transpose(1, 2).flatten(2, 3)  # [some, hkv, wide * group, d]
        low, high = held[:, :, :, 0].permute(0, 2, 3, 1), held[:, :, :, 1].permute(0, 2, 3, 1)
        score = torch.matmul(x.clamp(min=0), high) + torch.matmul(x.clamp(max=0), low)
        rank[lo: lo + step] = score.view(some, hkv, wide, hq // hkv, width).amax(3).transpose(1, 2)
    rank = rank.masked_fill(rank.isnan(), math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    ends = (column < FIRST) | (column >= blocks - LAST)
    kind = torch.where(column >= blocks, 0, torch.where(ends, 2, 1)).expand_as(rank)
    order = order.gather(-1, kind.gather(-1, order).sort(dim=-1, descending=True, stable=True).indices)[..., :budget]
    order = order.masked_fill(order >= blocks, 1 << 30).sort(-1).values
    order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]), value=1 << 30)
    return order.masked_fill(order == 1 << 30, -1).to(torch.int32)


def _plain_select(s):
    case = s["case"]
    q = s["q"] if s["q"].ndim == 4 else s["q"][:, None]
    chosen = _select(q, s["bounds"], s["tables"].long(), _seen(s), _heads(case)[3], case["budget"])
    return chosen if s["q"].ndim == 4 else chosen[:, 0]


def _attend(q, k, v, tables, seen, chosen):
    """softmax(q k^T / sqrt(d)) v for q [rows, wide, hq, d] over the blocks `chosen` [rows, wide, hkv, n]."""
    rows, wide, hq, d = q.shape
    bs, hkv = k.shape[1:3]
    n = chosen.shape[-1]
    out = torch.empty(rows, wide, hq, d, dtype=torch.float32, device=q.device)
    head = torch.arange(hkv, device=q.device)[None, None, :, None]
    step = max(1, (1 << 28) // (wide * hkv * n * bs * d))
    for lo in range(0, rows, step):
        pick = chosen[lo: lo + step].long()
        some = pick.shape[0]
        ids = tables[lo: lo + step][:, None, None].expand(some, wide, hkv, -1).gather(-1, pick.clamp(min=0))
        keys = k[ids, :, head].float().flatten(3, 4)  # [some, wide, hkv, n * bs, d]
        values = v[ids, :, head].float().flatten(3, 4)
        place = (pick[..., None] * bs + torch.arange(bs, device=q.device)).flatten(-2)
        live = (place >= 0) & (pick >= 0).repeat_interleave(bs, -1) & (place < seen[lo: lo + step][:, :, None, None])
        values = torch.where(live[..., None], values, 0.0)
        x = q[lo: lo + step].float().view(some, wide, hkv, hq // hkv, d)
        score = torch.matmul(x, keys.transpose(-1, -2)).mul_(d ** -0.5).masked_fill_(~live[:, :, :, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        weight = score.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
        total = weight.sum(-1, keepdim=True)
        out[lo: lo + step] = (torch.matmul(weight, values) / torch.where(total > 0, total, 1.0)).view(some, wide, hq, d)
    return out


def _plain_attend(s):
    q, chosen = (s["q"], s["chosen"]) if s["q"].ndim == 4 else (s["q"][:, None], s["chosen"][:, None])
    out = _attend(q, s["k"], s["v"], s["tables"].long(), _seen(s), chosen)
    return out.flatten(2, 3) if s["q"].ndim == 4 else out[:, 0]


def _plain_step(s):
    case, tables = s["case"], s["tables"].long()
    bs = _heads(case)[3]
    k, v, bounds = s["k"][0], s["v"][0], s["bounds"][0]
    live = (s["lens"] > 0).nonzero()[:, 0]
    _into_blocks(s["new_k"][live, 0], s["new_v"][live, 0], k, v, bounds, s["pos"].long()[live, 0], torch.ones_like(live),
                 torch.arange(live.numel(), device=live.device), tables[live], 1)
    chosen = _select(s["q"], bounds, tables, _seen(s), bs, case["budget"])
    out = _attend(s["q"], k, v, tables, _seen(s), chosen)
    return out.flatten(2, 3), s["k"], s["v"], s["bounds"]


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d, bs = _heads(case)
    if case["kind"] == "append":
        return _exact_append(case, s)
    lens, tables = s["lens"].tolist(), s["tables"].long()
    wide = case["wide"]
    limits = s["pos"].tolist() if s["pos"] is not None else [[n - 1] for n in lens]
    q = s["q"].double().view(len(lens), wide, hq, d)
    if case["kind"] == "step":
        k, v, bounds = s["k"][0].double(), s["v"][0].double(), s["bounds"][0].double()
        for b, n in enumerate(lens):
            if n > 0:
                _exact_token(k, v, bounds, tables[b], n - 1, s["new_k"][b, 0].double(), s["new_v"][b, 0].double(), bs)
    if case["kind"] == "select":
        bounds = s["bounds"].double()
        out = torch.full((len(lens), wide, hkv, case["budget"]), -1, dtype=torch.int32, device=q.device)
    else:
        out = torch.zeros(len(lens), wide, hq, d, dtype=torch.float64, device=q.device)
    if case["kind"] == "attend":
        k, v, chosen = s["k"], s["v"], s["chosen"].view(len(lens), wide, hkv, -1)
    group = hq // hkv
    for b, n in enumerate(lens):
        for t in range(wide):
            visible = min(n, limits[b][t] + 1)
            if visible <= 0:
                continue
            for h in range(hkv):
                x = q[b, t, h * group: (h + 1) * group]
                if case["kind"] != "attend":
                    pick = _exact_choice(x, bounds, tables[b], -(-visible // bs), h, case["budget"])
                    if case["kind"] == "select":
                        out[b, t, h, : len(pick)] = pick.to(torch.int32)
                        continue
                else:
                    pick = chosen[b, t, h]
                    pick = pick[pick >= 0].long()
                out[b, t, h * group: (h + 1) * group] = _exact_attention(x, k, v, tables[b], pick, visible, h, bs)
    if case["kind"] == "select":
        return out if s["q"].ndim == 4 else out[:, 0]
    if case["kind"] == "attend":
        return out.reshape(len(lens), wide, hq * d) if s["q"].ndim == 4 else out[:, 0]
    return out.reshape(len(lens), wide, hq * d), k[None], v[None], bounds[None]


def _exact_choice(x, bounds, table, n, h, budget):
    if n <= budget:
        return torch.arange(n, device=x.device)
    held = bounds[table[:n], h]  # [n, 2, d]
    score = torch.stack([torch.maximum(row * held[:, 0], row * held[:, 1]).sum(-1) for row in x]).amax(0)
    score[:FIRST] = math.inf
    score[n - LAST:] = math.inf
    return score.sort(dim=-1, descending=True, stable=True).indices[:budget].sort().values


def _exact_attention(x, k, v, table, pick, visible, h, bs):
    place = (pick[:, None] * bs + torch.arange(bs, device=x.device)).flatten()
    live = place < visible
    keys = k[table[pick], :, h].double().flatten(0, 1)[live]
    values = v[table[pick], :, h].double().flatten(0, 1)[live]
    return torch.softmax(x @ keys.T / math.sqrt(x.shape[-1]), -1) @ values


def _exact_token(k, v, bounds, table, p, new_k, new_v, bs):
    block, at = int(table[p // bs]), p % bs
    k[block, at], v[block, at] = new_k, new_v
    bounds[block, :, 0] = new_k if at == 0 else torch.minimum(bounds[block, :, 0], new_k)
    bounds[block, :, 1] = new_k if at == 0 else torch.maximum(bounds[block, :, 1], new_k)


def _exact_append(case, s):
    hq, hkv, d, bs = _heads(case)
    half = case["rot"] // 2
    angle = s["pos"].flatten().double()[:, None] * s["freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]  # a pair as one complex number, turned

    def rotated(x):
        x = x.double().flatten(0, 1)
        out = x.clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["pairs"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(x[..., first], x[..., second]) * turn
        out[..., first], out[..., second] = z.real, z.imag
        return out

    q, nk, nv = rotated(s["q"]), rotated(s["new_k"]), s["new_v"].double().flatten(0, 1)
    k, v, bounds, tables = s["k"].double(), s["v"].double(), s["bounds"].double(), s["tables"].tolist()
    at = 0
    for b, (n, c) in enumerate(_chunks(case)):
        p = c
        while p < c + n:
            end = min((p // bs + 1) * bs, c + n)
            block, o = tables[b][p // bs], p % bs
            keys = nk[at + p - c: at + end - c]
            k[block, o: o + end - p], v[block, o: o + end - p] = keys, nv[at + p - c: at + end - c]
            low, high = keys.amin(0), keys.amax(0)
            if o > 0:
                low, high = torch.minimum(low, bounds[block, :, 0]), torch.maximum(high, bounds[block, :, 1])
            bounds[block, :, 0], bounds[block, :, 1] = low, high
            p = end
        at += n
    return q.view(s["q"].shape), k, v, bounds
