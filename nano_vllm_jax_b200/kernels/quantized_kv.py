"""Wrappers of the kernels over the paged cache held in 8 bits: torch CUDA tensors in, C-ABI calls out.

One layer of the cache is K and V as `torch.float8_e4m3fn` `[num_pages, page_size, num_kv_heads, head_dim]` and a float32 scale
per page and kv head `[num_pages, num_kv_heads]` of K and of V: a value is number * scale.  The append makes the scales, powers of
two (`nvj_kv_append_quantized` in include/nvj_b200.h says how), so that a value is rounded once.  head_dim 64, 128 or
256, page_size 16, 32, 48 or 64; queries and new rows in bfloat16, float16 or float32.

The functions stand beside those of `paged_kv` for the caches of 16 and 32 bits and keep their conventions: caches are updated in
place and returned, outputs are float32, launches go to the current stream of the tensors' device, nothing synchronises
(unless `NVJ_CHECK_STATUS=1` asks for the device status word after each call), and there is no CPU path.  The reference
(nanovllm_jax/kv_cache.py:216-271) has no 8-bit cache.
"""

from __future__ import annotations

import torch

from .. import _lib
from .._lib import check
from . import paged_kv as _k

_FP8 = torch.float8_e4m3fn
DECODE_COLUMNS = 64  # query tokens per row x query heads per kv head up to which the decode kernel is the better one for a rectangular batch
HEAD_DIMS, PAGE_SIZES = (64, 128, 256), (16, 32, 48, 64)


def quantized_cache_supported(page_size: int, head_dim: int) -> bool:
    """Whether the kernels take an 8-bit cache of this page size and head dimension."""
    return page_size in PAGE_SIZES and head_dim in HEAD_DIMS


def _cache(k, v, k_scale, v_scale):
    """Shape of a layer's cache, checked."""
    for name, t in (("k_cache", k), ("v_cache", v), ("k_scale", k_scale), ("v_scale", v_scale)):
        _k._cuda(name, t)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.device != k.device:
            raise ValueError(f"{name} must be on the device of k_cache")
    if k.dtype != _FP8 or v.dtype != _FP8:
        raise ValueError("k_cache and v_cache must have dtype float8_e4m3fn")
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError("k_cache and v_cache must have one NHD shape [num_pages, page_size, num_kv_heads, head_dim]")
    pages, page_size, hkv, d = k.shape
    if not quantized_cache_supported(page_size, d):
        raise ValueError(f"an 8-bit cache has head_dim in {HEAD_DIMS} and page_size in {PAGE_SIZES}, not {d} and {page_size}")
    if hkv < 1:
        raise ValueError("an 8-bit cache has at least one kv head")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.dtype != torch.float32 or t.shape != (pages, hkv):
            raise ValueError(f"{name} must be float32 [num_pages, num_kv_heads]")
    if (k.data_ptr() | v.data_ptr()) & 15:
        raise ValueError("cache layers must start on a 16-byte boundary")
    return pages, page_size, hkv, d


def _ints(name, t, device):
    t = _k._i32(name, t)
    if t.device != device:
        raise ValueError(f"{name} must be on the device of k_cache")
    return t


def _rows(name, t, device):
    """Activations as the kernels read them: contiguous, from a 16-byte boundary on."""
    _k._cuda(name, t)
    if t.dtype not in _k._DTYPES:
        raise ValueError(f"unsupported {name} dtype {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on the device of k_cache")
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _on(device):
    """Launches go to the tensors' device, whichever is current."""
    return torch.cuda.device(device)


def kv_append_quantized(new_k, new_v, k_cache_layer, v_cache_layer, k_scale, v_scale, positions, block_table, *,
                        query_start_loc=None, token_row_ids=None, seq_lens=None):
    """Append new rows to one layer of the 8-bit cache, in place; returns (k_cache_layer, v_cache_layer, k_scale, v_scale).

    new_k, new_v `[rows, cols, Hkv, D]` at `positions` `[rows, cols]` of the rows of `block_table` `[table_rows, W]`; a packed batch
    (rows = 1) names every token's row in `token_row_ids` `[1, cols]`.  `query_start_loc` says which tokens count, as in
    `paged_kv.kv_append_slots`; rows with `seq_lens` <= 0, where given, are left alone.  The tokens that fall into one block
    stand together in the batch, as a row's consecutive positions do.
    """
    if _k.host().quantized_append(new_k, new_v, k_cache_layer, v_cache_layer, k_scale, v_scale, positions, block_table, query_start_loc,
                                  token_row_ids, seq_lens):
        return k_cache_layer, v_cache_layer, k_scale, v_scale
    pages, page_size, hkv, d = _cache(k_cache_layer, v_cache_layer, k_scale, v_scale)
    device = k_cache_layer.device
    if new_k.ndim != 4 or new_k.shape != new_v.shape or tuple(new_k.shape[2:]) != (hkv, d):
        raise ValueError("new_k and new_v must have one shape [rows, cols, num_kv_heads, head_dim], the heads those of the cache")
    if new_k.dtype != new_v.dtype:
        raise ValueError("new_k and new_v must have the same dtype")
    rows, cols = new_k.shape[:2]
    new_k, new_v = _rows("new_k", new_k, device), _rows("new_v", new_v, device)
    positions, block_table = _ints("positions", positions, device), _ints("block_table", block_table, device)
    if tuple(positions.shape) != (rows, cols):
        raise ValueError("positions must have shape [rows, cols]")
    if block_table.ndim != 2:
        raise ValueError("block_table must be a 2D tensor [rows, max_blocks_per_seq]")
    ids, qsl, qsl_rows, lens = None, None, 0, None
    if token_row_ids is not None:
        ids = _ints("token_row_ids", token_row_ids, device)
        if rows != 1 or tuple(ids.shape) != (rows, cols):
            raise ValueError("a packed batch has one row, and token_row_ids the shape of positions")
    elif rows > block_table.shape[0]:
        raise ValueError("positions and block_table batch dimensions must match")
    if query_start_loc is not None:
        qsl = _ints("query_start_loc", query_start_loc, device)
        qsl_rows = qsl.numel() - 1
        if qsl.ndim != 1 or qsl_rows < 0:
            raise ValueError("query_start_loc must have shape [rows + 1]")
    if seq_lens is not None:
        lens = _ints("seq_lens", seq_lens, device)
        if tuple(lens.shape) != (block_table.shape[0],):
            raise ValueError("seq_lens must have shape [table rows]")
    if rows * cols == 0:
        return k_cache_layer, v_cache_layer, k_scale, v_scale
    if block_table.numel() == 0 or pages == 0:
        raise ValueError("an append needs a block table and a pool that are not empty")
    with _on(device):
        st = _k._status_word(device)
        check(_lib.load().nvj_kv_append_quantized(
            new_k.data_ptr(), new_v.data_ptr(), _k._dt(new_k), positions.data_ptr(), block_table.data_ptr(), _k._ptr(ids),
            block_table.shape[0], block_table.shape[1], _k._ptr(qsl), qsl_rows, _k._ptr(lens), rows, cols, k_cache_layer.data_ptr(),
            v_cache_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, page_size, hkv, d, st.data_ptr(),
            _k._stream(device)), "nvj_kv_append_quantized")
        if _k._strict():
            _k._check_word(st, "nvj_kv_append_quantized")
    return k_cache_layer, v_cache_layer, k_scale, v_scale


def paged_decode_attention_quantized(q, k_cache_layer, v_cache_layer, k_scale, v_scale, block_table, seq_lens, scale, *, positions=None, form=0):
    """Decode attention over one layer of the 8-bit cache, for rows of one query token or a few.

    q `[B, Hq, D]` -> float32 `[B, Hq, D]`, or `[B, T, Hq, D]` -> `[B, T, Hq * D]`.  Token t of row b sees the keys p < seq_lens[b] and,
    with `positions` `[B, T]`, p <= positions[b, t]; one that sees none gives zeros.  Keys that no token of a row sees may hold anything.  `form`: 0 automatic, 1 mma.sync tiles on
    thread-block clusters, 2 tcgen05 tiles (head_dim 128 or 256).
    """
    out = _k.host().quantized_decode(q, k_cache_layer, v_cache_layer, k_scale, v_scale, block_table, seq_lens, scale, positions, form)
    if out is not None:
        return out
    pages, page_size, hkv, d = _cache(k_cache_layer, v_cache_layer, k_scale, v_scale)
    device = k_cache_layer.device
    if q.ndim not in (3, 4):
        raise ValueError("q must have shape [batch, num_q_heads, head_dim] or [batch, tokens, num_q_heads, head_dim]")
    batch, width = q.shape[0], (q.shape[1] if q.ndim == 4 else 1)
    hq = q.shape[-2]
    if q.shape[-1] != d:
        raise ValueError("q and cache head_dim must match")
    if hq == 0 or hq % hkv != 0:
        raise ValueError("num_q_heads must be divisible by num_kv_heads")
    q = _rows("q", q, device)
    block_table, seq_lens = _ints("block_table", block_table, device), _ints("seq_lens", seq_lens, device)
    if block_table.ndim != 2 or block_table.shape[0] != batch:
        raise ValueError("block_table must be a 2D tensor [batch, max_blocks_per_seq]")
    if tuple(seq_lens.shape) != (batch,):
        raise ValueError("seq_lens must have shape [batch]")
    if positions is not None:
        positions = _ints("positions", positions, device)
        if positions.numel() != batch * width:
            raise ValueError("positions must have shape [batch, tokens]")
    out = torch.empty((batch, hq, d) if q.ndim == 3 else (batch, width, hq * d), dtype=torch.float32, device=device)
    if out.numel() == 0:
        return out
    if _k._poison():
        out.fill_(float("nan"))
    lib = _lib.load()
    with _on(device):
        nbytes = lib.nvj_paged_decode_quantized_workspace_bytes(batch, width, block_table.shape[1], page_size, hkv, d, hq, int(form))
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        st = _k._status_word(device)
        check(lib.nvj_paged_decode_quantized(
            q.data_ptr(), _k._dt(q), k_cache_layer.data_ptr(), v_cache_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages,
            page_size, hkv, d, hq, block_table.data_ptr(), block_table.shape[1], seq_lens.data_ptr(), _k._ptr(positions), None, batch,
            width, float(scale), out.data_ptr(), st.data_ptr(), _k._ptr(scratch), nbytes, int(form), _k._stream(device)),
            "nvj_paged_decode_quantized")
        if _k._strict():
            _k._check_word(st, "nvj_paged_decode_quantized")
    return out


def packed_paged_prefill_attention_quantized(query, k_cache_layer, v_cache_layer, k_scale, v_scale, block_table, kv_lens, positions,
                                             query_start_loc, block_size, scale, num_key_value_groups, *, num_decode_rows=None,
                                             query_tile_pairs=None):
    """Ragged packed prefill over one layer of the 8-bit cache: query `[1, T, Hq, D]` -> float32 `[1, T, Hq * D]`, padded tokens 0.

    Masks and the two counts (`num_decode_rows`: rows of a single query token, `query_tile_pairs`: 64-token tiles of the other
    rows) as in `paged_kv.packed_paged_prefill_attention`; tokens that `query_start_loc`
    counts beyond the bucket are left out.  bfloat16 queries of the model's shape run on the tcgen05 tiles over bf16
    pages written for the call (exact; up to 1 GiB, from torch's allocator), others on tcgen05 tiles over the 8-bit blocks.
    """
    out = _k.host().quantized_prefill(query, k_cache_layer, v_cache_layer, k_scale, v_scale, block_table, kv_lens, positions, query_start_loc,
                                      block_size, scale, num_key_value_groups, num_decode_rows, query_tile_pairs)
    if out is not None:
        return out
    pages, page_size, hkv, d = _cache(k_cache_layer, v_cache_layer, k_scale, v_scale)
    device = k_cache_layer.device
    if query.ndim != 4 or query.shape[0] != 1:
        raise ValueError("packed prefill query must have shape [1, token_bucket, heads, head_dim]")
    _, tokens, hq, dq = query.shape
    if page_size != block_size or d != dq or hq != hkv * num_key_value_groups or hq == 0:
        raise ValueError("query / cache shapes do not agree")
    if positions.ndim != 2 or tuple(positions.shape) != (1, tokens):
        raise ValueError("packed positions must have shape [1, token_bucket]")
    query = _rows("query", query, device)
    block_table, kv_lens = _ints("block_table", block_table, device), _ints("kv_lens", kv_lens, device)
    positions, qsl = _ints("positions", positions, device), _ints("query_start_loc", query_start_loc, device)
    if block_table.ndim != 2:
        raise ValueError("block_table must be a 2D tensor [batch, max_blocks_per_seq]")
    rows, width = block_table.shape
    if tuple(kv_lens.shape) != (rows,):
        raise ValueError("kv_lens shape must align with block_table rows")
    if tuple(qsl.shape) != (rows + 1,):
        raise ValueError("query_start_loc must have shape [rows + 1]")
    out = torch.empty((1, tokens, hq * d), dtype=torch.float32, device=device)
    if tokens == 0:
        return out
    if _k._poison():
        out.fill_(float("nan"))
    lib = _lib.load()
    singles = -1 if num_decode_rows is None else int(num_decode_rows)
    pairs = -1 if query_tile_pairs is None else int(query_tile_pairs)
    with _on(device):
        nbytes = lib.nvj_paged_prefill_quantized_workspace_bytes(_k._dt(query), rows, width, page_size, hkv, d, hq, float(scale), singles, tokens, pairs)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        st = _k._status_word(device)
        check(lib.nvj_paged_prefill_quantized(
            query.data_ptr(), _k._dt(query), k_cache_layer.data_ptr(), v_cache_layer.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            pages, page_size, hkv, d, hq, block_table.data_ptr(), width, kv_lens.data_ptr(), positions.data_ptr(), qsl.data_ptr(), rows,
            tokens, float(scale), out.data_ptr(), st.data_ptr(), _k._ptr(scratch), nbytes, singles, pairs, _k._stream(device)),
            "nvj_paged_prefill_quantized")
        if _k._strict():
            _k._check_word(st, "nvj_paged_prefill_quantized")
    return out
