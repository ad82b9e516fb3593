"""Wrappers of the kernels for attention over selected blocks of the paged cache: torch CUDA tensors in, C-ABI calls out.

One layer of the cache is K and V in bfloat16, float16 or float32 `[num_pages, page_size, num_kv_heads, head_dim]`, head_dim a multiple
of 8 up to 256, and beside them the bounds of every page's keys in the same type `[num_pages, num_kv_heads, 2, head_dim]`: the smallest number of
each dimension in front of the largest.  `rope_kv_append` keeps them, rotating queries and keys by their positions on the way;
`select_blocks` takes for every query token the pages whose keys may score highest by them; `paged_decode_attention_selected` reads those
alone.  What the selection leaves out is left out of the softmax: the result is that of the whole row where `budget` covers it, and else an
approximation by its likeliest part.

The functions stand beside those of `paged_kv` and keep their conventions: caches are updated in place, attention is float32, launches
go to the current stream of the tensors' device, nothing synchronises (unless `NVJ_CHECK_STATUS=1` asks for the device status word after
each call), and there is no CPU path.  The reference (nanovllm_jax/kv_cache.py:852-998) reads every key of a row.
"""

from __future__ import annotations

import torch

from .. import _lib
from .._lib import check
from . import paged_kv as _k
from .quantized_kv import _ints, _on, _rows

MOST_COLUMNS = 45056  # block-table columns that a selection takes (nvj_select_blocks)
MOST_BUDGET = 2 ** 31 - 1
MOST_BLOCK_SIZE = 65536


def selective_cache_supported(dtype, head_dim: int) -> bool:
    """Whether the kernels take a cache of this type and head dimension with bounds beside it."""
    return dtype in _k._DTYPES and 8 <= head_dim <= 256 and head_dim % 8 == 0


def check_budget(budget: int, first: int, last: int) -> None:
    """A budget of blocks, the first and last ones of a row among them."""
    if budget < 1 or first < 0 or last < 0 or first + last > budget or budget > MOST_BUDGET:
        raise ValueError(f"budget must be positive, at most {MOST_BUDGET}, and hold the first and last blocks, not {budget} with {first} and {last}")


def _pages(name, t, like=None):
    _k._cuda(name, t)
    if t.ndim != 4 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and have the NHD shape [num_pages, page_size, num_kv_heads, head_dim]")
    if not selective_cache_supported(t.dtype, t.shape[3]) or t.shape[2] < 1 or t.shape[1] < 1:
        raise ValueError(f"{name} must be bfloat16, float16 or float32 with a head_dim that is a multiple of 8 up to 256, not {t.dtype} "
                         f"{tuple(t.shape)}")
    if t.data_ptr() & 15:
        raise ValueError("cache layers must start on a 16-byte boundary")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError("k_cache and v_cache must have one shape, dtype and device")
    return t


def _bounds(t, device):
    """Bounds [pages, hkv, 2, d] of a layer, checked."""
    _k._cuda("k_bounds", t)
    if t.ndim != 4 or t.shape[2] != 2 or t.shape[1] < 1 or not t.is_contiguous() or not selective_cache_supported(t.dtype, t.shape[3]):
        raise ValueError("k_bounds must be contiguous [num_pages, num_kv_heads, 2, head_dim] in bfloat16, float16 or float32, head_dim a "
                         f"multiple of 8 up to 256, not {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError("k_bounds must be on the device of the other operands")
    if t.data_ptr() & 15:
        raise ValueError("k_bounds must start on a 16-byte boundary")
    return t


def _strided(name, t, device, heads):
    """Rows of activations [rows, cols, heads, d] as the append reads them: (tensor, token stride, head stride)."""
    _k._cuda(name, t)
    if t.dtype not in _k._DTYPES:
        raise ValueError(f"unsupported {name} dtype {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on the device of k_cache")
    rows, cols, _, d = t.shape
    token = t.stride(1) if cols > 1 else (t.stride(0) if rows > 1 else heads * d)
    head = t.stride(2) if heads > 1 else d
    even = rows == 1 or cols == 1 or t.stride(0) == t.stride(1) * cols
    unit = 16 // t.element_size()
    if not even or (d > 1 and t.stride(3) != 1) or token % unit or head % unit or token < 0 or head < 0 or t.data_ptr() & 15:
        t = t.contiguous()
        t = t.clone() if t.data_ptr() & 15 else t
        token, head = heads * d, d
    return t, token, head


def rope_kv_append(query, k, v, k_cache_layer, v_cache_layer, positions, block_table, inv_freq, *, k_bounds=None, query_start_loc=None,
                   token_row_ids=None, seq_lens=None, interleaved=False):
    """Append new rows to one layer of the cache, keys and queries rotated by their positions; returns the rotated queries.

    query `[rows, cols, Hq, D]` or None, k, v `[rows, cols, Hkv, D]` of one dtype, views of a fused projection among them, at `positions` `[rows, cols]` of the rows of
    `block_table` `[table_rows, W]`; a packed batch (rows = 1) names every token's row in `token_row_ids` `[1, cols]`.  `query_start_loc`
    says which tokens count, as in `paged_kv.kv_append_slots`; rows with `seq_lens` <= 0, where given, are left alone.  `inv_freq`
    (float32, half the rotated dimensions; None or empty: no rotation) turns the pairs (x[i], x[i + n]), or with `interleaved` (x[2i], x[2i + 1]), by
    position * inv_freq[i].  Every query token is rotated.  `k_bounds`, where given, are brought up to date.  The tokens that fall into one block stand together in the
    batch, as a row's consecutive positions do.  Caches and bounds are updated in place.
    """
    done = _k.host().rope_append(query, k, v, k_cache_layer, v_cache_layer, positions, block_table, inv_freq, k_bounds, query_start_loc,
                                 token_row_ids, seq_lens, interleaved)
    if done is not None:
        return None if query is None else done
    _pages("k_cache", k_cache_layer)
    _pages("v_cache", v_cache_layer, k_cache_layer)
    device = k_cache_layer.device
    pages, page_size, hkv, d = k_cache_layer.shape
    if not isinstance(k, torch.Tensor) or not isinstance(v, torch.Tensor) or k.ndim != 4 or k.shape != v.shape or tuple(k.shape[2:]) != (hkv, d):
        raise ValueError("k and v must have one shape [rows, cols, num_kv_heads, head_dim], the heads those of the cache")
    rows, cols = k.shape[:2]
    if k.dtype != v.dtype or (query is not None and query.dtype != k.dtype):
        raise ValueError("query, k and v must have the same dtype")
    hq = 0
    if query is not None:
        if query.ndim != 4 or tuple(query.shape[:2]) != (rows, cols) or query.shape[3] != d or query.shape[2] < 1:
            raise ValueError("query must have shape [rows, cols, num_q_heads, head_dim], rows, cols and head_dim those of k")
        hq = query.shape[2]
    if k_bounds is not None:
        _bounds(k_bounds, device)
        if tuple(k_bounds.shape) != (pages, hkv, 2, d) or k_bounds.dtype != k_cache_layer.dtype:
            raise ValueError("k_bounds must be [num_pages, num_kv_heads, 2, head_dim] of the cache's dtype")
    rotary = 0
    if inv_freq is not None:
        _k._cuda("inv_freq", inv_freq)
        if inv_freq.dtype != torch.float32 or inv_freq.ndim != 1 or inv_freq.device != device or 2 * inv_freq.numel() > d:
            raise ValueError("inv_freq must be float32 of rank 1, of at most head_dim / 2 entries, on the device of k_cache")
        inv_freq = inv_freq.contiguous()
        rotary = 2 * inv_freq.numel()
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
    out = None if query is None else torch.empty((rows, cols, hq, d), dtype=query.dtype, device=device)
    if rows * cols == 0:
        return out
    if block_table.numel() == 0 or pages == 0:
        raise ValueError("an append needs a block table and a pool that are not empty")
    if out is not None and _k._poison():
        out.fill_(float("nan"))
    q, q_token, q_head = (None, 0, 0) if query is None else _strided("query", query, device, hq)
    k, k_token, k_head = _strided("k", k, device, hkv)
    v, v_token, v_head = _strided("v", v, device, hkv)
    with _on(device):
        st = _k._status_word(device)
        check(_lib.load().nvj_rope_kv_append(
            _k._ptr(q), q_token, q_head, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, _k._dt(k), _k._ptr(inv_freq), rotary,
            1 if interleaved else 0, positions.data_ptr(), block_table.data_ptr(), _k._ptr(ids), block_table.shape[0], block_table.shape[1],
            _k._ptr(qsl), qsl_rows, _k._ptr(lens), rows, cols, k_cache_layer.data_ptr(), v_cache_layer.data_ptr(), _k._ptr(k_bounds),
            _k._dt(k_cache_layer), pages, page_size, hq, hkv, d, _k._ptr(out), st.data_ptr(), _k._stream(device)), "nvj_rope_kv_append")
        if _k._strict():
            _k._check_word(st, "nvj_rope_kv_append")
    return out


def _tokens(q, hkv, d):
    """(batch, width, query heads) of q [batch, Hq, D] or [batch, tokens, Hq, D]."""
    if not isinstance(q, torch.Tensor) or q.ndim not in (3, 4):
        raise ValueError("q must have shape [batch, num_q_heads, head_dim] or [batch, tokens, num_q_heads, head_dim]")
    if q.shape[-1] != d:
        raise ValueError("q and cache head_dim must match")
    if q.shape[-2] == 0 or q.shape[-2] % hkv != 0:
        raise ValueError("num_q_heads must be divisible by num_kv_heads")
    return q.shape[0], (q.shape[1] if q.ndim == 4 else 1), q.shape[-2]


def _batch(block_table, seq_lens, positions, batch, width, device):
    block_table, seq_lens = _ints("block_table", block_table, device), _ints("seq_lens", seq_lens, device)
    if block_table.ndim != 2 or block_table.shape[0] != batch:
        raise ValueError("block_table must be a 2D tensor [batch, max_blocks_per_seq]")
    if tuple(seq_lens.shape) != (batch,):
        raise ValueError("seq_lens must have shape [batch]")
    if positions is not None:
        positions = _ints("positions", positions, device)
        if positions.numel() != batch * width:
            raise ValueError("positions must have shape [batch, tokens]")
    return block_table, seq_lens, positions


def select_blocks(q, k_bounds, block_table, seq_lens, block_size, budget, *, positions=None, first=1, last=1):
    """The blocks that each query token is to read: int32 columns of its row of `block_table`, ascending, -1 behind them.

    q `[B, Hq, D]` -> `[B, Hkv, budget]`, or `[B, T, Hq, D]` -> `[B, T, Hkv, budget]`.  Token t of row b sees the keys p < seq_lens[b] and, with
    `positions` `[B, T]`, p <= positions[b, t].  Of the blocks that hold them the `first` first and the `last` last are taken, and of the others those whose
    `sum(max(q, 0) * high + min(q, 0) * low)`, the largest of the kv head's query heads, is highest (ties: the lowest column), an upper bound of
    their keys' scores under a positive scale.  Scores rank as sums in 64 bits; one that is not a number ranks as infinity, and a block outside the pool
    (flagged) behind all others.
    """
    out = _k.host().select_blocks(q, k_bounds, block_table, seq_lens, block_size, budget, positions, first, last)
    if out is not None:
        return out
    if not isinstance(q, torch.Tensor):
        raise ValueError("q must be a CUDA tensor (there is no CPU path)")
    device = q.device
    k_bounds = _bounds(k_bounds, device)
    pages, hkv, _, d = k_bounds.shape
    batch, width, hq = _tokens(q, hkv, d)
    q = _rows("q", q, device)
    budget, first, last, block_size = int(budget), int(first), int(last), int(block_size)
    check_budget(budget, first, last)
    if not 1 <= block_size <= MOST_BLOCK_SIZE:
        raise ValueError(f"block_size must be positive and at most {MOST_BLOCK_SIZE}, not {block_size}")
    block_table, seq_lens, positions = _batch(block_table, seq_lens, positions, batch, width, device)
    if block_table.shape[1] > MOST_COLUMNS:
        raise ValueError(f"a selection takes block tables of up to {MOST_COLUMNS} columns, not {block_table.shape[1]}")
    out = torch.empty((batch, hkv, budget) if q.ndim == 3 else (batch, width, hkv, budget), dtype=torch.int32, device=device)
    if out.numel() == 0:
        return out
    if _k._poison():
        out.fill_(1 << 30)
    with _on(device):
        st = _k._status_word(device)
        check(_lib.load().nvj_select_blocks(
            q.data_ptr(), _k._dt(q), k_bounds.data_ptr(), _k._dt(k_bounds), pages, block_size, hkv, d, hq, block_table.data_ptr(),
            block_table.shape[1], seq_lens.data_ptr(), _k._ptr(positions), batch, width, budget, first, last, out.data_ptr(), st.data_ptr(),
            _k._stream(device)), "nvj_select_blocks")
        if _k._strict():
            _k._check_word(st, "nvj_select_blocks")
    return out


def paged_decode_attention_selected(q, k_cache_layer, v_cache_layer, block_table, seq_lens, selected, scale, *, positions=None):
    """Decode attention over the blocks that `selected` lists (int32 columns of the row's block table, as `select_blocks` gives them).

    q `[B, Hq, D]` with selected `[B, Hkv, n]` -> float32 `[B, Hq, D]`, or `[B, T, Hq, D]` with `[B, T, Hkv, n]` -> `[B, T, Hq * D]`.  Token t of row b sees, of
    the listed blocks' keys, those with p < seq_lens[b] and, with `positions` `[B, T]`, p <= positions[b, t]; one that sees none gives zeros.  Entries
    below 0 and blocks that the token does not see add nothing; a block that is listed twice counts twice.  Keys that it sees are finite numbers: another makes the
    outputs that it reaches infinite or NaN.
    """
    out = _k.host().selected_decode(q, k_cache_layer, v_cache_layer, block_table, seq_lens, selected, scale, positions)
    if out is not None:
        return out
    _pages("k_cache", k_cache_layer)
    _pages("v_cache", v_cache_layer, k_cache_layer)
    device = k_cache_layer.device
    pages, page_size, hkv, d = k_cache_layer.shape
    batch, width, hq = _tokens(q, hkv, d)
    q = _rows("q", q, device)
    block_table, seq_lens, positions = _batch(block_table, seq_lens, positions, batch, width, device)
    selected = _ints("selected", selected, device)
    if tuple(selected.shape[:-1]) != ((batch, hkv) if q.ndim == 3 else (batch, width, hkv)):
        raise ValueError("selected must have shape [batch, num_kv_heads, n] or [batch, tokens, num_kv_heads, n], as q has tokens or not")
    out = torch.empty((batch, hq, d) if q.ndim == 3 else (batch, width, hq * d), dtype=torch.float32, device=device)
    if out.numel() == 0:
        return out
    if _k._poison():
        out.fill_(float("nan"))
    with _on(device):
        st = _k._status_word(device)
        check(_lib.load().nvj_paged_decode_selected(
            q.data_ptr(), _k._dt(q), k_cache_layer.data_ptr(), v_cache_layer.data_ptr(), _k._dt(k_cache_layer), pages, page_size, hkv, d, hq,
            block_table.data_ptr(), block_table.shape[1], seq_lens.data_ptr(), _k._ptr(positions), selected.data_ptr(), selected.shape[-1],
            batch, width, float(scale), out.data_ptr(), st.data_ptr(), _k._stream(device)), "nvj_paged_decode_selected")
        if _k._strict():
            _k._check_word(st, "nvj_paged_decode_selected")
    return out
