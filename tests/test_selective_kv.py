"""Attention over selected blocks: what can be checked without a GPU (refusals, sizes, the plain selection)."""

import ctypes

import numpy as np
import pytest
import torch

import selective_reference as R
from nano_vllm_jax_b200 import _lib
from nano_vllm_jax_b200 import kv_cache as kvc
from nano_vllm_jax_b200.backends import B200Backend
from nano_vllm_jax_b200.host_pipeline import HostDecodePipeline
from nano_vllm_jax_b200.kernels import selective_kv as S

BF16 = torch.bfloat16
INVALID, UNSUPPORTED, TOO_LARGE = -1, -2, -5


def test_wrappers_refuse_tensors_that_are_not_on_a_gpu():
    q, k, i = torch.zeros(1, 1, 2, 64), torch.zeros(2, 16, 1, 64), torch.zeros(1, 1, dtype=torch.int32)
    bounds = torch.zeros(2, 1, 2, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.rope_kv_append(q, q[:, :, :1], q[:, :, :1], k, k, i, i, None)
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.select_blocks(q, bounds, i, i[0], 16, 4)
    with pytest.raises(ValueError, match="CUDA tensor"):
        S.paged_decode_attention_selected(q, k, k, i, i[0], i.view(1, 1, 1, 1), 1.0)


@pytest.mark.parametrize("budget,first,last", [(0, 0, 0), (1, 1, 1), (4, -1, 1), (4, 1, -1), (-3, 0, 0)])
def test_budgets_that_do_not_hold_the_ends_are_refused(budget, first, last):
    with pytest.raises(ValueError, match="budget"):
        S.check_budget(budget, first, last)
    with pytest.raises(ValueError, match="budget"):
        kvc.init_selective_kv_cache(kvc.KVCacheSpec(1, 4, 16, 2, 64, BF16), budget, first, last, device="cpu")


def test_allocation_counts_the_bounds():
    spec = kvc.KVCacheSpec(3, 1000, 16, 2, 64, BF16, max_kv_cache_bytes=10 * 3 * 2 * 64 * 2 * (2 * 16 + 2))
    cache = kvc.init_selective_kv_cache(spec, 8, device="cpu")
    assert cache.k_cache.shape == cache.v_cache.shape == (3, 10, 16, 2, 64) and cache.k_bounds.shape == (3, 10, 2, 2, 64)
    assert cache.k_bounds.dtype == BF16 and (cache.budget, cache.first, cache.last) == (8, 1, 1)
    assert [tuple(t.shape) for t in cache.layer(2)] == [(10, 16, 2, 64), (10, 16, 2, 64), (10, 2, 2, 64)]
    with pytest.raises(ValueError, match="too small"):
        kvc.init_selective_kv_cache(kvc.KVCacheSpec(3, 1000, 16, 2, 64, BF16, max_kv_cache_bytes=1000), 8, device="cpu")
    for dtype, d in ((torch.float8_e4m3fn, 64), (BF16, 260), (BF16, 20), (BF16, 0)):
        with pytest.raises(ValueError, match="multiple of 8"):
            kvc.init_selective_kv_cache(kvc.KVCacheSpec(1, 4, 16, 2, d, dtype), 8, device="cpu")


def test_the_backend_allocates_what_its_configuration_says():
    class Config:
        full_attention_selected_blocks = 12
        full_attention_selected_first = 2
        full_attention_selected_last = 3
    backend = B200Backend(Config(), device="cpu")
    cache = backend.allocate_kv_cache(kvc.KVCacheSpec(2, 6, 16, 2, 64, BF16), 4, 8)
    assert type(cache) is kvc.SelectiveKVCacheStorage and (cache.budget, cache.first, cache.last) == (12, 2, 3)
    with pytest.raises(ValueError, match="multiple of 8"):
        backend.allocate_kv_cache(kvc.KVCacheSpec(2, 6, 16, 2, 64, torch.float8_e4m3fn), 4, 8)
    Config.full_attention_selected_blocks = None
    assert type(B200Backend(Config(), device="cpu").allocate_kv_cache(kvc.KVCacheSpec(2, 6, 16, 2, 64, BF16), 4, 8)) is kvc.KVCacheStorage


def test_the_host_pipeline_refuses_a_selective_cache():
    cache = kvc.init_selective_kv_cache(kvc.KVCacheSpec(1, 4, 16, 2, 64, BF16), 8, device="cpu")
    with pytest.raises(ValueError, match="selective"):
        HostDecodePipeline(B200Backend(device="cpu"), cache, 2, 4, 16, 0.1, 4)


def test_a_selective_layer_is_one_of_a_cache_of_rank_5():
    flat = torch.zeros(1, 64, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="rank 5"):
        kvc.SelectiveKVCacheStorage(flat, flat, torch.zeros(1, 4, 2, 2, 64, dtype=BF16), 4).layer(0)


def _append(lib, **change):
    a = dict(q=16, qt=64, qh=64, k=16, kt=64, kh=64, v=16, vt=64, vh=64, act=0, freq=16, rot=64, pairs=0, pos=16, tab=16, ids=None, trows=1, w=1, qsl=None,
             qslr=0, lens=None, rows=1, cols=1, kc=16, vc=16, b=16, cache=0, blocks=1, bs=16, hq=1, hkv=1, d=64, out=16, st=16, stream=None)
    a.update(change)
    return lib.nvj_rope_kv_append(*a.values())


def test_append_arguments_are_checked_before_any_launch():
    lib = _lib.load()
    assert _append(lib, cols=0) == 0
    for change in ({"rows": -1}, {"rot": 66}, {"rot": 3}, {"k": None}, {"st": None}, {"out": None}, {"freq": None}, {"blocks": 0}, {"w": 0}, {"k": 8}, {"b": 8},
                   {"kt": 4}, {"qh": 60}, {"ids": 16, "rows": 2}, {"bs": 0}, {"hkv": 0}):
        assert _append(lib, **change) == INVALID, change
    for change in ({"act": 3}, {"cache": -1}, {"d": 68}, {"d": 264}, {"hkv": 1025}):
        assert _append(lib, **change) == UNSUPPORTED, change
    assert _append(lib, rows=1 << 16, cols=1 << 16) == TOO_LARGE


def _select(lib, **change):
    a = dict(q=16, qd=0, b=16, cd=0, blocks=4, bs=16, hkv=1, d=64, hq=4, tab=16, w=8, lens=16, pos=None, rows=1, width=1, budget=4, first=1, last=1, out=16,
             st=16, stream=None)
    a.update(change)
    return lib.nvj_select_blocks(*a.values())


def test_selection_arguments_are_checked_before_any_launch():
    lib = _lib.load()
    assert _select(lib, rows=0) == 0
    for change in ({"budget": 0}, {"first": 4}, {"first": -1}, {"last": 2 ** 31 - 1}, {"hq": 0}, {"hq": 3, "hkv": 2}, {"q": None}, {"lens": None}, {"out": None},
                   {"tab": None}, {"b": 24}, {"bs": 0}, {"rows": -1}):
        assert _select(lib, **change) == INVALID, change
    for change in ({"qd": 5}, {"cd": 3}, {"d": 4}, {"d": 257}):
        assert _select(lib, **change) == UNSUPPORTED, change
    for change in ({"w": S.MOST_COLUMNS + 1}, {"w": 40000, "bs": 60000}, {"rows": 1 << 20, "width": 1 << 10}):
        assert _select(lib, **change) == TOO_LARGE, change


def _attend(lib, **change):
    a = dict(q=16, qd=0, k=16, v=16, cd=0, blocks=4, bs=16, hkv=1, d=64, hq=4, tab=16, w=8, lens=16, pos=None, sel=16, n=4, rows=1, width=1, scale=1.0, out=16,
             st=16, stream=None)
    a.update(change)
    return lib.nvj_paged_decode_selected(*a.values())


def test_attention_arguments_are_checked_before_any_launch():
    lib = _lib.load()
    assert _attend(lib, width=0) == 0
    for change in ({"hq": 0}, {"hq": 3, "hkv": 2}, {"k": None}, {"sel": None}, {"out": 8}, {"n": -1}, {"bs": 0}, {"st": None}):
        assert _attend(lib, **change) == INVALID, change
    for change in ({"qd": 5}, {"cd": 3}, {"d": 4}, {"d": 257}):
        assert _attend(lib, **change) == UNSUPPORTED, change
    for change in ({"w": 1 << 20, "bs": 1 << 12}, {"n": 1 << 20, "bs": 1 << 12}, {"rows": 1 << 20, "width": 1 << 10}):
        assert _attend(lib, **change) == TOO_LARGE, change


def test_an_upper_bound_bounds():
    rng = np.random.default_rng(0)
    q, k = rng.standard_normal((4, 32)), rng.standard_normal((50, 16, 32))
    score = R.scores(q, np.stack((k.min(1), k.max(1)), 1))
    assert (np.einsum("gd,npd->npg", q, k).max((1, 2)) <= score + 1e-12).all()
    assert list(R.choose(score * 0, 9, 5, 1, 2)) == [0, 1, 2, 7, 8] and list(R.choose(score, 3, 5, 1, 1)) == [0, 1, 2, -1, -1]


def test_the_entry_points_are_bound():
    lib = _lib.load()
    assert all(isinstance(getattr(lib, n), ctypes._CFuncPtr) for n in ("nvj_rope_kv_append", "nvj_select_blocks", "nvj_paged_decode_selected"))
