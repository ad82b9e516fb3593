"""Limits of the caches whose decode reads selected blocks that need no GPU."""

import pytest
import torch

from nano_vllm_jax_b200 import kv_cache as kvc
from nano_vllm_jax_b200.backends import B200Backend
from nano_vllm_jax_b200.engine.resident_decode import DecodeStepGraph, ResidentDecodeMetadata
from nano_vllm_jax_b200.kernels import selective_kv as S


@pytest.mark.parametrize("budget", [2 ** 31, 2 ** 32 + 4, 10 ** 12])
def test_budgets_that_a_call_cannot_hold_are_refused(budget):
    with pytest.raises(ValueError, match="at most"):
        S.check_budget(budget, 1, 1)
    S.check_budget(2 ** 31 - 1, 1, 1)


def test_tables_that_a_selection_does_not_take_are_refused_at_allocation():
    class Config:
        full_attention_selected_blocks = 12
    spec = kvc.KVCacheSpec(1, 6, 16, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="block tables of up to"):
        B200Backend(Config(), device="cpu").allocate_kv_cache(spec, 4, S.MOST_COLUMNS + 1)
    assert type(B200Backend(Config(), device="cpu").allocate_kv_cache(spec, 4, S.MOST_COLUMNS)) is kvc.SelectiveKVCacheStorage
    assert type(B200Backend(device="cpu").allocate_kv_cache(spec, 4, S.MOST_COLUMNS + 1)) is kvc.KVCacheStorage


def test_a_decode_graph_refuses_pages_with_bounds_beside_them():
    """Its append writes the pages alone: the next selection would rank by bounds of other keys."""
    spec, meta = kvc.KVCacheSpec(1, 6, 16, 2, 64, torch.bfloat16), ResidentDecodeMetadata(2, 2, 16, device="cpu")
    cache = kvc.init_selective_kv_cache(spec, 4, device="cpu")
    with pytest.raises(ValueError, match="key bounds"):
        DecodeStepGraph(meta, cache.k_cache, cache.v_cache, 0, 0.1, 4)
    plain = B200Backend(device="cpu").allocate_kv_cache(spec, 4, 4)
    assert DecodeStepGraph(meta, plain.k_cache, plain.v_cache, 0, 0.1, 4).k_cache is plain.k_cache
