"""Decode through the backend with budgets of blocks that no row has."""

import numpy as np
import pytest
import torch

from nano_vllm_jax_b200 import kv_cache as kvc
from nano_vllm_jax_b200.backends import B200Backend
from test_gpu_selective_kv import BF16, MODEL, _gen, _i32, _normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("step", [True, False], ids=["step", "write_kv and attention"])
def test_a_budget_beyond_the_tables_reads_every_block(step):
    """Up to 2^31 - 1, which a row's list of that length would not hold: as a budget of the tables' columns."""
    hq, hkv, d, bs = MODEL
    rows, columns = 12, 20
    outs = []
    for budget in (columns, columns + 1, 10 ** 6, 2 ** 31 - 1):
        class Config:
            full_attention_selected_blocks = budget
            full_attention_selected_last = 2
        backend, g = B200Backend(Config()), _gen(31)
        cache = backend.allocate_kv_cache(kvc.KVCacheSpec(1, rows * columns, bs, hkv, d, BF16), rows, columns)
        for t in (cache.k_cache, cache.v_cache):
            t.copy_(_normal(g, BF16, *t.shape))
        cache.k_bounds.copy_(torch.stack((cache.k_cache.amin(2), cache.k_cache.amax(2)), 3))
        q, k, v = (_normal(g, BF16, rows, 1, h, d) for h in (hq, hkv, hkv))
        lens = np.arange(rows) * 29 + 1
        lens[3] = 0
        md = backend.build_attention_metadata(_i32(np.maximum(lens - 1, 0)[:, None]), _i32(np.arange(rows * columns).reshape(rows, columns)), _i32(lens), bs, False)
        if step:
            _, out = backend.write_kv_and_attention(0, q, k, v, cache, md, bs, d ** -0.5, hq // hkv, False)
        else:
            out = backend.attention(0, q, backend.write_kv(0, k, v, cache, md), md, bs, d ** -0.5, hq // hkv, False)
        outs.append(out)
    assert outs[0][4].any() and not outs[0][3].any()
    for out in outs[1:]:
        assert torch.equal(out, outs[0])
