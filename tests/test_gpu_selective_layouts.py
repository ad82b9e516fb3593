"""Selective caches at other layouts than the model's, with tables wider than the rows, and in mixed batches."""

import numpy as np
import pytest
import torch

import selective_reference as R
from nano_vllm_jax_b200 import kv_cache as kvc
from nano_vllm_jax_b200.backends import B200Backend
from nano_vllm_jax_b200.kernels import selective_kv as S
from test_gpu_selective_kv import BF16, F16, F32, MODEL, _f64, _gen, _i32, _normal, _tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [700, 4096, 16384])
def test_tables_far_wider_than_the_rows(width):
    """Padded tables, -1 behind a row's blocks: the selection and the attention of the tight ones."""
    for layout, types in ((MODEL, (BF16, BF16)), ((6, 3, 96, 16), (F32, F32)), ((32, 8, 128, 32), (F16, F16))):
        hq, hkv, d, bs = layout
        g, rng = _gen(24), np.random.default_rng(24)
        lens = [60 * bs, 3, 37 * bs + 1, 0]
        tight, pool = _tables(rng, [max(n, 1) for n in lens], bs)
        wide = np.full((4, width), -1)
        for b, n in enumerate(lens):
            wide[b, : -(-n // bs)] = tight[b, : -(-n // bs)]
        k, v = _normal(g, types[1], pool, bs, hkv, d), _normal(g, types[1], pool, bs, hkv, d)
        bounds = torch.stack((k.amin(1), k.amax(1)), 2).contiguous()
        q = _normal(g, types[0], 4, hq, d)
        made = []
        for table in (tight, wide):
            chosen = S.select_blocks(q, bounds, _i32(table), _i32(lens), bs, 9)
            made.append((chosen, S.paged_decode_attention_selected(q, k, v, _i32(table), _i32(lens), chosen, d ** -0.5)))
        for a, b in zip(*made):
            assert torch.equal(a, b)


class _Config:
    full_attention_selected_blocks = 5
    full_attention_selected_first = 1
    full_attention_selected_last = 2


def _bounds_hold(cache, layer, tables, lens):
    k, _, b = cache.layer(layer)
    bs = k.shape[1]
    for r, n in enumerate(lens):
        for c in range(-(-n // bs)):
            held = k[tables[r, c], : min(bs, n - c * bs)]
            assert torch.equal(b[tables[r, c]], torch.stack((held.amin(0), held.amax(0)), 1))


@pytest.mark.parametrize("layout,dtype", [((32, 8, 128, 32), F16), ((6, 3, 96, 16), BF16), ((4, 4, 64, 48), F32), ((16, 1, 40, 7), BF16), ((34, 2, 64, 16), BF16)], ids=str)
@pytest.mark.parametrize("width", [1, 3])
@pytest.mark.parametrize("columns", [0, 300], ids=["tight tables", "wide tables"])
def test_backend_steps_at_other_layouts(layout, dtype, width, columns):
    """A rectangular prefill, then decode steps of one or several tokens, a padded row among them; the second layer of two."""
    hq, hkv, d, bs = layout
    backend = B200Backend(_Config())
    cache = backend.allocate_kv_cache(kvc.KVCacheSpec(2, 120, bs, hkv, d, dtype), 4, 64)
    g, rng = _gen(28), np.random.default_rng(28)
    first = 9 * bs + 3
    lens = np.array([first, first, first])
    tables = np.full((4, max(columns, 14)), -1)
    tables[:, :14] = rng.permutation(120)[: 4 * 14].reshape(4, 14)
    scale, layer = d ** -0.5, 1
    q, k, v = (_normal(g, dtype, 3, first, h, d) for h in (hq, hkv, hkv))
    md = backend.build_attention_metadata(_i32(np.tile(np.arange(first), (3, 1))), _i32(tables[:3]), _i32(lens), bs, True,
                                          query_start_loc=_i32(np.arange(4) * first))
    cache = backend.write_kv(layer, k, v, cache, md)
    _bounds_hold(cache, layer, tables, lens)
    for step in range(4):
        lens = lens + width
        pos = np.concatenate([lens[:, None] - width + np.arange(width), np.zeros((1, width), np.int64)])
        every = np.concatenate([lens, [0]])
        q, k, v = (_normal(g, dtype, 4, width, h, d) for h in (hq, hkv, hkv))
        md = backend.build_attention_metadata(_i32(pos), _i32(tables), _i32(every), bs, False, query_start_loc=_i32(np.arange(5) * width))
        cache, out = backend.write_kv_and_attention(layer, q, k, v, cache, md, bs, scale, hq // hkv, False)
        kk, vv, b = (_f64(t) for t in cache.layer(layer))
        chosen = R.select(_f64(q), b, np.maximum(tables, 0), every, pos, bs, 5, 1, 2)
        want, tol = R.attend(_f64(q), kk, vv, np.maximum(tables, 0), every, pos, chosen, scale, bs, gamma=3 * d * 2.0 ** -23, weight_bits=16)
        assert (np.abs(_f64(out).reshape(want.shape) - want) <= tol).all() and not out[3].any()
    _bounds_hold(cache, layer, tables, lens)
    assert not cache.k_cache[0].any() and not cache.k_bounds[0].any()


def test_decode_rows_of_a_mixed_batch_read_every_key():
    """A packed step of decode rows and a prompt's chunk: bounds are kept, and every row's attention is that of a cache without a selection."""
    hq, hkv, d, bs = MODEL
    backend, plain = B200Backend(_Config()), B200Backend()
    cache = backend.allocate_kv_cache(kvc.KVCacheSpec(1, 120, bs, hkv, d, BF16), 4, 64)
    g, rng = _gen(29), np.random.default_rng(29)
    tables = rng.permutation(120)[: 3 * 30].reshape(3, 30)
    cached, new = np.array([300, 0, 17]), np.array([1, 150, 1])
    for step, (c, n) in enumerate(((np.zeros(3, int), cached), (cached, new))):
        q, k, v = (_normal(g, BF16, 1, int(n.sum()), h, d) for h in (hq, hkv, hkv))
        pos = np.concatenate([np.arange(a, a + b) for a, b in zip(c, n)])[None]
        ids = np.repeat(np.arange(3), n)[None]
        md = backend.build_attention_metadata(_i32(pos), _i32(tables), _i32(c + n), bs, True, query_start_loc=_i32(np.concatenate([[0], np.cumsum(n)])),
                                              token_row_ids=_i32(ids), query_lens_host=list(n))
        cache, out = backend.write_kv_and_attention(0, q, k, v, cache, md, bs, d ** -0.5, hq // hkv, True)
    assert type(cache) is kvc.SelectiveKVCacheStorage
    assert torch.equal(out, plain.attention(0, q, kvc.KVCacheStorage(cache.k_cache, cache.v_cache), md, bs, d ** -0.5, hq // hkv, True))
    _bounds_hold(cache, 0, tables, cached + new)


def test_the_backend_step_replayed_from_a_graph(monkeypatch):
    """Captured once, replayed with other tokens, positions and lengths: as a twin's steps made one by one."""
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")  # (reading the status back is no part of a graph)
    hq, hkv, d, bs = 6, 3, 96, 16
    rows, backend, g = 5, B200Backend(_Config()), _gen(30)
    caches = [backend.allocate_kv_cache(kvc.KVCacheSpec(1, 200, bs, hkv, d, BF16), rows, 40) for _ in range(2)]
    for t in (caches[0].k_cache, caches[0].v_cache):
        t.copy_(_normal(g, BF16, *t.shape))
    caches[0].k_bounds.copy_(torch.stack((caches[0].k_cache.amin(2), caches[0].k_cache.amax(2)), 3))
    for a, b in zip((caches[1].k_cache, caches[1].v_cache, caches[1].k_bounds), (caches[0].k_cache, caches[0].v_cache, caches[0].k_bounds)):
        a.copy_(b)
    q, k, v = (_normal(g, BF16, rows, 1, h, d) for h in (hq, hkv, hkv))
    tables, pos, lens = _i32(np.arange(200).reshape(rows, 40)), _i32(np.zeros((rows, 1))), _i32(np.zeros(rows))
    start = np.array([100, 15, 0, 600, 320])

    def fill(step):
        for t in (q, k, v):
            t.copy_(_normal(g, BF16, *t.shape))
        pos.copy_(_i32((start + step)[:, None]))
        lens.copy_(_i32(start + step + 1))

    def run(cache):
        md = backend.build_attention_metadata(pos, tables, lens, bs, False)
        return backend.write_kv_and_attention(0, q, k, v, cache, md, bs, d ** -0.5, hq // hkv, False)[1]
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for cache in caches:  # (the twin's bounds widen by this step's keys too)
            run(cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(caches[0])
    for step in range(20):
        fill(step)
        graph.replay()
        assert torch.equal(out, run(caches[1]))
    for a, b in zip((caches[0].k_cache, caches[0].v_cache, caches[0].k_bounds), (caches[1].k_cache, caches[1].v_cache, caches[1].k_bounds)):
        assert torch.equal(a, b)
