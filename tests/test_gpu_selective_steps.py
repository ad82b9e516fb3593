"""Append, selection and attention together, as a serving program runs them: through the backend, from a graph, on several streams."""

import numpy as np
import pytest
import torch

import selective_reference as R
from nano_vllm_jax_b200 import kv_cache as kvc
from nano_vllm_jax_b200.backends import B200Backend
from nano_vllm_jax_b200.kernels import paged_kv as K
from nano_vllm_jax_b200.kernels import selective_kv as S

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HKV, GROUPS, D, BS = 2, 4, 256, 16
SCALE = D ** -0.5


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _f64(t):
    return t.double().cpu().numpy()


def _tokens(g, n, dtype=BF16):
    return [torch.randn(n, 1, h, D, generator=g, device="cuda").to(dtype) for h in (HKV * GROUPS, HKV, HKV)]


def _backend(budget, first=1, last=2, layers=2, blocks=400, dtype=BF16):
    class Config:
        full_attention_selected_blocks = budget
        full_attention_selected_first = first
        full_attention_selected_last = last
    backend = B200Backend(Config())
    cache = backend.allocate_kv_cache(kvc.KVCacheSpec(layers, blocks, BS, HKV, D, dtype), 8, 64)
    return backend, cache


def _prefill(backend, cache, layer, tables, lens, g, dtype=BF16):
    """The first tokens of every row, packed, through the backend."""
    n = int(sum(lens))
    q, k, v = (torch.randn(1, n, h, D, generator=g, device="cuda").to(dtype) for h in (HKV * GROUPS, HKV, HKV))
    pos = np.concatenate([np.arange(x) for x in lens])[None]
    ids = np.concatenate([np.full(x, r) for r, x in enumerate(lens)])[None]
    md = backend.build_attention_metadata(_i32(pos), _i32(tables), _i32(lens), BS, True, query_start_loc=_i32(np.concatenate([[0], np.cumsum(lens)])),
                                          token_row_ids=_i32(ids), query_lens_host=list(lens))
    cache, out = backend.write_kv_and_attention(layer, q, k, v, cache, md, BS, SCALE, GROUPS, True)
    plain = B200Backend().attention(layer, q, kvc.KVCacheStorage(cache.k_cache, cache.v_cache), md, BS, SCALE, GROUPS, True)
    assert torch.equal(out, plain)  # a prefill reads every key, as over any cache
    return cache


def _check_bounds(cache, layer, tables, lens):
    k, _, b = cache.layer(layer)
    for r, n in enumerate(lens):
        for c in range(-(-n // BS)):
            held = k[tables[r, c], : min(BS, n - c * BS)]
            assert torch.equal(b[tables[r, c]], torch.stack((held.amin(0), held.amax(0)), 1))


def _expected(q, cache, layer, tables, lens, positions, budget, first, last):
    """Selection and attention in 64 bits over what the cache holds."""
    k, v, b = (_f64(t) for t in cache.layer(layer))
    chosen = R.select(_f64(q), b, tables, lens, positions, BS, budget, first, last)
    return chosen, R.attend(_f64(q), k, v, tables, lens, positions, chosen, SCALE, BS, gamma=3 * D * 2.0 ** -23, weight_bits=16)


@pytest.mark.parametrize("dtype", [BF16, F32, F16])
def test_prefill_and_decode_steps_through_the_backend(dtype):
    budget, first, last = 7, 1, 2
    backend, cache = _backend(budget, first, last, dtype=dtype)
    g, rng = torch.Generator(device="cuda").manual_seed(1), np.random.default_rng(1)
    lens = np.array([250, 17, 1, 96, 130])
    tables = rng.permutation(400)[: 5 * 20].reshape(5, 20)
    for layer in range(2):
        cache = _prefill(backend, cache, layer, tables, lens, g, dtype)
        _check_bounds(cache, layer, tables, lens)
    for step in range(20):  # past the end of a block in every row
        lens = lens + 1
        md = backend.build_attention_metadata(_i32(lens[:, None] - 1), _i32(tables), _i32(lens), BS, False)
        for layer in range(2):
            q, k, v = _tokens(g, 5, dtype)
            cache, out = backend.write_kv_and_attention(layer, q, k, v, cache, md, BS, SCALE, GROUPS, False)
            assert type(cache) is kvc.SelectiveKVCacheStorage
            if step % 5 == 0:
                _, (want, tol) = _expected(q, cache, layer, tables, lens, lens[:, None] - 1, budget, first, last)
                assert (np.abs(_f64(out).reshape(want.shape) - want) <= tol).all()
    for layer in range(2):
        _check_bounds(cache, layer, tables, lens)


def test_verification_of_several_tokens_and_padded_rows():
    budget = 6
    backend, cache = _backend(budget, layers=1)
    g, rng = torch.Generator(device="cuda").manual_seed(2), np.random.default_rng(2)
    lens = np.array([200, 33, 150])
    tables = rng.permutation(400)[: 4 * 16].reshape(4, 16)
    cache = _prefill(backend, cache, 0, tables[:3], lens, g)
    lens = np.concatenate([lens + 4, [0]])  # the last row is padding
    pos = np.maximum(lens[:, None] - 4 + np.arange(4), 0)
    q, k, v = (torch.randn(4, 4, h, D, generator=g, device="cuda").to(BF16) for h in (HKV * GROUPS, HKV, HKV))
    md = backend.build_attention_metadata(_i32(pos), _i32(tables), _i32(lens), BS, False, query_start_loc=_i32([0, 4, 8, 12, 16]))
    before = cache.k_cache[0, tables[3, 0]].clone()
    cache, out = backend.write_kv_and_attention(0, q, k, v, cache, md, BS, SCALE, GROUPS, False)
    _check_bounds(cache, 0, tables, lens)
    assert torch.equal(cache.k_cache[0, tables[3, 0]], before)
    _, (want, tol) = _expected(q, cache, 0, tables, lens, pos, budget, 1, 2)
    assert (np.abs(_f64(out).reshape(want.shape) - want) <= tol).all() and not out[3].any()


def test_a_budget_that_covers_the_row_gives_full_attention():
    g, rng = torch.Generator(device="cuda").manual_seed(3), np.random.default_rng(3)
    lens = np.array([250, 17, 96])
    tables = rng.permutation(400)[: 3 * 20].reshape(3, 20)
    outs = []
    for budget in (16, 20, 100):  # as many as the longest row's blocks, as the tables' columns, more
        backend, cache = _backend(budget, layers=1)
        g.manual_seed(3)
        cache = _prefill(backend, cache, 0, tables, lens - 1, g)
        q, k, v = _tokens(g, 3)
        md = backend.build_attention_metadata(_i32(lens[:, None] - 1), _i32(tables), _i32(lens), BS, False)
        cache, out = backend.write_kv_and_attention(0, q, k, v, cache, md, BS, SCALE, GROUPS, False)
        _check_bounds(cache, 0, tables, lens)
        outs.append(_f64(out))
    chosen, (want, tol) = _expected(q, cache, 0, tables, lens, lens[:, None] - 1, 16, 1, 2)
    for out in outs:
        assert (np.abs(out.reshape(want.shape) - want) <= tol).all()


def test_the_backend_refuses_what_a_selection_cannot_serve():
    backend, cache = _backend(4, layers=1)
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = _tokens(g, 1)
    md = backend.build_attention_metadata(_i32([[99]]), _i32(np.arange(8)[None]), _i32([100]), BS, False)
    with pytest.raises(ValueError, match="positive scale"):
        backend.attention(0, q, cache, md, BS, -1.0, GROUPS, False)
    with pytest.raises(ValueError, match="do not agree"):
        backend.attention(0, q, cache, md, 32, SCALE, GROUPS, False)
    md.positions = None
    with pytest.raises(ValueError, match="positions"):
        backend.write_kv(0, k, v, cache, md)


def test_block_copies_take_the_bounds_along():
    backend, cache = _backend(4)
    cache.k_cache.normal_(), cache.v_cache.normal_(), cache.k_bounds.normal_()
    before = [t.clone() for t in (cache.k_cache, cache.v_cache, cache.k_bounds)]
    src, dst = _i32([3, 7, 11]), _i32([399, 0, 50])
    cache.copy_blocks(src, dst)
    for t, old in zip((cache.k_cache, cache.v_cache, cache.k_bounds), before):
        want = old.clone()
        want[:, dst.long()] = old[:, src.long()]
        assert torch.equal(t, want)


def test_block_copies_flag_and_skip_blocks_outside_the_pool(monkeypatch):
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")
    backend, cache = _backend(4)
    cache.k_cache.normal_(), cache.v_cache.normal_(), cache.k_bounds.normal_()
    blocks = cache.k_cache.shape[1]
    before = [t.clone() for t in (cache.k_cache, cache.v_cache, cache.k_bounds)]
    cache.copy_blocks(_i32([3, blocks, 5, -1]), _i32([9, 10, blocks + 7, 12]))
    with pytest.raises(K.DeviceStatusError, match="outside the pool"):
        K.check_device_status()
    for t, old in zip((cache.k_cache, cache.v_cache, cache.k_bounds), before):
        old[:, 9] = old[:, 3]
        assert torch.equal(t, old)


def _rotated_step(g, state, q, k, v, pos, lens, freq, budget, layer=0):
    kc, vc, b = state
    turned = S.rope_kv_append(q, k, v, kc, vc, pos, g, freq, k_bounds=b, seq_lens=lens)
    chosen = S.select_blocks(turned, b, g, lens, BS, budget, positions=pos)
    return turned, chosen, S.paged_decode_attention_selected(turned, kc, vc, g, lens, chosen, SCALE, positions=pos)


def _rotated_setup(seed, rows, blocks=300):
    g, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    kc, vc = (torch.randn(blocks, BS, HKV, D, generator=g, device="cuda").to(BF16) for _ in range(2))
    b = torch.stack((kc.amin(1), kc.amax(1)), 2).contiguous()
    tables = rng.permutation(blocks)[: rows * 24].reshape(rows, 24)
    freq = torch.from_numpy((1e7 ** (-np.arange(32) / 32)).astype(np.float32)).cuda()
    return g, (kc, vc, b), tables, freq


def test_rotation_selection_and_attention_replayed_from_a_graph():
    """Captured once, replayed with other queries, positions and lengths: every replay equals the calls made one by one."""
    rows, budget = 6, 8
    g, state, tables, freq = _rotated_setup(5, rows)
    twin = [t.clone() for t in state]
    q, k, v = _tokens(g, rows)
    tab, pos, lens = _i32(tables), _i32(np.zeros((rows, 1))), _i32(np.zeros(rows))
    start = np.array([100, 15, 0, 200, 371, 16])

    def fill(step):
        g.manual_seed(step)
        for t, new in zip((q, k, v), _tokens(g, rows)):
            t.copy_(new)
        pos.copy_(_i32((start + step)[:, None]))
        lens.copy_(_i32(start + step + 1))
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    strict = __import__("os").environ
    old = strict.get("NVJ_CHECK_STATUS")
    strict["NVJ_CHECK_STATUS"] = "0"  # (reading the status back is no part of a graph)
    try:
        with torch.cuda.stream(side):
            _rotated_step(tab, state, q, k, v, pos, lens, freq, budget)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _rotated_step(tab, state, q, k, v, pos, lens, freq, budget)
        for step in range(12):
            fill(step)
            graph.replay()
            want = _rotated_step(tab, twin, q, k, v, pos, lens, freq, budget)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            for a, b in zip(state, twin):
                assert torch.equal(a, b)
    finally:
        strict["NVJ_CHECK_STATUS"] = old if old is not None else "0"
    K.check_device_status()


def test_calls_on_two_streams_do_not_disturb_each_other():
    rows, budget = 5, 9
    made = []
    for seed in (6, 7):
        g, state, tables, freq = _rotated_setup(seed, rows)
        q, k, v = _tokens(g, rows)
        lens = np.array([300, 20, 0, 384, 129])
        pos = np.maximum(lens - 1, 0)[:, None]
        made.append((state, _i32(tables), q, k, v, _i32(pos), _i32(lens), freq))
    alone = []
    for state, tab, *rest in made:
        alone.append(_rotated_step(tab, [t.clone() for t in state], *rest, budget))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(10):
        both = [[], []]
        for i, (state, tab, *rest) in enumerate(made):
            copy = [t.clone() for t in state]
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                both[i] = (_rotated_step(tab, copy, *rest, budget), copy)
        torch.cuda.synchronize()
        for (got, _), want in zip(both, alone):
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_results_do_not_change_from_run_to_run():
    g, state, tables, freq = _rotated_setup(8, 12, blocks=400)
    q, k, v = _tokens(g, 12)
    lens = np.arange(12) * 31 + 2
    args = (q, k, v, _i32(lens[:, None] - 1), _i32(lens), freq, 7)
    first = _rotated_step(_i32(tables), [t.clone() for t in state], *args)
    for _ in range(5):
        again = _rotated_step(_i32(tables), [t.clone() for t in state], *args)
        for a, b in zip(first, again):
            assert torch.equal(a, b)
