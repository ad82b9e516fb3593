"""Attention over the 8-bit cache where scales, masks, tables and batches have edges, against 64-bit sums (test_gpu_quantized_kv.py has the ordinary cases)."""

import numpy as np
import pytest
import torch

import quantized_reference as R
from nano_vllm_jax_b200.kernels import paged_kv as K
from nano_vllm_jax_b200.kernels import quantized_kv as Q

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
MODEL = (8, 2, 256, 16)  # query heads, kv heads, head_dim, block size


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _f64(t):
    return t.double().cpu().numpy()


def _gpu(codes, scale):
    return torch.from_numpy(codes.copy()).cuda().view(torch.float8_e4m3fn), torch.from_numpy(scale.astype(np.float32)).cuda()


def _rows(rng, lens, shape):
    """A pool without spare blocks: tables, and [(bytes, scales)] of K and of V, values about 1."""
    _, hkv, d, bs = shape
    need = [-(-n // bs) for n in lens]
    ids, tables, at = rng.permutation(sum(need)), np.zeros((len(lens), max(need)), np.int64), 0
    for r, n in enumerate(need):
        tables[r, :n] = ids[at: at + n]
        at += n
    state = []
    for _ in range(2):
        codes = rng.integers(0, 256, (sum(need), bs, hkv, d)).astype(np.uint8)
        codes[(codes & 127) == 127] = 1
        state.append((codes, np.full((sum(need), hkv), 2.0 ** -8)))
    return tables, state


def _attend(route, q, state, tables, lens, limits, shape, scale):
    """q [rows, tokens, hq, d]; token t of row r sees keys below limits[r][t].  Routes: the decode forms 1 and 2, and "prefill"."""
    hq, hkv, d, bs = shape
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    args = (k, v, ks, vs, _i32(tables), _i32(lens))
    rows, tokens = q.shape[:2]
    if route == "prefill":
        out = Q.packed_paged_prefill_attention_quantized(q.reshape(1, rows * tokens, hq, d), *args, _i32(np.asarray(limits).reshape(1, -1) - 1),
                                                         _i32(np.arange(rows + 1) * tokens), bs, scale, hq // hkv, num_decode_rows=0)
    else:
        out = Q.paged_decode_attention_quantized(q, *args, scale, positions=_i32(np.asarray(limits) - 1), form=route)
    return _f64(out).reshape(q.shape)


TERM_BITS = {1: 22, 2: 20, "prefill": 22}  # of a route's softmax weights


def _check(out, q, state, tables, lens, limits, scale, term_bits):
    q = _f64(q)
    for r, n in enumerate(lens):
        k, v = (R.gather(codes, s, tables[r], n) for codes, s in state)
        want = R.attend(q[r], k, v, np.arange(n)[None] < np.minimum(limits[r], n)[:, None], scale)
        off = np.abs(out[r] - want).max()
        assert np.isfinite(out[r]).all() and off <= R.tolerance(q[r], k, v, scale, term_bits), (r, n, off)


# ------------------------------------------------------------------------------------------------ scales far apart

def _quiet(pattern, blocks):
    """Which of a row's blocks are the quiet ones."""
    b = np.arange(blocks)
    return {"first": b == 0, "last": b == blocks - 1, "front": b < blocks // 2, "back": b >= blocks // 2, "every other": b % 2 == 0, "all but one": b != blocks // 3}[pattern]


PATTERNS = ("first", "last", "front", "back", "every other", "all but one")
DECODES = [(MODEL, 1, BF16), ((32, 8, 128, 16), 1, F16), ((32, 8, 128, 32), 2, F32), ((24, 2, 128, 64), 1, BF16), (MODEL, 5, BF16), (MODEL, 4, F32), ((6, 6, 64, 48), 1, BF16)]


# Exponents of the V scales of a row's quiet and other blocks.  The append gives a block of zeros 2^-117, and values about 1 2^-8.  Scores are alike
# on both sides, so that the keys of the quiet blocks, which add next to nothing to the weighted sum, are half of the sum of the weights.
@pytest.mark.parametrize("quiet,loud", [(-117, -8), (-117, 30), (-100, 60), (-60, 30)])
@pytest.mark.parametrize("shape,tokens,dtype", DECODES)
@pytest.mark.parametrize("form", [1, 2])
def test_decode_over_blocks_whose_scales_lie_far_apart(form, shape, tokens, dtype, quiet, loud):
    hq, hkv, d, bs = shape
    if form == 2 and d < 128:
        pytest.skip("the tcgen05 form is for head_dim 128 and 256")
    rng = np.random.default_rng(50)
    lens = [160 + 7 * i for i in range(len(PATTERNS))] + [3000 + 11 * i for i in range(len(PATTERNS))]
    tables, state = _rows(rng, lens, shape)
    for r, n in enumerate(lens):
        blocks = -(-n // bs)
        still = _quiet(PATTERNS[r % len(PATTERNS)], blocks)
        state[1][1][tables[r, :blocks]] = np.where(still, 2.0 ** quiet, 2.0 ** loud)[:, None]
        if quiet == -117:
            state[1][0][tables[r, :blocks][still]] = 0
    state[1][1][tables[0, :10], 0] = 2.0 ** -8  # (a head of its own: nothing far apart there)
    q = torch.from_numpy(rng.standard_normal((len(lens), tokens, hq, d))).to(dtype).cuda()
    limits = np.array(lens)[:, None] - tokens + 1 + np.arange(tokens)[None]
    out = _attend(form, q, state, tables, lens, limits, shape, d ** -0.5)
    _check(out, q, state, tables, lens, limits, d ** -0.5, TERM_BITS[form])


@pytest.mark.parametrize("power", [-117, 100])
@pytest.mark.parametrize("form", [1, 2])
def test_decode_over_values_of_extreme_scales(form, power):
    hq, hkv, d, bs = MODEL
    rng = np.random.default_rng(51)
    lens = [40, 2500, 300]
    tables, state = _rows(rng, lens, MODEL)
    state[1][1][:] = 2.0 ** power
    q = torch.from_numpy(rng.standard_normal((3, 1, hq, d))).to(BF16).cuda()
    limits = np.array(lens)[:, None]
    _check(_attend(form, q, state, tables, lens, limits, MODEL, 1 / 16), q, state, tables, lens, limits, 1 / 16, TERM_BITS[form])


# A row's last block is 2^80 as loud as the others and only its last token sees it: what the other tokens see is summed as well as in a row without it.
@pytest.mark.parametrize("length", [96, 144, 1000 * 16])
@pytest.mark.parametrize("form", [1, 2])
def test_decode_of_tokens_that_do_not_see_the_loud_block(form, length):
    hq, hkv, d, bs = MODEL
    rng = np.random.default_rng(52)
    lens = [length + bs]
    tables, state = _rows(rng, lens, MODEL)
    state[1][1][:] = 2.0 ** -60
    state[1][1][tables[0, -1]] = 2.0 ** 20
    q = torch.from_numpy(rng.standard_normal((1, 3, hq, d))).to(BF16).cuda()
    limits = np.array([[length - 5, length, length + bs]])
    out = _attend(form, q, state, tables, lens, limits, MODEL, 1 / 16)
    for t, n in enumerate(limits[0]):
        _check(out[:, t: t + 1], q[:, t: t + 1], state, tables, [n], limits[:, t: t + 1], 1 / 16, TERM_BITS[form])


# (shape and query type; few rows of few tokens, whose keys clusters of CTAs share, or tokens enough for a CTA per tile)
TILES = [((32, 8, 128, 16), F16), ((16, 1, 256, 16), BF16), (MODEL, F32), ((16, 2, 64, 32), BF16), (MODEL, BF16)]  # (the last: pages and their tiles)


@pytest.mark.parametrize("quiet,loud", [(-117, -8), (-117, 30), (-100, 60), (-60, 30)])
@pytest.mark.parametrize("shape,dtype", TILES)
@pytest.mark.parametrize("tokens", [3, 130])
def test_prefill_over_blocks_whose_scales_lie_far_apart(tokens, shape, dtype, quiet, loud):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(53)
    lens = [160 + 7 * i for i in range(len(PATTERNS))] + ([3000 + 11 * i for i in range(len(PATTERNS))] if tokens < 100 else [])
    tables, state = _rows(rng, lens, shape)
    for r, n in enumerate(lens):
        blocks = -(-n // bs)
        still = _quiet(PATTERNS[r % len(PATTERNS)], blocks)
        state[1][1][tables[r, :blocks]] = np.where(still, 2.0 ** quiet, 2.0 ** loud)[:, None]
        if quiet == -117:
            state[1][0][tables[r, :blocks][still]] = 0
    state[1][1][tables[0, :160 // bs], 0] = 2.0 ** -8  # (a head of its own: nothing far apart there)
    q = torch.from_numpy(rng.standard_normal((len(lens), tokens, hq, d))).to(dtype).cuda()
    limits = np.array(lens)[:, None] - tokens + 1 + np.arange(tokens)[None]
    out = _attend("prefill", q, state, tables, lens, limits, shape, d ** -0.5)
    _check(out, q, state, tables, lens, limits, d ** -0.5, 16 if shape == MODEL and dtype == BF16 else 22)


@pytest.mark.parametrize("power", [-117, 100])
@pytest.mark.parametrize("shape,dtype", TILES[:4])
def test_prefill_over_values_of_extreme_scales(shape, dtype, power):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(54)
    lens = [40, 2500, 300]
    tables, state = _rows(rng, lens, shape)
    state[1][1][:] = 2.0 ** power
    q = torch.from_numpy(rng.standard_normal((3, 2, hq, d))).to(dtype).cuda()
    limits = np.array(lens)[:, None] - 1 + np.arange(2)[None]
    _check(_attend("prefill", q, state, tables, lens, limits, shape, d ** -0.5), q, state, tables, lens, limits, d ** -0.5, 22)


@pytest.mark.parametrize("length", [96, 144, 5000 * 16])
@pytest.mark.parametrize("shape,dtype", TILES[:3])
def test_prefill_of_tokens_that_do_not_see_the_loud_block(shape, dtype, length):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(55)
    lens = [length + bs]
    tables, state = _rows(rng, lens, shape)
    state[1][1][:] = 2.0 ** -100
    state[1][1][tables[0, -1]] = 2.0 ** 60
    q = torch.from_numpy(rng.standard_normal((1, 3, hq, d))).to(dtype).cuda()
    limits = np.array([[length - 5, length, length + bs]])
    out = _attend("prefill", q, state, tables, lens, limits, shape, d ** -0.5)
    for t, n in enumerate(limits[0]):
        _check(out[:, t: t + 1], q[:, t: t + 1], state, tables, [n], limits[:, t: t + 1], d ** -0.5, 22)


# ------------------------------------------------------------------------------------------------ masks and tables

@pytest.mark.parametrize("route,shape,dtype", [(1, MODEL, BF16), (1, (6, 6, 64, 48), F32), (2, MODEL, BF16), (2, (32, 8, 128, 32), F16)] + [("prefill", *t) for t in TILES])
def test_keys_that_no_token_of_the_row_sees_may_hold_anything(route, shape, dtype):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(56)
    lens = [200, 64, 1000, 90]
    seen = [[130, 131], [0, 0], [990, 700], [65, 64]]  # keys that a row's two tokens see
    tables, state = _rows(rng, lens, shape)
    for codes, _ in state:
        for r, limits in enumerate(seen):
            for key in range(max(limits), lens[r]):
                codes[tables[r, key // bs], key % bs] = 127
    q = torch.from_numpy(rng.standard_normal((4, 2, hq, d))).to(dtype).cuda()
    out = _attend(route, q, state, tables, lens, np.array(seen), shape, d ** -0.5)
    assert not out[1].any()
    if route != "prefill":  # (a decode row may as well name the largest position there is)
        free = _attend(route, q[3:], state, tables[3:], [64], np.full((1, 2), 1 << 31), shape, d ** -0.5)
        _check(free, q[3:], state, tables[3:], [64], np.full((1, 2), 64), d ** -0.5, TERM_BITS[route])
    _check(out, q, state, tables, [max(s) for s in seen], np.array(seen), d ** -0.5, 16 if route == "prefill" and shape == MODEL and dtype == BF16 else TERM_BITS[route])


@pytest.mark.parametrize("route,shape,dtype", [(1, MODEL, BF16), (2, MODEL, BF16)] + [("prefill", *t) for t in TILES])
def test_blocks_outside_the_pool_reach_nothing(route, shape, dtype, monkeypatch):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(57)
    lens = [200, 2000, 70, bs]
    tables, state = _rows(rng, lens, shape)
    q = torch.from_numpy(rng.standard_normal((4, 3, hq, d))).to(dtype).cuda()
    limits = np.array(lens)[:, None] - 2 + np.arange(3)[None]
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")
    broken = tables.copy()
    pool = len(state[0][0])
    broken[0, 0], broken[0, 100 // bs], broken[1, 1000 // bs], broken[1, 1984 // bs], broken[3, 0] = pool, -1, 1 << 30, pool, -(1 << 31)
    out = _attend(route, q, state, broken, lens, limits, shape, d ** -0.5)
    with pytest.raises(K.DeviceStatusError, match="device status 2 "):
        K.check_device_status()
    q = _f64(q)
    for r, n in enumerate(lens):
        good = np.repeat(broken[r, : -(-n // bs)] == tables[r, : -(-n // bs)], bs)[:n]
        k, v = (R.gather(codes, s, tables[r], n) for codes, s in state)
        want = R.attend(q[r], k, v, (np.arange(n)[None] < limits[r][:, None]) & good[None], d ** -0.5)
        term_bits = 16 if route == "prefill" and shape == MODEL and dtype == BF16 else TERM_BITS[route]
        assert np.abs(out[r] - want).max() <= R.tolerance(q[r], k, v, d ** -0.5, term_bits), r


# ------------------------------------------------------------------------------------------------ packed batches

def _packed(rng, rows, shape, dtype):
    """Rows [(new, cached)] in a bucket without padding, as the call takes them, and what to check them with."""
    hq, hkv, d, bs = shape
    lens = [n + c for n, c in rows]
    tables, state = _rows(rng, lens, shape)
    total = sum(n for n, _ in rows)
    q = torch.from_numpy(rng.standard_normal((1, total, hq, d))).to(dtype).cuda()
    positions, qsl = np.concatenate([np.arange(c, c + n) for n, c in rows])[None], np.cumsum([0] + [n for n, _ in rows])
    return q, tables, state, lens, positions, qsl


@pytest.mark.parametrize("shape,dtype,cached", [((16, 2, 64, 32), F16, 60), (MODEL, BF16, 30), (MODEL, BF16, 2000), ((32, 8, 128, 16), F32, 900)])
def test_rows_without_tokens_behind_a_full_bucket(shape, dtype, cached):
    # (the batch is padded to its rows, not to its tokens: query_start_loc of the last rows is the bucket)
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(58)
    rows = [(1, cached + i) for i in range(40)] + [(0, 5)] + [(3, cached)] + [(1, 7)] + [(0, cached)] * 85
    q, tables, state, lens, positions, qsl = _packed(rng, rows, shape, dtype)
    around = _i32(np.concatenate([np.full(4, 1 << 30), positions[0], np.full(4, 1 << 30)]))  # nobody's numbers on either side
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    tokens = positions.shape[1]
    out = _f64(Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), around[4: 4 + tokens][None], _i32(qsl), bs, d ** -0.5,
                                                          hq // hkv)).reshape(tokens, hq, d)
    for r, (n, c) in enumerate(rows):
        at = slice(qsl[r], qsl[r + 1])
        if n:
            _check(out[None, at], q[:, at], state, tables[r: r + 1], [lens[r]], [c + 1 + np.arange(n)], d ** -0.5, 16 if shape == MODEL and n > 1 else 20)


# A bucket that is too small for its rows, as a layout that was flagged hands it on: tokens beyond it are neither read nor written.  The arrays of the
# call lie inside larger ones, so that the test sees what lands behind them.
def _too_small(call, q, positions, qsl, bucket, out_shape):
    (tokens, hq, d) = q.shape
    out = torch.full((tokens, hq, d), 7.0, device="cuda")
    call(q[:bucket][None], _i32(positions)[:bucket][None], _i32(qsl), out[:bucket])
    torch.cuda.synchronize()
    assert bool((out[bucket:] == 7.0).all())
    return _f64(out[:bucket])


@pytest.mark.parametrize("shape,dtype,cached", [((16, 2, 64, 32), F16, 60), (MODEL, BF16, 30), (MODEL, BF16, 2000), ((32, 8, 128, 16), F32, 900)])
@pytest.mark.parametrize("rows,bucket", [([(1, 1)] * 30, 20), ([(1, 1)] * 9 + [(70, 3)] + [(1, 1)] * 9, 50), ([(200, 0), (1, 5), (1, 5)], 200), ([(5, 9)] * 7, 8)])
def test_tokens_beyond_the_bucket_are_left_out(shape, dtype, cached, rows, bucket):
    from nano_vllm_jax_b200 import _lib
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(59)
    rows = [(n, c * cached) for n, c in rows]
    q, tables, state, lens, positions, qsl = _packed(rng, rows, shape, dtype)
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    t, l, lib = _i32(tables), _i32(lens), _lib.load()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(q, positions, qsl, out):
        args = (K._dt(q), len(rows), tables.shape[1], bs, hkv, d, hq, d ** -0.5, -1, bucket, -1)
        scratch = torch.empty(lib.nvj_paged_prefill_quantized_workspace_bytes(*args), dtype=torch.uint8, device="cuda")
        _lib.check(lib.nvj_paged_prefill_quantized(
            q.data_ptr(), K._dt(q), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k.shape[0], bs, hkv, d, hq, t.data_ptr(), tables.shape[1],
            l.data_ptr(), positions.data_ptr(), qsl.data_ptr(), len(rows), bucket, d ** -0.5, out.data_ptr(), status.data_ptr(), scratch.data_ptr(),
            scratch.numel(), -1, -1, torch.cuda.current_stream().cuda_stream), "prefill")

    out = _too_small(call, q[0], positions[0], qsl, bucket, q.shape[1:])
    for r, (n, c) in enumerate(rows):
        at = slice(min(qsl[r], bucket), min(qsl[r + 1], bucket))
        if at.stop > at.start:
            _check(out[None, at], q[:, at], state, tables[r: r + 1], [lens[r]], [c + 1 + np.arange(at.stop - at.start)], d ** -0.5, 16 if shape == MODEL else 20)


@pytest.mark.parametrize("cached", [30, 3000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_beyond_the_bucket_of_a_bf16_cache_are_left_out(dtype, cached):
    from nano_vllm_jax_b200 import _lib
    hq, hkv, d, bs = MODEL
    rng = np.random.default_rng(60)
    lib = _lib.load()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for rows, bucket in (([(1, cached)] * 30, 20), ([(1, cached)] * 9 + [(70, 3)] + [(1, cached)] * 9, 50), ([(1, cached)] * 300, 280)):
        lens = [n + c for n, c in rows]
        width = -(-max(lens) // bs)
        tables = rng.integers(0, 200, (len(rows), width))  # (rows share blocks)
        k, v = (torch.from_numpy(rng.standard_normal((200, bs, hkv, d))).to(BF16).cuda() for _ in range(2))
        total = sum(n for n, _ in rows)
        q = torch.from_numpy(rng.standard_normal((total, hq, d))).to(dtype).cuda()
        positions, qsl = np.concatenate([np.arange(c, c + n) for n, c in rows]), np.cumsum([0] + [n for n, _ in rows])
        t, l = _i32(tables), _i32(lens)
        scratch = K._workspace(q.device, len(rows)).buf

        def call(q, positions, qsl, out):
            _lib.check(lib.nvj_paged_prefill_packed(
                q.data_ptr(), K._dt(q), k.data_ptr(), v.data_ptr(), K._dt(k), k.shape[0], bs, hkv, d, hq, t.data_ptr(), width, l.data_ptr(), positions.data_ptr(),
                qsl.data_ptr(), len(rows), bucket, d ** -0.5, out.data_ptr(), status.data_ptr(), scratch.data_ptr(), scratch.numel(), 0,
                torch.cuda.current_stream().cuda_stream), "prefill")

        out = _too_small(call, q, positions, qsl, bucket, q.shape[1:])
        kk, vv = _f64(k), _f64(v)
        for r in sorted({0, 3, len(rows) // 2, len(rows) - 1}):
            n, c = rows[r]
            at = slice(min(qsl[r], bucket), min(qsl[r + 1], bucket))
            if at.stop > at.start:
                x, y = (a[tables[r]].reshape(-1, hkv, d)[:lens[r]] for a in (kk, vv))
                seen = np.arange(lens[r])[None] < c + 1 + np.arange(at.stop - at.start)[:, None]
                want = R.attend(_f64(q[at]), x, y, seen, d ** -0.5)
                assert np.abs(out[at] - want).max() <= R.tolerance(_f64(q[at]), x, y, d ** -0.5, 8), r  # (weights rounded to bf16)


def test_a_cache_without_heads_is_refused():
    k = torch.zeros(4, 16, 0, 256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.ones(4, 0, device="cuda")
    q, tables, lens = torch.zeros(2, 8, 256, device="cuda"), _i32([[0, 1], [2, 3]]), _i32([3, 4])
    for call in (lambda: Q.paged_decode_attention_quantized(q, k, k, s, s, tables, lens, 1.0),
                 lambda: Q.packed_paged_prefill_attention_quantized(q[None], k, k, s, s, tables, lens, _i32([[0, 1]]), _i32([0, 1, 2]), 16, 1.0, 4),
                 lambda: Q.kv_append_quantized(q[:, None, :0], q[:, None, :0], k, k, s, s, _i32([[0], [0]]), tables)):
        with pytest.raises(ValueError, match="kv head"):
            call()


# One number of a query 2^power times the others, and keys that are small there, so that the others decide: they keep their bits.
@pytest.mark.parametrize("route,tokens,power", [(1, 1, 14), (2, 1, 8), (2, 1, 14), (2, 2, 14), (1, 5, 12), (2, 5, 8), (2, 5, 12), ("prefill", 3, 14)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_queries_with_one_large_number(route, tokens, power, dtype):
    hq, hkv, d, bs = MODEL
    rng = np.random.default_rng(61)
    lens = [300, 2100]
    tables, state = _rows(rng, lens, MODEL)
    state[0][0][..., 7] &= 0x87  # (2^-6 at most, times the scale)
    down = 64.0 if dtype == F16 else 1.0  # (f16 ends at 65504)
    q = rng.standard_normal((2, tokens, hq, d)) / down
    q[..., 7] *= 2.0 ** power
    q = torch.from_numpy(q).to(dtype).cuda()
    limits = np.array(lens)[:, None] - tokens + 1 + np.arange(tokens)[None]
    out = _attend(route, q, state, tables, lens, limits, MODEL, down / 16)
    _check(out, q, state, tables, lens, limits, down / 16, 16 if route == "prefill" and dtype == BF16 else TERM_BITS[route])
