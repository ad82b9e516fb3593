"""The 8-bit paged cache on the GPU: append bit for bit, attention against 64-bit sums, in the places where they can go wrong."""

import numpy as np
import pytest
import torch

import quantized_reference as R
from nano_vllm_jax_b200.kernels import paged_kv as K
from nano_vllm_jax_b200.kernels import quantized_kv as Q

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# query heads, kv heads, head_dim, block size
FORMS = (1, 2)  # mma.sync tiles on clusters, tcgen05 tiles
SHAPES = [(8, 2, 256, 16), (32, 8, 128, 16), (16, 2, 64, 32), (6, 6, 64, 48), (24, 2, 128, 64), (16, 1, 256, 16), (5, 1, 128, 32), (2, 2, 256, 64)]


def _f64(t):
    return t.double().cpu().numpy()


def _pool(rng, blocks, shape, spread=3):
    """Random bytes that are numbers (no NaN), and scales of many sizes."""
    _, hkv, d, bs = shape
    codes = rng.integers(0, 256, (blocks, bs, hkv, d)).astype(np.uint8)
    codes[(codes & 127) == 127] = 1
    return codes, 2.0 ** rng.integers(-8 - spread, -7 + spread, (blocks, hkv))


def _gpu(codes, scale):
    return torch.from_numpy(codes.copy()).cuda().view(torch.float8_e4m3fn), torch.from_numpy(scale.astype(np.float32)).cuda()


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _tables(rng, lens, bs, blocks, extra=1):
    need = [-(-max(int(n), 0) // bs) for n in lens]
    perm, o = rng.permutation(blocks), 0
    tables = np.zeros((len(lens), max(need + [0]) + extra), np.int32)
    for r, n in enumerate(need):
        tables[r, :n] = perm[o: o + n]
        o += n
    assert o <= blocks
    return tables


# ------------------------------------------------------------------------------------------------ append

def _append_case(shape, rows, dtype, seed, loud=1.0, packed=True, pad=3):
    """(kernel's state, reference's state) after one append of rows [(new tokens, cached tokens)]."""
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(seed)
    tables = _tables(rng, [n + c for n, c in rows], bs, 200)
    state = [_pool(rng, 200, shape), _pool(rng, 200, shape)]
    cols = sum(n for n, _ in rows) + pad if packed else max(n for n, _ in rows)
    new = [torch.from_numpy(rng.standard_normal((1 if packed else len(rows), cols, hkv, d)) * loud).to(dtype).cuda() for _ in range(2)]
    positions, ids, at = np.zeros(new[0].shape[:2], np.int32), np.zeros(new[0].shape[:2], np.int32), []
    tokens, o = [None] * positions.size, 0
    for r, (n, c) in enumerate(rows):
        for t in range(n):
            i = o + t if packed else r * cols + t
            positions.reshape(-1)[i], ids.reshape(-1)[i] = c + t, r
            tokens[i] = (int(tables[r, (c + t) // bs]), (c + t) % bs)
        o += n
    qsl = np.cumsum([0] + [n for n, _ in rows])
    gpu = [_gpu(*s) for s in state]
    Q.kv_append_quantized(*new, gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1], _i32(positions), _i32(tables), query_start_loc=_i32(qsl),
                          token_row_ids=_i32(ids) if packed else None)
    for (codes, scale), x in zip(state, new):
        R.append(codes, scale, _f64(x).reshape(-1, hkv, d), tokens, bs)
    return gpu, state


def _same(gpu, state):
    for (numbers, scale), (codes, want) in zip(gpu, state):
        assert np.array_equal(_f64(scale), want)
        got = numbers.view(torch.uint8).cpu().numpy()
        nan = (codes & 127) == 127
        assert np.array_equal((got & 127) == 127, nan) and np.array_equal(got[~nan], codes[~nan])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_append_of_ragged_rows(shape, dtype):
    rows = [(1, 0), (1, 15), (1, 16), (33, 7), (1, 63), (0, 20), (70, 64), (5, 46), (200, 3)]
    _same(*_append_case(shape, rows, dtype, 1))


@pytest.mark.parametrize("loud", [2.0 ** -30, 1e-3, 30.0, 1e4, 2.0 ** 70])
@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[3]])
def test_append_of_quiet_and_loud_rows(shape, loud):
    # quiet: blocks keep their scale and the new numbers are small or zero; loud: the blocks' old rows are rescaled, down to zero
    _same(*_append_case(shape, [(1, 3), (2, 15), (20, 9), (1, 0)], F32, 2, loud))


@pytest.mark.parametrize("rows", [[(1, c) for c in range(0, 80, 3)], [(3, 5), (1, 15), (17, 30), (0, 4)]])
@pytest.mark.parametrize("shape", SHAPES[:4])
def test_append_of_a_rectangular_batch(shape, rows):
    _same(*_append_case(shape, rows, BF16, 3, packed=False))


def test_append_of_many_tokens_in_windows():
    _same(*_append_case(SHAPES[0], [(777, 5), (1, 31), (900, 16), (300, 301)], BF16, 4, 3.0))
    _same(*_append_case(SHAPES[4], [(777, 5), (1, 31), (900, 16), (300, 301)], F32, 5, 3.0))


def test_append_keeps_nan_holds_infinities_and_zeros():
    hq, hkv, d, bs = shape = SHAPES[0]
    state = [_pool(np.random.default_rng(0), 4, shape) for _ in range(2)]
    gpu = [_gpu(*s) for s in state]
    x = torch.zeros(1, 6, hkv, d)
    x[0, 0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3.0])
    x[0, 1, 1, 5] = 3.3e38
    x[0, 2, 0, 7] = -1e-39
    x[0, 3] = float("nan")
    x[0, 3, 1, 0] = 2.0
    tokens = [(2, 0), (2, 1), (2, 2), (1, 4), (3, 15), None]  # the last block's row: zeros alone
    tables = _i32([[2], [1], [3]])
    for dtype in (F32, BF16):
        new = x.to(dtype).cuda()
        Q.kv_append_quantized(new, new, gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1], _i32([[0, 1, 2, 4, 15, 0]]), tables,
                              query_start_loc=_i32([0, 3, 4, 5]), token_row_ids=_i32([[0, 0, 0, 1, 2, 0]]))
        for codes, scale in state:
            R.append(codes, scale, _f64(new)[0], tokens, bs)
        _same(gpu, state)


def test_append_takes_a_block_s_tokens_in_any_order_and_its_first_one_begins_it():
    hq, hkv, d, bs = shape = SHAPES[4]
    rng = np.random.default_rng(6)
    state = [_pool(rng, 4, shape) for _ in range(2)]
    gpu = [_gpu(*s) for s in state]
    order = rng.permutation(64)  # a run longer than a warp
    new = torch.from_numpy(rng.standard_normal((1, 64, hkv, d))).to(F32).cuda()
    Q.kv_append_quantized(new, new, gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1], _i32(order[None]), _i32([[3]]), token_row_ids=_i32(np.zeros((1, 64))))
    for codes, scale in state:
        R.append(codes, scale, _f64(new)[0], [(3, int(o)) for o in order], bs)
    _same(gpu, state)


def test_append_twice_changes_nothing_more():
    gpu, state = _append_case(SHAPES[1], [(9, 4), (1, 40)], BF16, 7, 50.0)
    again, _ = _append_case(SHAPES[1], [(9, 4), (1, 40)], BF16, 7, 50.0)
    for a, b in zip(gpu, again):
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def test_append_skips_inactive_rows_and_flags_what_lies_outside(monkeypatch):
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(8)
    state = [_pool(rng, 6, shape) for _ in range(2)]
    new = torch.randn(5, 1, hkv, d, device="cuda")
    gpu = [_gpu(*s) for s in state]
    Q.kv_append_quantized(new, new, gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1], _i32(np.zeros((5, 1))), _i32(np.zeros((5, 1))),
                          seq_lens=_i32([0, -1, 0, 0, 0]))
    _same(gpu, state)
    for positions, table, word in (([32, -1, 0, 0, 1 << 30], np.full((5, 2), 2), 4), ([0] * 5, [[6, 0], [-1, 0], [1 << 30, 0], [9, 0], [2, 0]], 2)):
        lens = _i32([1, 1, 0, 1, 1]) if word == 2 else _i32([1, 1, 0, 0, 1])
        monkeypatch.setenv("NVJ_CHECK_STATUS", "0")
        Q.kv_append_quantized(new, new, gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1], _i32(positions)[:, None], _i32(table), seq_lens=lens)
        if word == 2:  # the last row alone is written
            for codes, scale in state:
                R.append(codes, scale, _f64(new)[:, 0], [None] * 4 + [(2, 0)], bs)
        _same(gpu, state)
        with pytest.raises(K.DeviceStatusError, match=f"device status {word} "):
            K.check_device_status()


def test_append_and_attention_take_strided_operands():
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(9)
    state = [_pool(rng, 9, shape) for _ in range(2)]
    wide = torch.from_numpy(rng.standard_normal((3, 2, 2 * hkv, d + 8))).to(BF16).cuda()
    views = [wide[:, :, :hkv, 1: d + 1], wide[:, :, hkv:, 8:]]
    gpu = [_gpu(*s) for s in state]
    Q.kv_append_quantized(*views, gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1], _i32([[3, 4], [15, 16], [0, 1]]), _i32([[1, 0, 0], [5, 6, 0], [8, 0, 0]]))
    for (codes, scale), x in zip(state, views):
        R.append(codes, scale, _f64(x).reshape(6, hkv, d), [(1, 3), (1, 4), (5, 15), (6, 0), (8, 0), (8, 1)], bs)
    _same(gpu, state)
    q = torch.randn(3, hq, d + 8, device="cuda").to(BF16)[:, :, 3: d + 3]
    out = Q.paged_decode_attention_quantized(q, gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1], _i32([[1, 0, 0], [5, 6, 0], [8, 0, 0]]),
                                             _i32([5, 17, 2]), 0.05)
    assert torch.equal(out, Q.paged_decode_attention_quantized(q.contiguous(), gpu[0][0], gpu[1][0], gpu[0][1], gpu[1][1],
                                                               _i32([[1, 0, 0], [5, 6, 0], [8, 0, 0]]), _i32([5, 17, 2]), 0.05))


# ------------------------------------------------------------------------------------------------ attention

def _poison_behind(state, tables, lens, bs):
    """NaN in every row of a used block behind the row's last key: it must reach nothing."""
    for codes, _ in state:
        for r, n in enumerate(lens):
            if n > 0 and n % bs:
                codes[tables[r, n // bs], n % bs:] = 127


def _check(out, q, state, tables, lens, limits, scale, term_bits=22):
    """out, q [rows][t, hq, d]; limits[r][t]: keys that token t of row r may see at most."""
    for r, n in enumerate(lens):
        n = max(int(n), 0)
        k, v = (R.gather(codes, s, tables[r], n) for codes, s in state)
        seen = np.arange(n)[None] < np.minimum(np.asarray(limits[r]), n)[:, None]
        want = R.attend(q[r], k, v, seen, scale)
        off = np.abs(out[r] - want).max() if want.size else 0.0
        assert np.isfinite(out[r]).all() and off <= R.tolerance(q[r], k, v, scale, term_bits), (r, n, off)


TERM_BITS = {1: 22, 2: 20}  # of a form's softmax weights


def _forms(shape):
    return FORMS if shape[2] >= 128 else (1,)


def _queries(rng, shape, dtype):
    q = torch.from_numpy(rng.standard_normal(shape)).to(dtype)
    return q.cuda(), _f64(q)


LENGTHS = [0, 1, 15, 16, 17, 31, 32, 63, 64, 65, 100, 255, 300, 0, 77, 700]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(shape, dtype):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(10)
    tables = _tables(rng, LENGTHS, bs, 200)
    state = [_pool(rng, 200, shape) for _ in range(2)]
    _poison_behind(state, tables, LENGTHS, bs)
    q, q64 = _queries(rng, (len(LENGTHS), hq, d), dtype)
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    for form in _forms(shape):
        out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(LENGTHS), d ** -0.5, form=form)
        assert out.dtype == F32 and out.shape == q.shape
        _check(_f64(out)[:, None], q64[:, None], state, tables, LENGTHS, [[n] for n in LENGTHS], d ** -0.5, TERM_BITS[form])
        # the same rows one at a time (clusters of other sizes, other ranges)
        for r in (1, 9, 15):
            one = Q.paged_decode_attention_quantized(q[r: r + 1], k, v, ks, vs, _i32(tables[r: r + 1]), _i32(LENGTHS[r: r + 1]), d ** -0.5, form=form)
            _check(_f64(one)[:, None], q64[r: r + 1, None], state, tables[r: r + 1], LENGTHS[r: r + 1], [LENGTHS[r: r + 1]], d ** -0.5, TERM_BITS[form])


@pytest.mark.parametrize("width", [2, 3, 5, 9, 17])
@pytest.mark.parametrize("shape,dtype", [(SHAPES[0], BF16), (SHAPES[1], F32), (SHAPES[2], F16), (SHAPES[6], BF16)])
def test_rows_of_several_tokens(shape, dtype, width):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(width)
    lens = [0, 1, 16, 33, 130, 64, 517]
    tables = _tables(rng, lens, bs, 100)
    state = [_pool(rng, 100, shape) for _ in range(2)]
    _poison_behind(state, tables, lens, bs)
    q, q64 = _queries(rng, (len(lens), width, hq, d), dtype)
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    limits = rng.integers(-2, 40, (len(lens), width)) + np.array(lens)[:, None] - 20  # some see nothing, some more than there is
    limits[3] = 33
    args = (q, k, v, ks, vs, _i32(tables), _i32(lens), d ** -0.5)
    for form in _forms(shape):
        out = Q.paged_decode_attention_quantized(*args, positions=_i32(limits - 1), form=form)
        assert out.shape == (len(lens), width, hq * d)
        _check(_f64(out).reshape(q64.shape), q64, state, tables, lens, limits, d ** -0.5, TERM_BITS[form])
        free = Q.paged_decode_attention_quantized(*args, form=form)
        _check(_f64(free).reshape(q64.shape), q64, state, tables, lens, [[n] * width for n in lens], d ** -0.5, TERM_BITS[form])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.07, 1.5])
def test_any_scale_of_the_scores(scale, dtype, form):
    # 1.5: scores of tens, a softmax that is nearly one-hot, maxima that move
    hq, hkv, d, bs = shape = SHAPES[1]
    rng = np.random.default_rng(11)
    lens = [40, 300, 7]
    tables = _tables(rng, lens, bs, 60)
    state = [_pool(rng, 60, shape, spread=1) for _ in range(2)]
    q, q64 = _queries(rng, (3, hq, d), dtype)
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), scale, form=form)
    _check(_f64(out)[:, None], q64[:, None], state, tables, lens, [[n] for n in lens], scale, TERM_BITS[form])


@pytest.mark.parametrize("route", [1, 2, "prefill"])
def test_blocks_of_very_different_scales(route):
    # V: one block in four 2^100 as loud, and one row of quiet blocks alone; K: the loud ones' scores are -1000s, so that the quiet blocks decide
    hq, hkv, d, bs = shape = SHAPES[1]
    rng = np.random.default_rng(12)
    lens = [160, 160, 90]
    tables = _tables(rng, lens, bs, 40)
    state = [_pool(rng, 40, shape) for _ in range(2)]
    q = np.abs(rng.standard_normal((3, hq, d)))
    state[0][0][:] &= 127  # keys of positive numbers ..
    state[0][1][:] = 2.0 ** -9
    state[1][1][:] = 2.0 ** -60
    for r in (0, 1):
        for b in range(0, 10, 4):
            state[1][1][tables[r, b]] = 2.0 ** 40
            state[0][1][tables[r, b]] = 1.0
            state[0][0][tables[r, b]] = 0x80 | 0x70  # .. but for the loud blocks'
    q[1] *= -1  # row 1: the loud blocks win
    qg = torch.from_numpy(q).to(BF16).cuda()
    q64 = _f64(qg)
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    args = (k, v, ks, vs, _i32(tables), _i32(lens))
    if route != "prefill":
        out = Q.paged_decode_attention_quantized(qg, *args, d ** -0.5, form=route)
    else:
        out = Q.packed_paged_prefill_attention_quantized(qg[None], *args, _i32([[159, 159, 89]]), _i32([0, 1, 2, 3]), bs, d ** -0.5, hq // hkv,
                                                         num_decode_rows=0)
    out = _f64(out).reshape(3, hq, d)
    for r, n in enumerate(lens):
        kk, vv = (R.gather(codes, s, tables[r], n) for codes, s in state)
        want = R.attend(q64[r: r + 1], kk, vv, np.ones((1, n), bool), d ** -0.5)[0]
        # relative to the values that the softmax is about: the quiet ones in rows 0 and 2
        loudest = np.abs(vv).max() if r == 1 else np.abs(vv[np.abs(vv).max((1, 2)) < 1]).max()
        within = R.tolerance(q64[r: r + 1], kk, vv, d ** -0.5, TERM_BITS.get(route, 22)) / np.abs(vv).max() * loudest
        assert np.abs(out[r] - want).max() <= within


@pytest.mark.parametrize("route", [1, 2, "prefill"])
def test_one_loud_key_over_many_quiet_ones(route):
    # one key's weight is 2^10 of each of the 8000 others', which together decide: they must keep their bits
    hq, hkv, d, bs = shape = SHAPES[1]
    rng = np.random.default_rng(25)
    n = 8000
    tables = rng.permutation(n // bs)[None]
    state = [_pool(rng, n // bs, shape, spread=1) for _ in range(2)]
    state[0][0][:], state[0][1][:] = 0x38, 1.0  # keys of ones; one of twos
    state[0][0][tables[0, 130], 3] = 0x40
    state[1][1][:] = 2.0 ** -8
    q = np.full((1, hq, d), 10 * np.log(2) / d * 8)
    qg = torch.from_numpy(q).to(F16).cuda()
    q64 = _f64(qg)
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    args = (k, v, ks, vs, _i32(tables), _i32([n]))
    if route == "prefill":
        out = Q.packed_paged_prefill_attention_quantized(qg[None], *args, _i32([[n - 1]]), _i32([0, 1]), bs, 1 / 8, hq // hkv, num_decode_rows=0)
    else:
        out = Q.paged_decode_attention_quantized(qg, *args, 1 / 8, form=route)
    kk, vv = (R.gather(codes, s, tables[0], n) for codes, s in state)
    want = R.attend(q64, kk, vv, np.ones((1, n), bool), 1 / 8)[0]
    off = _f64(out).reshape(hq, d) - want
    # a weight is at least 2^-18 of itself right (above), the sums cut 2^-23 of their size n / 8 times in the mean half a place
    assert np.linalg.norm(off) <= 1e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("queries", [2.0 ** 40, 2.0 ** -40, 0.0])
def test_queries_of_any_size(queries, form):
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(13)
    lens = [50, 20]
    tables = _tables(rng, lens, bs, 10)
    state = [_pool(rng, 10, shape) for _ in range(2)]
    state[0][1][:] *= 1 / queries if queries else 1
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    for dtype in (BF16, F32):
        q = torch.from_numpy(rng.standard_normal((2, hq, d)) * queries).to(dtype).cuda()
        out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), 1 / 16, form=form)
        _check(_f64(out)[:, None], _f64(q)[:, None], state, tables, lens, [[n] for n in lens], 1 / 16, TERM_BITS[form])


@pytest.mark.parametrize("form", FORMS)
def test_nan_and_infinite_queries_stay_in_their_row_and_head(form):
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(14)
    lens = [50, 40]
    tables = _tables(rng, lens, bs, 10)
    state = [_pool(rng, 10, shape) for _ in range(2)]
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    q = torch.from_numpy(rng.standard_normal((2, hq, d))).to(BF16).cuda()
    clean = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), 1 / 16, form=form)
    q[0, 3, 7], q[1, 6, 0] = float("nan"), float("inf")
    out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), 1 / 16, form=form)
    assert torch.isnan(out[0, 3]).all() and torch.isnan(out[1, 6]).all()
    out[0, 3], out[1, 6] = clean[0, 3], clean[1, 6]
    assert torch.equal(out, clean)


def test_what_lies_outside_the_pool_or_the_table_is_flagged(monkeypatch):
    hq, hkv, d, bs = shape = SHAPES[1]
    rng = np.random.default_rng(15)
    state = [_pool(rng, 8, shape) for _ in range(2)]
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    q, q64 = _queries(rng, (2, hq, d), BF16)
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")
    tables = np.array([[1, 8, 3], [4, 5, -7]])
    for form in (None, 1, 2):
        if form is None:
            out = Q.packed_paged_prefill_attention_quantized(q[None], k, v, ks, vs, _i32(tables), _i32([48, 40]), _i32([[47, 39]]), _i32([0, 1, 2]), bs,
                                                             d ** -0.5, hq // hkv, num_decode_rows=0)[0].view(2, hq, d)
        else:
            out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32([48, 40]), d ** -0.5, form=form)
        for r, good in ((0, [0, 2]), (1, [0, 1])):  # the other blocks' keys alone
            kk, vv = (R.gather(codes, s, tables[r][good], 32) for codes, s in state)
            want = R.attend(q64[r: r + 1], kk, vv, np.ones((1, 32), bool), d ** -0.5)[0]
            assert np.abs(_f64(out[r]) - want).max() <= R.tolerance(q64[r: r + 1], kk, vv, d ** -0.5, TERM_BITS.get(form, 22))
        with pytest.raises(K.DeviceStatusError, match="device status 2 "):
            K.check_device_status()
    for form in FORMS:
        long = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32([[1, 2], [3, 4]]), _i32([33, 1 << 30]), d ** -0.5, form=form)
        with pytest.raises(K.DeviceStatusError, match="device status 4 "):
            K.check_device_status()
        assert torch.equal(long, Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32([[1, 2], [3, 4]]), _i32([32, 32]), d ** -0.5, form=form))


def test_blocks_beyond_four_gigabytes():
    hq, hkv, d, bs = shape = SHAPES[0]
    blocks = (1 << 32) // (bs * hkv * d) + 50
    free, _ = torch.cuda.mem_get_info()
    if free < 4 * blocks * bs * hkv * d:
        pytest.skip("needs 18 GB of free device memory")
    rng = np.random.default_rng(16)
    state = [_pool(rng, 6, shape) for _ in range(2)]
    far = np.array([0, blocks - 1, blocks - 40, 7, blocks // 2 + 3, blocks - 2])
    big = []
    for codes, scale in state:
        numbers = torch.zeros((blocks, bs, hkv, d), dtype=torch.uint8, device="cuda")
        scales = torch.ones((blocks, hkv), device="cuda")
        numbers[far], scales[far] = torch.from_numpy(codes).cuda(), torch.from_numpy(scale).float().cuda()
        big.append((numbers.view(torch.float8_e4m3fn), scales))
    new = torch.from_numpy(rng.standard_normal((2, 1, hkv, d))).to(BF16).cuda()
    local = np.array([[0, 1, 2], [3, 4, 5]])
    Q.kv_append_quantized(new, new, big[0][0], big[1][0], big[0][1], big[1][1], _i32([[40], [47]]), _i32(far[local]))
    for codes, scale in state:
        R.append(codes, scale, _f64(new)[:, 0], [(2, 8), (5, 15)], bs)
    _same([(n.view(torch.uint8)[far].view(torch.float8_e4m3fn), s[far]) for n, s in big], state)
    q, q64 = _queries(rng, (2, hq, d), BF16)
    for form in FORMS:
        out = Q.paged_decode_attention_quantized(q, big[0][0], big[1][0], big[0][1], big[1][1], _i32(far[local]), _i32([41, 48]), 1 / 16, form=form)
        _check(_f64(out)[:, None], q64[:, None], state, local, [41, 48], [[41], [48]], 1 / 16, TERM_BITS[form])
    for dtype in (BF16, F32):
        out = Q.packed_paged_prefill_attention_quantized(q.to(dtype)[None], big[0][0], big[1][0], big[0][1], big[1][1], _i32(far[local]), _i32([41, 48]),
                                                         _i32([[40, 47]]), _i32([0, 1, 2]), bs, 1 / 16, 4, num_decode_rows=0)
        _check(_f64(out).reshape(2, 1, hq, d), q64[:, None], state, local, [41, 48], [[41], [48]], 1 / 16, 16)


@pytest.mark.parametrize("shape,form", [(SHAPES[3], 1), (SHAPES[6], 2)])
def test_more_rows_than_a_grid_dimension_holds(shape, form):
    hq, hkv, d, bs = shape
    rows = 65536 + 5
    rng = np.random.default_rng(17)
    state = [_pool(rng, 30, shape) for _ in range(2)]
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    tables, lens = rng.integers(0, 30, (rows, 1)), rng.integers(0, bs + 1, rows)
    q = torch.randn((rows, hq, d), device="cuda").to(BF16)
    out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), d ** -0.5, form=form)
    assert torch.isfinite(out).all()
    pick = [0, 1, 40000, 65534, 65535, 65536, rows - 1]
    _check(_f64(out[pick])[:, None], _f64(q[pick])[:, None], state, tables[pick], lens[pick], [[n] for n in lens[pick]], d ** -0.5, TERM_BITS[form])


# ------------------------------------------------------------------------------------------------ packed prefill

PACKED = [[(5, 0), (1, 40), (130, 3), (0, 9), (17, 100), (1, 0), (64, 64)], [(1, 30), (1, 5), (1, 64)], [(300, 0)], [(3, 500)]]


@pytest.mark.parametrize("rows", PACKED)
@pytest.mark.parametrize("shape,dtype", [(s, BF16) for s in SHAPES] + [(SHAPES[0], F32), (SHAPES[0], F16), (SHAPES[1], F32), (SHAPES[2], F16)])
def test_packed_prefill(shape, dtype, rows):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(18)
    lens = [n + c for n, c in rows]
    tables = _tables(rng, lens, bs, 120)
    state = [_pool(rng, 120, shape) for _ in range(2)]
    _poison_behind(state, tables, lens, bs)
    total, pad = sum(n for n, _ in rows), 7
    q, q64 = _queries(rng, (1, total + pad, hq, d), dtype)
    positions = np.concatenate([np.arange(c, c + n) for n, c in rows] + [np.zeros(pad)])[None]
    qsl = np.cumsum([0] + [n for n, _ in rows])
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    singles = sum(n == 1 for n, _ in rows)
    tiles = sum(-(-n // 64) for n, _ in rows if n > 1)
    counts = [dict(), dict(num_decode_rows=singles, query_tile_pairs=tiles)]
    if singles:
        counts.append(dict(num_decode_rows=0))  # (then the tiles serve them)
    term_bits = 16 if shape == SHAPES[0] and dtype == BF16 else 22  # the tcgen05 tiles' weights are two bf16 terms
    for count in counts:
        out = Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), _i32(positions), _i32(qsl), bs, d ** -0.5,
                                                         hq // hkv, **count)
        assert out.shape == (1, total + pad, hq * d) and not out[0, total:].any()
        got = _f64(out).reshape(-1, hq, d)
        _check([got[a:b] for a, b in zip(qsl, qsl[1:])], [q64[0, a:b] for a, b in zip(qsl, qsl[1:])], state, tables, lens,
               [c + 1 + np.arange(n) for n, c in rows], d ** -0.5, term_bits)


@pytest.mark.parametrize("shape,dtype", [(SHAPES[0], BF16), (SHAPES[0], F32), (SHAPES[1], BF16)])
def test_packed_prefill_of_rows_without_keys_and_of_fewer_keys_than_positions(shape, dtype):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(19)
    rows, lens = [(20, 0), (1, 0), (33, 10), (70, 0)], [0, 0, 25, 41]
    tables = _tables(rng, [48] * 4, bs, 40)
    state = [_pool(rng, 40, shape) for _ in range(2)]
    q, q64 = _queries(rng, (1, 124, hq, d), dtype)
    positions = np.concatenate([np.arange(c, c + n) for n, c in rows])[None]
    qsl = np.cumsum([0] + [n for n, _ in rows])
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    out = Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), _i32(positions), _i32(qsl), bs, d ** -0.5, hq // hkv)
    got = _f64(out).reshape(-1, hq, d)
    _check([got[a:b] for a, b in zip(qsl, qsl[1:])], [q64[0, a:b] for a, b in zip(qsl, qsl[1:])], state, tables, lens,
           [c + 1 + np.arange(n) for n, c in rows], d ** -0.5, 16 if dtype == BF16 and shape == SHAPES[0] else 22)


def test_a_table_too_wide_for_the_pages_goes_to_the_other_tiles():
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(20)
    lens = [100, 37]
    narrow = _tables(rng, lens, bs, 20)
    wide = np.zeros((2, 20000), np.int32)
    wide[:, : narrow.shape[1]] = narrow
    state = [_pool(rng, 20, shape) for _ in range(2)]
    q, q64 = _queries(rng, (1, 137, hq, d), BF16)
    positions, qsl = np.concatenate([np.arange(n) for n in lens])[None], np.array([0, 100, 137])
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    out = Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, _i32(wide), _i32(lens), _i32(positions), _i32(qsl), bs, 1 / 16, 4)
    got = _f64(out).reshape(-1, hq, d)
    _check([got[:100], got[100:]], [q64[0, :100], q64[0, 100:]], state, narrow, lens, [1 + np.arange(n) for n in lens], 1 / 16)


@pytest.mark.parametrize("keys,tokens", [(9000, 5000), (25000, 4700), (16449, 5100)])  # (no split of the key ranges: accumulators are emptied once, or three times)
def test_packed_prefill_over_many_keys(keys, tokens):
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(21)
    blocks = -(-keys // bs)
    state = [_pool(rng, blocks, shape, spread=1) for _ in range(2)]
    tables = rng.permutation(blocks)[None]
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    q, q64 = _queries(rng, (1, tokens, hq, d), BF16)
    positions = np.arange(keys - tokens, keys)[None]
    out = _f64(Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32([keys]), _i32(positions), _i32([0, tokens]), bs, 1 / 16, 4,
                                                          num_decode_rows=0)).reshape(tokens, hq, d)
    pick = [0, 63, 64, 100, tokens // 2 + 1, tokens - 1]
    _check([out[pick]], [q64[0, pick]], state, tables, [keys], [positions[0, pick] + 1], 1 / 16, 16)


def _long_prefill(shape, dtype, rows, counts, term_bits, seed, spread=1):
    """`rows` of (new, cached) tokens, checked at some of their tokens."""
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(seed)
    lens = [n + c for n, c in rows]
    blocks = sum(-(-n // bs) for n in lens)
    order, tables, at = rng.permutation(blocks), np.zeros((len(rows), max(-(-n // bs) for n in lens)), np.int64), 0
    for r, n in enumerate(lens):
        tables[r, : -(-n // bs)] = order[at: at + -(-n // bs)]
        at += -(-n // bs)
    state = [_pool(rng, blocks, shape, spread=spread) for _ in range(2)]
    _poison_behind(state, tables, lens, bs)
    (k, ks), (v, vs) = (_gpu(*x) for x in state)
    total = sum(n for n, _ in rows)
    q, q64 = _queries(rng, (1, total, hq, d), dtype)
    positions, qsl = np.concatenate([np.arange(c, c + n) for n, c in rows])[None], np.cumsum([0] + [n for n, _ in rows])
    out = _f64(Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), _i32(positions), _i32(qsl), bs, d ** -0.5, hq // hkv,
                                                          **counts)).reshape(total, hq, d)
    for r, (n, c) in enumerate(rows):
        pick = sorted({0, n // 3, 2 * n // 3, n - 1})
        at = [qsl[r] + i for i in pick]
        _check([out[at]], [q64[0, at]], state, tables[r: r + 1], lens[r: r + 1], [[c + 1 + i for i in pick]], d ** -0.5, term_bits)


# few query tokens: clusters share a tile's keys; at 40000 keys and more each CTA empties its sums into scratch
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(32, 8, 128, 16), (16, 1, 256, 16), (24, 2, 128, 64), (6, 6, 64, 48), (8, 2, 256, 32)])
@pytest.mark.parametrize("rows", [[(2, 700)], [(20, 3000), (3, 17), (5, 0)], [(9, 45000)], [(17, 33000), (2, 70)]])
def test_prefill_of_few_tokens_over_many_keys(shape, dtype, rows):
    _long_prefill(shape, dtype, rows, dict(num_decode_rows=0, query_tile_pairs=len(rows)), 22, 31)


# tiles enough for every SM: a CTA takes all keys of its rows, and empties its sums into the output every 4096 of them
@pytest.mark.parametrize("shape,dtype", [((32, 8, 128, 16), F16), ((16, 1, 256, 16), F32), ((16, 8, 64, 32), BF16)])
def test_prefill_of_many_tokens_over_many_keys(shape, dtype):
    _long_prefill(shape, dtype, [(610, 8500), (700, 3487)], dict(num_decode_rows=0), 22, 32)


# the caller's count of tiles only sets how many CTAs share one: too small, too large or nothing
@pytest.mark.parametrize("tiles", [None, 0, 1, 10 ** 6])
def test_prefill_with_any_count_of_tiles(tiles):
    _long_prefill((32, 8, 128, 16), BF16, [(150, 900), (70, 0), (2, 333)], dict(num_decode_rows=0, query_tile_pairs=tiles), 22, 33)


# rows of several windows of 32 tiles per warp; a block outside the pool in a later window
@pytest.mark.parametrize("shape,dtype", [((6, 6, 64, 48), BF16), ((16, 2, 64, 32), F16), ((32, 8, 64, 16), F32), ((4, 1, 128, 16), BF16)])
def test_long_rows_on_the_mma_sync_tiles(shape, dtype, monkeypatch):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(37)
    rows, width = 130, 20000 // bs
    lens = rng.integers(1, width * bs + 1, rows)
    lens[:4] = [width * bs, 8193, 16400, 1]
    tables = rng.integers(0, 90, (rows, width))  # (rows share blocks)
    state = [_pool(rng, 90, shape, spread=1) for _ in range(2)]
    (k, ks), (v, vs) = (_gpu(*x) for x in state)
    q, q64 = _queries(rng, (rows, hq, d), dtype)
    out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), d ** -0.5, form=1)
    pick = [0, 1, 2, 3, 77, 129]
    _check(_f64(out[pick])[:, None], q64[pick][:, None], state, tables[pick], lens[pick], [[n] for n in lens[pick]], d ** -0.5)
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")
    for bad in (90, -3, 1 << 30):
        broken = tables.copy()
        broken[0, 12000 // bs] = bad
        got = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(broken), _i32(lens), d ** -0.5, form=1)
        with pytest.raises(K.DeviceStatusError, match="device status 2 "):
            K.check_device_status()
        seen = np.arange(lens[0]) // bs != 12000 // bs
        kk, vv = (R.gather(codes, x, tables[0], lens[0]) for codes, x in state)
        want = R.attend(q64[:1], kk[seen], vv[seen], np.ones((1, seen.sum()), bool), d ** -0.5)[0]
        assert np.abs(_f64(got[0]) - want).max() <= R.tolerance(q64[:1], kk, vv, d ** -0.5)
        assert torch.equal(got[1:], out[1:])


TILES = [((32, 8, 128, 16), F16), ((16, 1, 256, 16), BF16), ((8, 2, 256, 16), F32), ((16, 2, 64, 32), BF16)]  # shapes of the 8-bit tiles


def _prefill(q, state_gpu, tables, lens, rows, shape, scale):
    (k, ks), (v, vs) = state_gpu
    positions, qsl = np.concatenate([np.arange(c, c + n) for n, c in rows])[None], np.cumsum([0] + [n for n, _ in rows])
    return Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), _i32(positions), _i32(qsl), shape[3], scale,
                                                      shape[0] // shape[1], num_decode_rows=0)


@pytest.mark.parametrize("scale", [0.0, -0.07, 1.5])
@pytest.mark.parametrize("shape,dtype", TILES)
def test_prefill_tiles_with_any_scale_of_the_scores_and_queries_of_any_size(shape, dtype, scale):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(34)
    rows = [(70, 200), (3, 61)]
    lens = [n + c for n, c in rows]
    tables = _tables(rng, lens, bs, 60)
    for size in (1.0, 2.0 ** 12, 2.0 ** -12):
        state = [_pool(rng, 60, shape, spread=1) for _ in range(2)]
        state[0][1][:] /= size
        q = torch.from_numpy(rng.standard_normal((1, 73, hq, d)) * size).to(dtype).cuda()
        out = _f64(_prefill(q, [_gpu(*x) for x in state], tables, lens, rows, shape, scale)).reshape(73, hq, d)
        q64 = _f64(q)[0]
        _check([out[:70], out[70:]], [q64[:70], q64[70:]], state, tables, lens, [c + 1 + np.arange(n) for n, c in rows], scale)


@pytest.mark.parametrize("shape,dtype", TILES)
def test_prefill_tiles_keep_nan_and_infinite_queries_in_their_row_and_head_and_nan_values_visible(shape, dtype):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(35)
    rows = [(40, 300), (9, 0)]
    lens = [n + c for n, c in rows]
    tables = _tables(rng, lens, bs, 60)
    state = [_pool(rng, 60, shape) for _ in range(2)]
    gpu = [_gpu(*x) for x in state]
    q = torch.from_numpy(rng.standard_normal((1, 49, hq, d))).to(dtype).cuda()
    clean = _prefill(q, gpu, tables, lens, rows, shape, d ** -0.5).view(49, hq, d)
    odd = q.clone()
    odd[0, 5, 3, 7], odd[0, 44, 0, 0] = float("nan"), float("-inf")
    out = _prefill(odd, gpu, tables, lens, rows, shape, d ** -0.5).view(49, hq, d)
    assert torch.isnan(out[5, 3]).all() and torch.isnan(out[44, 0]).all()
    out[5, 3], out[44, 0] = clean[5, 3], clean[44, 0]
    assert torch.equal(out, clean)
    gpu[1][0].view(torch.uint8)[tables[0, 1], 2, hkv - 1, 9] = 127  # a value that all of row 0's tokens see
    out = _prefill(q, gpu, tables, lens, rows, shape, d ** -0.5).view(49, hq, d)
    heads = slice((hkv - 1) * (hq // hkv), hq)
    assert torch.isnan(out[:40, heads, 9]).all()
    out[:40, heads, 9] = clean[:40, heads, 9]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("shape,dtype", TILES)
def test_prefill_tiles_from_a_graph_on_another_stream_and_bit_for_bit(shape, dtype):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(36)
    rows = [(30, 500), (100, 7)]
    lens = [n + c for n, c in rows]
    tables = _tables(rng, lens, bs, 80)
    gpu = [_gpu(*_pool(rng, 80, shape)) for _ in range(2)]
    q = torch.from_numpy(rng.standard_normal((1, 130, hq, d))).to(dtype).cuda()
    want = _prefill(q, gpu, tables, lens, rows, shape, d ** -0.5)
    (k, ks), (v, vs) = gpu
    positions, qsl = np.concatenate([np.arange(c, c + n) for n, c in rows])[None], np.cumsum([0] + [n for n, _ in rows])
    args = [_i32(x) for x in (tables, lens, positions, qsl)]
    from nano_vllm_jax_b200.engine.resident_decode import CapturedStep
    steps = [CapturedStep(lambda: Q.packed_paged_prefill_attention_quantized(q, k, v, ks, vs, *args, bs, d ** -0.5, hq // hkv, num_decode_rows=0)) for _ in range(2)]
    for step in steps:
        step.capture()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        for step in steps:
            step.result.fill_(float("nan"))
        torch.cuda.synchronize()
        for step, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                step.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(step.result, want) for step in steps)


# ------------------------------------------------------------------------------------------------ refusals

def test_the_other_entry_points_refuse_8_bit_caches():
    hq, hkv, d, bs = SHAPES[0]
    k5 = torch.zeros(1, 4, bs, hkv, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    k, v = k5[0], k5[0].clone()
    tables, lens, q = _i32([[0, 1], [2, 3]]), _i32([3, 4]), torch.zeros(2, 1, hq, d, device="cuda", dtype=BF16)
    new, pos = torch.zeros(2, 1, hkv, d, device="cuda", dtype=BF16), _i32([[2], [3]])
    calls = [lambda: K.paged_decode_attention(q, k, v, tables, lens, 0.1),
             lambda: K.paged_decode_attention_wide(q, k, v, tables, lens, pos, 0.1),
             lambda: K.paged_decode_attention_with_kv_append(q, new, new, k5, k5.clone(), tables, lens, pos, 0, bs, 0.1, hq // hkv),
             lambda: K.packed_paged_prefill_attention(q.reshape(1, 2, hq, d), k, v, tables, lens, pos.reshape(1, 2), _i32([0, 1, 2]), bs, 0.1, hq // hkv),
             lambda: K.kv_append_slots(new, new, _i32([[2], [35]]), k, v),
             lambda: K.copy_blocks(k5, k5.clone(), _i32([0]), _i32([1]))]
    for call in calls:
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
    torch.cuda.synchronize()
    assert not k5.view(torch.uint8).any() and not v.view(torch.uint8).any()


def test_wrappers_refuse_what_does_not_fit_together():
    hq, hkv, d, bs = SHAPES[0]
    k = torch.zeros(4, bs, hkv, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.ones(4, hkv, device="cuda")
    tables, lens = _i32([[0, 1], [2, 3]]), _i32([3, 4])
    q, new, pos = torch.zeros(2, hq, d, device="cuda"), torch.zeros(2, 1, hkv, d, device="cuda"), _i32([[0], [0]])

    def decode(q=q, k=k, s=s, tables=tables, lens=lens, **more):
        return Q.paged_decode_attention_quantized(q, k, k, s, s, tables, lens, 1.0, **more)

    def append(new=new, k=k, s=s, pos=pos, tables=tables, **more):
        return Q.kv_append_quantized(new, new, k, k, s, s, pos, tables, **more)

    for call, change, match in [
            (decode, {"k": k.view(torch.uint8)}, "float8_e4m3fn"), (decode, {"k": k[:, :8].contiguous()}, "page_size"),
            (decode, {"k": k[..., :32].contiguous()}, "head_dim"), (decode, {"s": s.half()}, "float32"), (decode, {"s": s[:3]}, "num_kv_heads"),
            (decode, {"k": k.transpose(1, 2)}, "contiguous"), (decode, {"q": q[0]}, "shape"), (decode, {"q": q[:, :7]}, "divisible"),
            (decode, {"q": q[..., :128]}, "head_dim"), (decode, {"q": q.double()}, "dtype"), (decode, {"tables": tables.long()}, "int32"),
            (decode, {"tables": tables[:1]}, "block_table"), (decode, {"lens": lens[:1]}, "seq_lens"), (decode, {"positions": lens[:1]}, "positions"),
            (append, {"new": new[..., :128]}, "heads"), (append, {"new": new[0]}, "shape"), (append, {"pos": pos[:1]}, "positions"),
            (append, {"tables": tables[:1]}, "batch"), (append, {"token_row_ids": pos}, "packed"), (append, {"seq_lens": lens[:1]}, "seq_lens"),
            (append, {"pos": pos.long()}, "int32"), (append, {"tables": tables[:, :0]}, "empty"), (append, {"new": new.to(torch.float64)}, "dtype")]:
        with pytest.raises(ValueError, match=match):
            call(**change)
    with pytest.raises(ValueError, match="positions"):
        Q.packed_paged_prefill_attention_quantized(q[None], k, k, s, s, tables, lens, pos, _i32([0, 1, 2]), bs, 1.0, 4)
    with pytest.raises(ValueError, match="agree"):
        Q.packed_paged_prefill_attention_quantized(q[None], k, k, s, s, tables, lens, pos.T.contiguous(), _i32([0, 1, 2]), bs, 1.0, 2)
    with pytest.raises(ValueError, match="query_start_loc"):
        Q.packed_paged_prefill_attention_quantized(q[None], k, k, s, s, tables, lens, pos.T.contiguous(), _i32([0, 1]), bs, 1.0, 4)


# ------------------------------------------------------------------------------------------------ streams and graphs

def test_on_another_stream_and_replayed_from_a_graph():
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(22)
    lens = [40, 300, 17, 0]
    tables = _tables(rng, [n + 1 for n in lens], bs, 60)
    state = [_pool(rng, 60, shape) for _ in range(2)]
    gpu = [_gpu(*s) for s in state]
    k, ks, v, vs = gpu[0][0], gpu[0][1], gpu[1][0], gpu[1][1]
    q, q64 = _queries(rng, (4, hq, d), BF16)
    new = torch.from_numpy(rng.standard_normal((4, 1, hkv, d))).to(BF16).cuda()
    t, l, p = _i32(tables), _i32(lens), _i32(np.maximum(np.array(lens) - 1, 0)[:, None])

    def step():
        Q.kv_append_quantized(new, new, k, v, ks, vs, p, t, seq_lens=l)
        return Q.paged_decode_attention_quantized(q, k, v, ks, vs, t, l, 1 / 16)

    from nano_vllm_jax_b200.engine.resident_decode import CapturedStep
    captured = CapturedStep(step)
    first = captured.capture()
    for codes, scale in state:
        R.append(codes, scale, _f64(new)[:, 0], [(int(tables[r, (n - 1) // bs]), (n - 1) % bs) if n else None for r, n in enumerate(lens)], bs)
    for _ in range(3):
        captured.result.fill_(float("nan"))
        out = captured.replay()
        torch.cuda.synchronize()
        _same(gpu, state)
        _check(_f64(out)[:, None], q64[:, None], state, tables, lens, [[n] for n in lens], 1 / 16)
        assert torch.equal(out, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    K.check_device_status()


def test_two_captured_prefills_and_an_eager_one_do_not_share_scratch():
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(23)
    from nano_vllm_jax_b200.engine.resident_decode import CapturedStep
    made = []
    for seed in range(2):
        state = [_pool(rng, 40, shape) for _ in range(2)]
        (k, ks), (v, vs) = (_gpu(*s) for s in state)
        tables, q = _tables(rng, [200, 70], bs, 40), torch.from_numpy(rng.standard_normal((1, 150, hq, d))).to(BF16).cuda()
        pos = np.concatenate([np.arange(100, 200), np.arange(20, 70)])[None]
        args = (q, k, v, ks, vs, _i32(tables), _i32([200, 70]), _i32(pos), _i32([0, 100, 150]), bs, 1 / 16, 4)
        step = CapturedStep(lambda args=args: Q.packed_paged_prefill_attention_quantized(*args, num_decode_rows=0))
        made.append((step, step.capture().clone(), args))
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(3):
        for (step, _, _), s in zip(made, streams):
            step.result.fill_(float("nan"))
        torch.cuda.synchronize()
        for (step, _, _), s in zip(made, streams):
            with torch.cuda.stream(s):
                step.replay()
        eager = Q.packed_paged_prefill_attention_quantized(*made[0][2], num_decode_rows=0)
        torch.cuda.synchronize()
        assert torch.equal(eager, made[0][1])
        for step, want, _ in made:
            assert torch.equal(step.result, want)


def test_the_same_inputs_give_the_same_bits():
    hq, hkv, d, bs = shape = SHAPES[0]
    rng = np.random.default_rng(24)
    lens = [3000, 1, 900]
    tables = _tables(rng, lens, bs, 260)
    state = [_pool(rng, 260, shape) for _ in range(2)]
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    q, _ = _queries(rng, (3, hq, d), BF16)
    for form in FORMS:
        first = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), 1 / 16, form=form)
        for _ in range(5):
            assert torch.equal(first, Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), 1 / 16, form=form))


@pytest.mark.parametrize("shape,dtype,rows,hi", [(SHAPES[0], BF16, 300, 700), (SHAPES[1], F16, 40, 1500), (SHAPES[4], F32, 9, 2500), (SHAPES[6], BF16, 1, 9000)])
def test_rows_cut_over_many_ranges_of_the_tcgen05_tiles(shape, dtype, rows, hi):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(rows)
    lens = rng.integers(0, hi + 1, rows)
    lens[0] = hi
    tables = _tables(rng, lens, bs, int((-(-lens // bs)).sum()))
    state = [_pool(rng, int(tables.max()) + 1, shape) for _ in range(2)]
    _poison_behind(state, tables, lens, bs)
    q, q64 = _queries(rng, (rows, hq, d), dtype)
    (k, ks), (v, vs) = (_gpu(*s) for s in state)
    out = Q.paged_decode_attention_quantized(q, k, v, ks, vs, _i32(tables), _i32(lens), d ** -0.5, form=2)
    _check(_f64(out)[:, None], q64[:, None], state, tables, lens, [[n] for n in lens], d ** -0.5, TERM_BITS[2])
