"""Append with rotation and key bounds, selection of blocks, attention over them: each against its plain form in 64 bits, and together."""

import numpy as np
import pytest
import torch

import selective_reference as R
from nano_vllm_jax_b200.kernels import paged_kv as K
from nano_vllm_jax_b200.kernels import selective_kv as S

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}  # a rounding, relative
MODEL = (8, 2, 256, 16)  # query heads, kv heads, head_dim, block size
LAYOUTS = [MODEL, (32, 8, 128, 32), (16, 2, 64, 16), (4, 4, 64, 48), (24, 2, 128, 64), (6, 3, 96, 16), (5, 1, 40, 7), (16, 1, 256, 16)]
TYPES = [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16), (BF16, F32), (F16, BF16)]


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _f64(t):
    return t.double().cpu().numpy()


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _freq(n, base=1e7):
    return (base ** (-np.arange(n) / max(1, n))).astype(np.float32)


def _bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _tables(rng, room, bs, spare=3, extra=2):
    need = [-(-r // bs) for r in room]
    ids, at = rng.permutation(sum(need) + spare), 0
    tables = np.zeros((len(room), max(need) + extra), np.int64)
    for r, n in enumerate(need):
        tables[r, :n] = ids[at: at + n]
        at += n
    return tables, sum(need) + spare


# ------------------------------------------------------------------------------------------------ append

def _check_append(seed, layout, types, runs, rot, pairs, form="packed", pad=0, bounded=True, with_q=True, base=1e7):
    """`runs`: (position of the first new token, number of them) of each row; `form` packed, rows (rectangular), fused (views of a projection)."""
    hq, hkv, d, bs = layout
    act, held = types
    g, rng = _gen(seed), np.random.default_rng(seed)
    tables, pool = _tables(rng, [c + n for c, n in runs], bs)
    k0, v0 = _normal(g, held, pool, bs, hkv, d), _normal(g, held, pool, bs, hkv, d)
    b0 = torch.stack((k0.amin(1), k0.amax(1)), 2).contiguous()
    cols = max(n for _, n in runs) if form == "rows" else sum(n for _, n in runs) + pad
    rows = len(runs) if form == "rows" else 1
    if form == "fused":
        x = _normal(g, act, rows, cols, (hq + 2 * hkv) * d)
        q, nk, nv = (t.unflatten(-1, (-1, d)) for t in x.split((hq * d, hkv * d, hkv * d), -1))
    else:
        q, nk, nv = (_normal(g, act, rows, cols, h, d) for h in (hq, hkv, hkv))
    if form == "rows":
        pos = np.array([[c + i if i < n else 0 for i in range(cols)] for c, n in runs])
        owner, qsl = np.repeat(np.arange(rows), cols), np.concatenate([[0], np.cumsum([n for _, n in runs])])
        live = np.array([[i < n for i in range(cols)] for _, n in runs]).ravel()
        ids = None
    else:
        pos = np.concatenate([np.arange(c, c + n) for c, n in runs] + [np.zeros(pad, np.int64)])[None]
        owner = np.concatenate([np.full(n, r) for r, (_, n) in enumerate(runs)] + [np.zeros(pad, np.int64)])
        qsl = np.concatenate([[0], np.cumsum([n for _, n in runs])])
        live = np.arange(cols) < qsl[-1]
        ids = _i32(owner[None])
    freq = _freq(rot // 2, base)
    k, v, b = k0.clone(), v0.clone(), b0.clone()
    out = S.rope_kv_append(q if with_q else None, nk, nv, k, v, _i32(pos), _i32(tables), torch.from_numpy(freq).cuda(), k_bounds=b if bounded else None,
                           query_start_loc=_i32(qsl), token_row_ids=ids, interleaved=pairs)
    flat = pos.ravel()

    def close(got, x, dtype):
        """Cosine and sine are good to 2^-22 (2 ulp), a product and the sum to 2^-24 each; then one rounding, subnormal steps included."""
        want, both = R.rotate(x, flat, freq, pairs), R.partners(x, rot // 2, pairs)
        slip = 2.0 ** -21 * both
        return np.abs(got - want) <= slip + HALF[dtype] * (np.abs(want) + slip) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps

    if with_q:
        assert close(_f64(out).reshape(-1, hq, d), _f64(q).reshape(-1, hq, d), act).all()
    else:
        assert out is None
    # what was written: every live token in its place, everything else as it was
    want_k, want_v, want_b = k0.clone(), v0.clone(), b0.clone()
    got_k = _f64(k)
    xs = _f64(nk).reshape(-1, hkv, d)
    stored_v = nv.reshape(-1, hkv, d).to(held)
    touched = {}
    ok = close(got_k[tables[owner, flat // bs], flat % bs], xs, held)  # (padded tokens' places are not looked at)
    assert ok[live].all()
    for i in np.flatnonzero(live):
        block, o = tables[owner[i], flat[i] // bs], flat[i] % bs
        want_k[block, o], want_v[block, o] = k[block, o], stored_v[i]
        touched.setdefault(int(block), []).append(int(o))
    assert np.array_equal(_bits(k), _bits(want_k)) and np.array_equal(_bits(v), _bits(want_v))
    if bounded:
        for block, offsets in touched.items():
            new = k[block, offsets]
            low, high = new.amin(0), new.amax(0)
            if 0 not in offsets:
                low, high = torch.minimum(low, b0[block, :, 0]), torch.maximum(high, b0[block, :, 1])
            want_b[block] = torch.stack((low, high), 1)
    assert torch.equal(b, want_b)


@pytest.mark.parametrize("layout", LAYOUTS[:6] + LAYOUTS[7:], ids=str)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
def test_append_packed_rows_at_all_depths(layout, types):
    d, bs = layout[2:]
    runs = [(0, 5), (3, 1), (bs - 1, 2), (bs, bs), (2 * bs + 1, 3 * bs), (5, 40), (7 * bs - 3, 1)]
    _check_append(1, layout, types, runs, min(64, d), False, pad=9)
    _check_append(2, layout, types, runs, d, True, form="fused")


@pytest.mark.parametrize("rot", [0, 2, 16, 20, 34, 48, 64, 128, 250, 256])
@pytest.mark.parametrize("pairs", [False, True])
def test_append_rotary_dims(rot, pairs):
    runs = [(100, 17), (0, 1), (63, 2)]
    _check_append(rot, MODEL, (BF16, BF16), runs, rot, pairs)
    _check_append(rot + 1, (3, 3, 128, 16), (F32, F32), [(77, 1), (5, 9)], min(rot, 128), pairs, form="fused")
    _check_append(rot + 2, (6, 2, 64, 16), (F16, F16), [(31, 70)], min(rot, 64), pairs)


def test_append_decode_batches_and_rectangles():
    for layout in (MODEL, (32, 8, 128, 32), (6, 3, 96, 16), (2, 2, 8, 1)):
        d = layout[2]
        _check_append(5, layout, (BF16, BF16), [(c, 1) for c in (0, 1, 15, 16, 17, 300, 31, 32)], min(d, 64), False, form="rows")
        _check_append(6, layout, (BF16, F32), [(0, 3), (14, 5), (31, 1), (9, 0), (64, 2)], min(d, 64), False, form="rows")
        _check_append(7, layout, (F32, BF16), [(0, 40), (14, 33)], 0, False, form="rows", with_q=False)
        _check_append(8, layout, (F32, F16), [(10, 20)], min(d, 64), True, bounded=False)


def test_append_far_positions_keep_their_angles():
    """Positions whose angle a product in 32 bits would put 2^-24 * 2e6 = 0.1 aside."""
    _check_append(9, (2, 1, 64, 16), (F32, F32), [(2 ** 17 - 3, 5)], 64, False, base=1e4)
    g = _gen(3)
    q, kv = _normal(g, F32, 3, 1, 2, 64), _normal(g, F32, 3, 1, 1, 64)
    k, v = torch.zeros(1, 1, 1, 64, device="cuda"), torch.zeros(1, 1, 1, 64, device="cuda")
    pos = np.array([[2 ** 21 + 1], [2 ** 30 + 12345], [2 ** 31 - 1]])
    freq = _freq(32, 1e4)
    out = S.rope_kv_append(q, kv, kv, k, v, _i32(pos), torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.from_numpy(freq).cuda(),
                           seq_lens=_i32([0, 0, 0]))
    x = _f64(q)[:, 0]
    want = R.rotate(x, pos.ravel(), freq, False)
    # the reference's own angle is off by 2^-53 of it, as the kernel's is: 2^-22
    assert (np.abs(_f64(out)[:, 0] - want) <= 2.0 ** -19 * R.partners(x, 32, False)).all()
    assert not k.any() and not v.any()


def test_append_bounds_keep_what_is_not_a_number_and_infinities():
    g = _gen(4)
    k, v = (torch.zeros(3, 16, 2, 64, dtype=BF16, device="cuda") for _ in range(2))
    b = torch.zeros(3, 2, 2, 64, dtype=BF16, device="cuda")
    nk = _normal(g, BF16, 1, 20, 2, 64)
    nk[0, 3, 0, 5], nk[0, 4, 1, 6], nk[0, 17, 1, 7] = float("nan"), float("inf"), -float("inf")
    ids = torch.zeros(1, 20, dtype=torch.int32, device="cuda")
    S.rope_kv_append(None, nk, nk, k, v, _i32([np.arange(20)]), _i32([[2, 0]]), None, k_bounds=b, token_row_ids=ids)
    assert b[2, 0, :, 5].isnan().all() and b[2, 1, 1, 6] == float("inf") and b[0, 1, 0, 7] == -float("inf")
    rest = torch.stack((nk[0, :16].amin(0), nk[0, :16].amax(0)), 1)
    assert torch.equal(b[2].nan_to_num(7.0), rest.nan_to_num(7.0))
    # a NaN stays when the block goes on
    S.rope_kv_append(None, nk[:, :1], nk[:, :1], k, v, _i32([[9]]), _i32([[2, 0]]), None, k_bounds=b)
    assert b[2, 0, :, 5].isnan().all()
    assert not b[1].any()


def test_append_strides_that_are_not_whole_vectors_are_copied():
    g = _gen(5)
    base = _normal(g, BF16, 1, 6, 3 * 64 + 1)
    odd = base[..., 1:].unflatten(-1, (3, 64))
    args = [odd, odd[:, :, :1], odd[:, :, 1:2]]
    outs = []
    for operands in (args, [t.contiguous() for t in args]):
        k, v = (torch.zeros(1, 16, 1, 64, dtype=BF16, device="cuda") for _ in range(2))
        q = S.rope_kv_append(*operands, k, v, _i32([np.arange(6)]), _i32([[0]]), torch.from_numpy(_freq(32)).cuda(),
                             token_row_ids=torch.zeros(1, 6, dtype=torch.int32, device="cuda"))
        outs.append((q, k, v))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("what,table,pos,rows", [("page", [[0, 99]], 17, [[0]]), ("page", [[-1, 0]], 3, [[0]]), ("length", [[0, 1]], 32, [[0]]),
                                                 ("length", [[0, 1]], -1, [[0]]), ("row", [[0, 1]], 3, [[1]]), ("row", [[0, 1]], 3, [[-1]])])
def test_append_flags_and_skips_places_that_are_not_there(what, table, pos, rows):
    g = _gen(6)
    k, v = (_normal(g, BF16, 2, 16, 2, 256) for _ in range(2))
    b = _normal(g, BF16, 2, 2, 2, 256)
    before = [t.clone() for t in (k, v, b)]
    new = _normal(g, BF16, 1, 1, 2, 256)
    with pytest.raises(K.DeviceStatusError, match="sequence length" if what == "length" else "outside the pool"):
        S.rope_kv_append(None, new, new, k, v, _i32([[pos]]), _i32(table), None, k_bounds=b, token_row_ids=_i32(rows))
    for t, u in zip((k, v, b), before):
        assert torch.equal(t, u)


# ------------------------------------------------------------------------------------------------ selection

def _selection(seed, layout, types, lens, positions, budget, first, last, change=None):
    hq, hkv, d, bs = layout
    act, held = types
    g, rng = _gen(seed), np.random.default_rng(seed)
    tables, pool = _tables(rng, [max(n, 1) for n in lens], bs)
    width = 1 if positions is None else np.asarray(positions).shape[1]
    q = _normal(g, act, len(lens), width, hq, d)
    k = _normal(g, held, pool, 4, hkv, d)
    bounds = torch.stack((k.amin(1), k.amax(1)), 2).contiguous()
    if change is not None:
        change(q, bounds, tables)
    out = S.select_blocks(q if positions is not None else q[:, 0], bounds, _i32(tables), _i32(lens), bs, budget,
                          positions=None if positions is None else _i32(positions), first=first, last=last)
    want = R.select(_f64(q), _f64(bounds), tables, lens, None if positions is None else np.asarray(positions), bs, budget, first, last)
    got = out.cpu().numpy()
    assert np.array_equal(got.reshape(want.shape), want)
    return got


@pytest.mark.parametrize("layout", LAYOUTS[:6] + LAYOUTS[7:], ids=str)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
def test_selection_of_rows_of_all_lengths(layout, types):
    bs = layout[3]
    lens = [0, 1, bs, 3 * bs, 8 * bs, 8 * bs + 1, 9 * bs - 1, 40 * bs + 3, 17 * bs, 33 * bs, 301 * bs]
    _selection(1, layout, types, lens, None, 8, 1, 2)


@pytest.mark.parametrize("budget,first,last", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (3, 1, 2), (4, 0, 4), (5, 2, 1), (64, 1, 1), (100, 7, 20), (200, 0, 0)])
def test_selection_budgets(budget, first, last):
    _selection(2, MODEL, (BF16, BF16), [16 * n for n in (1, 2, 5, 64, 65, 100, 101, 180, 201, 399)], None, budget, first, last)


def test_selection_of_several_tokens_and_masks():
    pos = [[-1, 0, 5, 400], [395, 396, 397, 398], [15, 16, 31, 32], [1000, 1000, 1000, 2 ** 31 - 1], [-5, -2 ** 31, 3, 500]]
    for layout in (MODEL, (6, 3, 96, 16), (16, 2, 64, 16)):
        _selection(3, layout, (BF16, BF16), [400, 399, 300, 640, 0], pos, 6, 1, 2)


@pytest.mark.parametrize("columns", [2000, 6000, S.MOST_COLUMNS - 2])  # (two more in the tables)
def test_selection_from_long_rows(columns):
    _selection(4, (4, 1, 64, 1), (BF16, BF16), [columns, columns - 1, 700], None, 257, 1, 2)


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (F16, F16)], ids=str)
def test_ties_go_to_the_lowest_column(types):
    def same(q, bounds, tables):
        bounds[:] = bounds[:1]

    def few(q, bounds, tables):
        bounds[:] = bounds[torch.arange(len(bounds), device="cuda") % 3]

    def zero(q, bounds, tables):
        bounds.zero_()

    def no_query(q, bounds, tables):
        q.zero_()
    for change in (same, few, zero, no_query):
        for layout in (MODEL, (6, 2, 48, 16)):
            _selection(5, layout, types, [16 * 70, 16 * 2300], None, 33, 1, 2, change)


def test_scores_that_fp32_cannot_tell_apart_are_told_apart():
    """Blocks of one large score and differences far below its rounding: 2^-30 of it and less."""
    def near(q, bounds, tables):
        q[:] = torch.randn_like(q[:1, :1])
        bounds[:] = bounds[:1]
        bounds[:, :, :, 0] *= 1000.0
        bounds[:, :, :, 3] = torch.randn(len(bounds), 1, 1, device="cuda").abs() * 2.0 ** -14
        bounds[:, :, 0, 3] *= -1
    for seed, layout in ((6, MODEL), (7, (8, 2, 128, 16)), (8, (4, 2, 80, 16))):
        for types in ((BF16, BF16), (F32, F32), (F32, BF16)):
            _selection(seed, layout, types, [16 * 500, 16 * 40, 16 * 2600], None, 32, 1, 2, near)


def test_small_and_large_numbers():
    for factor_q, factor_b in ((1e-30, 1e-30), (1e18, 1e18), (1e30, 1e-30), (1e-38, 1.0)):
        def scaled(q, bounds, tables):
            q *= factor_q
            bounds *= factor_b
        for layout in (MODEL, (6, 3, 96, 16)):
            _selection(9, layout, (F32, F32), [16 * 90, 16 * 300], None, 20, 1, 1, scaled)
            if factor_q >= 1.0 or factor_b >= 1.0:  # (products that fp32 would lose: the ranks by 64 bits all the same)
                _selection(10, layout, (BF16, BF16), [16 * 90, 16 * 300], None, 20, 1, 1, scaled)


@pytest.mark.parametrize("layout", [MODEL, (6, 3, 96, 16)], ids=str)
def test_bounds_that_are_not_finite_rank_first(layout):
    def odd(q, bounds, tables):
        bounds[tables[1, 7], 0, 1, 3] = float("inf")
        bounds[tables[1, 50], 0, 0, 9] = -float("inf")
        bounds[tables[1, 30], 0, :, 2] = float("nan")
    got = _selection(11, layout, (BF16, BF16), [16 * 20, 16 * 60], None, 6, 1, 1, odd)
    assert {7, 30, 50} <= set(got[1].reshape(layout[1], 6)[0])
    got = _selection(12, layout, (BF16, BF16), [16 * 20, 16 * 60], None, 4, 1, 1, odd)  # three for two places
    assert list(got[1].reshape(layout[1], 4)[0]) == [0, 7, 30, 59]

    def query(q, bounds, tables):
        q[1, 0, 0, 3] = float("nan")
    got = _selection(13, layout, (BF16, BF16), [16 * 20, 16 * 60], None, 6, 1, 1, query)
    assert list(got[1].reshape(layout[1], 6)[0]) == [0, 1, 2, 3, 4, 59]


def test_a_selection_flags_blocks_outside_the_pool_and_ranks_them_last():
    g = _gen(14)
    k = _normal(g, BF16, 40, 4, 2, 256)
    bounds = torch.stack((k.amin(1), k.amax(1)), 2).contiguous()
    tables = np.arange(40)[None].copy()
    tables[0, [5, 9]] = [40, -1]
    q = _normal(g, BF16, 1, 8, 256)
    with pytest.raises(K.DeviceStatusError, match="outside the pool"):
        S.select_blocks(q, bounds, _i32(tables), _i32([640]), 16, 38)
    with pytest.raises(K.DeviceStatusError, match="sequence length"):
        S.select_blocks(q, bounds, _i32(np.arange(40)[None]), _i32([641]), 16, 38)


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32)], ids=str)
def test_rows_of_negative_lengths_see_nothing(types):
    """Down to the smallest integer, whatever the position says."""
    g = _gen(15)
    k = _normal(g, types[1], 40, 16, 2, 128)
    bounds = torch.stack((k.amin(1), k.amax(1)), 2).contiguous()
    tables, lens, pos = _i32(np.tile(np.arange(40), (4, 1))), _i32([-1, -2 ** 31, 0, 600]), _i32([[7], [600], [0], [-2 ** 31]])
    q = _normal(g, types[0], 4, 1, 8, 128)
    chosen = S.select_blocks(q, bounds, tables, lens, 16, 5, positions=pos)
    assert (chosen == -1).all()
    everything = _i32(np.tile(np.arange(40), (4, 1, 2, 1)))
    assert (S.paged_decode_attention_selected(q, k, k, tables, lens, everything, 0.1, positions=pos) == 0).all()


# ------------------------------------------------------------------------------------------------ attention

def _attention(seed, layout, types, lens, positions, entries, scale=None, spoil=True):
    """Random lists: the ends, repeats, columns behind the row, gaps."""
    hq, hkv, d, bs = layout
    act, held = types
    g, rng = _gen(seed), np.random.default_rng(seed)
    tables, pool = _tables(rng, [max(n, 1) for n in lens], bs)
    width = 1 if positions is None else np.asarray(positions).shape[1]
    q = _normal(g, act, len(lens), width, hq, d)
    k, v = _normal(g, held, pool, bs, hkv, d), _normal(g, held, pool, bs, hkv, d)
    chosen = rng.integers(-2, tables.shape[1] + 3, (len(lens), width, hkv, entries))
    for b, n in enumerate(lens):
        chosen[b, :, :, rng.integers(0, entries)] = max(0, (n - 1) // bs)
    used_k, used_v = _f64(k), _f64(v)
    if spoil:  # what no token sees may hold anything
        seen = [max(R.visible(lens, positions, b, t) for t in range(width)) for b in range(len(lens))] if positions is None or width == 1 else lens
        for b, n in enumerate(seen):
            for p in range(max(0, n), tables.shape[1] * bs):
                c = p // bs
                if c < -(-max(lens[b], 1) // bs):
                    k[tables[b, c], p % bs], v[tables[b, c], p % bs] = float("nan"), float("inf")
    scale = d ** -0.5 if scale is None else scale
    shape = (len(lens), width, hkv, entries) if positions is not None else (len(lens), hkv, entries)
    out = S.paged_decode_attention_selected(q if positions is not None else q[:, 0], k, v, _i32(tables), _i32(lens), _i32(chosen.reshape(shape)), scale,
                                            positions=None if positions is None else _i32(positions))
    want, tol = R.attend(_f64(q), used_k, used_v, tables, lens, None if positions is None else np.asarray(positions), chosen, scale, bs,
                         gamma=3 * d * 2.0 ** -23, weight_bits=16)
    got = _f64(out).reshape(want.shape)
    assert (np.abs(got - want) <= tol).all()  # (tokens without keys: zeros)


@pytest.mark.parametrize("layout", LAYOUTS[:6] + LAYOUTS[7:], ids=str)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
def test_attention_over_listed_blocks(layout, types):
    bs = layout[3]
    _attention(1, layout, types, [0, 1, bs, bs + 1, 7 * bs - 1, 40 * bs + 3, 5], None, 9)
    _attention(2, layout, types, [20 * bs + 5, 3, 0], [[20 * bs, 20 * bs + 4, -1], [0, 1, 2], [0, 0, 0]], 5)


@pytest.mark.parametrize("entries", [1, 2, 3, 4, 17, 64, 65, 130])
def test_attention_list_lengths(entries):
    for layout in (MODEL, (32, 8, 128, 32), (16, 2, 64, 16)):
        _attention(3, layout, (BF16, BF16), [2100, 130, 2000], None, entries)


def test_attention_batches_of_all_sizes():
    for rows in (1, 2, 5, 40, 90, 170):
        _attention(rows, MODEL, (BF16, BF16), [17 * (i % 23) for i in range(rows)], None, 6)


def test_attention_over_lists_longer_than_a_warp_looks_ahead():
    """Lists of hundreds of tiles with one CTA for each, so that a warp fetches places several times; most rows see little of theirs."""
    lens = [5 if i % 20 else 700 + i for i in range(160)]
    for layout, types, entries in (((16, 2, 64, 16), (BF16, BF16), 300), ((8, 2, 128, 16), (F32, F32), 150), ((8, 2, 64, 32), (F16, F16), 170)):
        _attention(6, layout, types, lens, None, entries)


def test_blocks_beyond_offsets_of_32_bits():
    """The last blocks of a pool of 2.46e9 numbers of K: appended, selected and attended as the first ones of a small pool."""
    hq, hkv, d, bs, pool = 8, 2, 128, 16, 600_000
    g = _gen(31)
    small = [torch.zeros(40, bs, hkv, d, dtype=BF16, device="cuda") for _ in range(2)] + [torch.zeros(40, hkv, 2, d, dtype=BF16, device="cuda")]
    large = [torch.empty(pool, bs, hkv, d, dtype=BF16, device="cuda") for _ in range(2)] + [torch.empty(pool, hkv, 2, d, dtype=BF16, device="cuda")]
    for t in large:
        t[-40:] = 0
    n = 37 * bs + 5
    q, nk, nv = (_normal(g, BF16, 1, n, h, d) for h in (hq, hkv, hkv))
    one = _normal(g, BF16, 1, hq, d)
    ids, freq = torch.zeros(1, n, dtype=torch.int32, device="cuda"), torch.from_numpy(_freq(32)).cuda()
    outs = []
    for (k, v, b), first in ((small, 0), (large, pool - 40)):
        table = _i32([np.arange(40)[::-1] + first])
        turned = S.rope_kv_append(q, nk, nv, k, v, _i32([np.arange(n)]), table, freq, k_bounds=b, token_row_ids=ids)
        chosen = S.select_blocks(one, b, table, _i32([n]), bs, 9)
        out = S.paged_decode_attention_selected(one, k, v, table, _i32([n]), chosen, d ** -0.5)
        outs.append((turned, chosen, out, k[-40:], v[-40:], b[-40:]))
    for x, y in zip(*outs):
        assert torch.equal(x, y)


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0, 1e-4])
def test_attention_scales(scale):
    for layout, types in ((MODEL, (BF16, BF16)), ((32, 8, 128, 32), (F16, F16)), ((6, 3, 96, 16), (F32, F32))):
        _attention(4, layout, types, [300, 77], None, 7, scale=scale)


def test_attention_flags_blocks_outside_the_pool():
    g = _gen(15)
    k, v = _normal(g, BF16, 4, 16, 2, 256), _normal(g, BF16, 4, 16, 2, 256)
    q = _normal(g, BF16, 1, 8, 256)
    chosen = _i32([[[0, 1, 2], [0, 1, 2]]])
    for bad in (4, -1, 2 ** 31 - 1):
        with pytest.raises(K.DeviceStatusError, match="outside the pool"):
            S.paged_decode_attention_selected(q, k, v, _i32([[0, bad, 2]]), _i32([48]), chosen, 0.1)
    with pytest.raises(K.DeviceStatusError, match="sequence length"):
        S.paged_decode_attention_selected(q, k, v, _i32([[0, 1, 2]]), _i32([49]), chosen, 0.1)


# ------------------------------------------------------------------------------------------------ refusals and empty calls

def _small():
    g = _gen(20)
    k, v = _normal(g, BF16, 6, 16, 2, 64), _normal(g, BF16, 6, 16, 2, 64)
    return dict(k=k, v=v, b=torch.stack((k.amin(1), k.amax(1)), 2).contiguous(), q=_normal(g, BF16, 2, 1, 8, 64), kv=_normal(g, BF16, 2, 1, 2, 64),
                pos=_i32([[3], [20]]), tab=_i32([[0, 1, 2], [3, 4, 5]]), lens=_i32([4, 21]), sel=_i32(np.zeros((2, 1, 2, 2))), freq=torch.ones(32, device="cuda"))


def _bad(s, **change):
    return dict(s, **{k: f(s[k]) for k, f in change.items()})


@pytest.mark.parametrize("change,match", [
    (dict(k=lambda t: t.half()), "one shape, dtype"), (dict(k=lambda t: t[:, :, :, :20].contiguous(), v=lambda t: t[:, :, :, :20].contiguous()), "multiple of 8"),
    (dict(k=lambda t: t.transpose(1, 2)), "NHD"), (dict(kv=lambda t: t[..., :32]), "heads those of the cache"), (dict(q=lambda t: t.float()), "same dtype"),
    (dict(q=lambda t: t[:1]), "query must have shape"), (dict(b=lambda t: t.float()), "cache's dtype"), (dict(b=lambda t: t[:5].contiguous()), "k_bounds"),
    (dict(b=lambda t: t.transpose(0, 1)), "k_bounds must be contiguous"), (dict(pos=lambda t: t.long()), "int32"), (dict(pos=lambda t: t[:1]), "positions must have shape"),
    (dict(tab=lambda t: t[:1]), "batch dimensions"), (dict(tab=lambda t: t[0]), "2D"), (dict(tab=lambda t: t[:, :0]), "not empty"), (dict(lens=lambda t: t[:1]), "seq_lens"),
    (dict(freq=lambda t: t.double()), "inv_freq"), (dict(freq=lambda t: torch.ones(33, device="cuda")), "inv_freq")])
def test_append_refusals(change, match):
    s = _bad(_small(), **change)
    with pytest.raises(ValueError, match=match):
        S.rope_kv_append(s["q"], s["kv"], s["kv"], s["k"], s["v"], s["pos"], s["tab"], s["freq"], k_bounds=s["b"], seq_lens=s["lens"])


@pytest.mark.parametrize("change,match", [
    (dict(q=lambda t: t[..., :32]), "head_dim must match"), (dict(q=lambda t: t[:, :, :3]), "divisible"), (dict(q=lambda t: t.double()), "dtype"),
    (dict(q=lambda t: t[0, 0]), "q must have shape"), (dict(b=lambda t: t[:, :, :1]), "k_bounds"), (dict(tab=lambda t: t[:1]), "block_table"),
    (dict(lens=lambda t: t.long()), "int32"), (dict(pos=lambda t: t[:1]), "positions"),
    (dict(tab=lambda t: torch.zeros(2, S.MOST_COLUMNS + 1, dtype=torch.int32, device="cuda")), "columns")])
def test_selection_refusals(change, match):
    s = _bad(_small(), **change)
    with pytest.raises(ValueError, match=match):
        S.select_blocks(s["q"], s["b"], s["tab"], s["lens"], 16, 2, positions=s["pos"])


@pytest.mark.parametrize("budget,first,last,block", [(0, 0, 0, 16), (2, 2, 1, 16), (2, -1, 1, 16), (2, 1, 2 ** 62, 16), (2, 2 ** 62, 2 ** 62, 16), (2, 1, 1, 0)])
def test_selection_refuses_budgets(budget, first, last, block):
    s = _small()
    with pytest.raises(ValueError, match="budget|block_size"):
        S.select_blocks(s["q"], s["b"], s["tab"], s["lens"], block, budget, first=first, last=last)


@pytest.mark.parametrize("change,match", [
    (dict(sel=lambda t: t[:, 0]), "selected"), (dict(sel=lambda t: t[:1]), "selected"), (dict(sel=lambda t: t.long()), "int32"), (dict(k=lambda t: t.float()), "one shape"),
    (dict(q=lambda t: t[..., :32]), "head_dim"), (dict(q=lambda t: t[:, :, :3]), "divisible"), (dict(lens=lambda t: t[:1]), "seq_lens")])
def test_attention_refusals(change, match):
    s = _bad(_small(), **change)
    with pytest.raises(ValueError, match=match):
        S.paged_decode_attention_selected(s["q"], s["k"], s["v"], s["tab"], s["lens"], s["sel"], 0.1)


def test_empty_batches_and_lists():
    s = _small()
    none = _i32(np.zeros((0, 3)))
    assert S.select_blocks(s["q"][:0], s["b"], none, s["lens"][:0], 16, 2).shape == (0, 1, 2, 2)
    assert S.paged_decode_attention_selected(s["q"][:0], s["k"], s["v"], none, s["lens"][:0], s["sel"][:0], 0.1).shape == (0, 1, 512)
    assert S.rope_kv_append(s["q"][:0], s["kv"][:0], s["kv"][:0], s["k"], s["v"], s["pos"][:0], s["tab"], s["freq"]).shape == (0, 1, 8, 64)
    assert not S.paged_decode_attention_selected(s["q"], s["k"], s["v"], s["tab"], s["lens"], s["sel"][..., :0], 0.1).any()
    assert not S.paged_decode_attention_selected(s["q"], s["k"], s["v"], s["tab"][:, :0], _i32([0, 0]), s["sel"], 0.1).any()
    assert (S.select_blocks(s["q"], s["b"], s["tab"][:, :0], _i32([0, 0]), 16, 2) == -1).all()
    before = s["b"].clone()
    S.rope_kv_append(None, s["kv"], s["kv"], s["k"], s["v"], s["pos"], s["tab"], None, k_bounds=s["b"], seq_lens=_i32([0, -5]))
    assert torch.equal(s["b"], before)


def test_metadata_that_is_not_contiguous_is_read_as_it_is():
    g = _gen(21)
    s = _small()
    wide = torch.zeros(2, 6, dtype=torch.int32, device="cuda")
    wide[:, ::2] = s["tab"]
    q = _normal(g, BF16, 2, 8, 2, 64).transpose(1, 2)  # [2, 2, 8, 64]
    pos = _i32([[3, 3], [19, 20]])
    a = S.select_blocks(q, s["b"], wide[:, ::2], s["lens"], 16, 1, positions=pos, first=0, last=0)
    b = S.select_blocks(q.contiguous(), s["b"], s["tab"], s["lens"], 16, 1, positions=pos, first=0, last=0)
    assert torch.equal(a, b)
    x = S.paged_decode_attention_selected(q, s["k"], s["v"], wide[:, ::2], s["lens"], a, 0.1, positions=pos)
    y = S.paged_decode_attention_selected(q.contiguous(), s["k"], s["v"], s["tab"], s["lens"], b, 0.1, positions=pos)
    assert torch.equal(x, y)
