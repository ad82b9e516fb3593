"""The layout of a packed step made on the device, against the same walk in Python; and the 8-bit cache's operators in a run, as a server uses them."""

import numpy as np
import pytest
import torch

import quantized_reference as R
from nano_vllm_jax_b200.backends import B200Backend
from nano_vllm_jax_b200.engine.device_blocks import DeviceBlockPool
from nano_vllm_jax_b200.engine.resident_decode import CapturedStep, ResidentDecodeMetadata
from nano_vllm_jax_b200.kernels import paged_kv as K
from nano_vllm_jax_b200.kv_cache import AttentionMetadata, KVCacheSpec

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _walk(cached, new, tables, free, head, bs, bucket):
    """The same in Python; `tables` is changed in place."""
    positions, ids, slots, qsl = [], [], [], [0]
    for r, (c, n) in enumerate(zip(cached, new)):
        for b in range(-(-c // bs), -(-(c + n) // bs)):
            tables[r, b] = free[head]
            head += 1
        for p in range(c, c + n):
            positions.append(p)
            ids.append(r)
            slots.append(tables[r, p // bs] * bs + p % bs)
        qsl.append(len(positions))
    pad = bucket - len(positions)
    return (np.array([positions + [0] * pad]), np.array([ids + [0] * pad]), np.array([slots + [-1] * pad]), np.array(qsl),
            np.array(cached) + np.array(new), np.array([head]))


def _case(rng, rows, most_cached, most_new, bs):
    cached, new = rng.integers(0, most_cached + 1, rows), rng.integers(0, most_new + 1, rows)
    width = -(-(most_cached + most_new) // bs) + 2
    tables = rng.integers(0, 1000, (rows, width))
    need = int((-(-(cached + new) // bs) + (-cached // bs)).sum())
    return cached, new, tables, rng.permutation(need + 30), need


@pytest.mark.parametrize("rows,most_cached,most_new,bs,pad", [(1, 0, 1, 16, 0), (1, 40, 30, 16, 5), (7, 100, 50, 16, 3), (256, 500, 1, 16, 0), (513, 33, 9, 1, 2),
                                                             (3, 0, 3000, 32, 40), (1025, 70, 20, 7, 1), (40, 64, 64, 64, 0), (5, 20, 0, 16, 4)])
def test_layout_is_the_walk_s(rows, most_cached, most_new, bs, pad):
    rng = np.random.default_rng(rows)
    cached, new, tables, free, need = _case(rng, rows, most_cached, most_new, bs)
    bucket = int(new.sum()) + pad
    got_tables = _i32(tables)
    got = K.build_packed_layout(_i32(cached), _i32(new), got_tables, _i32(free), _i32([11]), bs, bucket)
    want = _walk(cached, new, tables, free, 11, bs, bucket)
    for name, g, w in zip(got._fields, got, want):
        assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), w), name
    assert np.array_equal(got_tables.cpu().numpy(), tables)


def test_the_most_rows_there_can_be():
    rows, bs = 16384, 16
    rng = np.random.default_rng(1)
    cached, new = rng.integers(0, 60, rows), rng.integers(0, 3, rows)
    tables, free = rng.integers(0, 1000, (rows, 4)), rng.permutation(rows)
    got_tables = _i32(tables)
    got = K.build_packed_layout(_i32(cached), _i32(new), got_tables, _i32(free), _i32([0]), bs, int(new.sum()))
    for g, w in zip(got, _walk(cached, new, tables, free, 0, bs, int(new.sum()))):
        assert np.array_equal(g.cpu().numpy(), w)
    assert np.array_equal(got_tables.cpu().numpy(), tables)
    with pytest.raises(K.NvjError):
        K.build_packed_layout(_i32(np.zeros(16385)), _i32(np.zeros(16385)), _i32(np.zeros((16385, 4))), _i32([0]), _i32([0]), bs, 0)


def test_no_rows_and_no_tokens():
    none = _i32(np.zeros(0))
    got = K.build_packed_layout(none, none, _i32(np.zeros((0, 4))), _i32([5]), _i32([3]), 16, 6)
    assert got.query_start_loc.tolist() == [0] and got.free_head.tolist() == [3] and got.seq_lens.numel() == 0
    assert got.slot_mapping.tolist() == [[-1] * 6] and not got.positions.any() and not got.token_row_ids.any()
    got = K.build_packed_layout(_i32([4, 0]), _i32([0, 0]), _i32([[1], [2]]), none, _i32([0]), 16, 0)
    assert got.query_start_loc.tolist() == [0, 0, 0] and got.seq_lens.tolist() == [4, 0] and got.positions.shape == (1, 0)


def test_what_does_not_fit_is_flagged_and_left_out(monkeypatch):
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")

    def word(code):
        with pytest.raises(K.DeviceStatusError, match=f"device status {code} "):
            K.check_device_status()

    tables = _i32(np.full((4, 2), 77))
    got = K.build_packed_layout(_i32([30, -1, 5, 40]), _i32([3, 4, 2, 1]), tables, _i32(range(9)), _i32([0]), 16, 4)
    word(4)  # a row past its table, a negative length, a row that was past it before: row 2 alone is served
    assert got.query_start_loc.tolist() == [0, 0, 0, 2, 2] and got.positions.tolist() == [[5, 6, 0, 0]]
    assert got.slot_mapping.tolist() == [[77 * 16 + 5, 77 * 16 + 6, -1, -1]] and got.free_head.tolist() == [0] and bool((tables == 77).all())
    tables = _i32(np.zeros((2, 3)))
    got = K.build_packed_layout(_i32([0, 0]), _i32([20, 20]), tables, _i32([8, 9, 10]), _i32([0]), 16, 40)
    word(2)  # the list ends in the second row
    assert tables.tolist() == [[8, 9, 0], [10, -1, 0]] and got.free_head.tolist() == [4]
    assert got.slot_mapping[0, 35:].tolist() == [10 * 16 + 15] + [-1] * 4
    for head in (-5, 3, 1 << 30):
        got = K.build_packed_layout(_i32([0]), _i32([2]), _i32([[0]]), _i32([8, 9, 10]), _i32([head]), 16, 2)
        word(2)
        assert got.slot_mapping.tolist() == [[-1, -1]]
    got = K.build_packed_layout(_i32([0, 0]), _i32([3, 4]), _i32([[0], [0]]), _i32([8, 9]), _i32([0]), 16, 5)
    word(4)  # a bucket too small
    assert got.query_start_loc.tolist() == [0, 3, 7] and got.slot_mapping.tolist() == [[128, 129, 130, 144, 145]]


def test_ids_whose_slots_pass_32_bits_have_none():
    # (1 << 28) * 16 is 0 in 32 bits: the slot of another row's token
    tables = _i32([[1 << 28, 0], [7, 0], [(1 << 27) - 1, 0]])
    got = K.build_packed_layout(_i32([5, 16, 14]), _i32([2, 1, 2]), tables, _i32([(1 << 31) - 1]), _i32([0]), 16, 5)
    assert got.slot_mapping.tolist() == [[-1, -1, -1, (1 << 31) - 2, (1 << 31) - 1]] and tables[1, 1].item() == (1 << 31) - 1


def test_wrapper_refuses_what_does_not_fit_together():
    good = dict(cached_lens=_i32([1, 2]), new_lens=_i32([1, 1]), block_tables=_i32([[0], [1]]), free_blocks=_i32([4]), free_head=_i32([0]), block_size=16,
                token_bucket=4)
    for change in ({"cached_lens": good["cached_lens"].long()}, {"new_lens": _i32([1])}, {"block_tables": _i32([0, 1])}, {"free_head": _i32([0, 1])},
                   {"free_blocks": _i32([[4]])}, {"block_size": 0}, {"token_bucket": -1}, {"block_tables": _i32(np.zeros((2, 4)))[:, ::2]},
                   {"free_head": torch.zeros(1, dtype=torch.int32)}):
        with pytest.raises(ValueError):
            K.build_packed_layout(**(good | change))


def test_captured_layouts_follow_their_inputs():
    cached, new, tables, _, _ = _case(np.random.default_rng(5), 20, 50, 30, 16)
    c, n, t, f, h = _i32(cached), _i32(new), _i32(tables), _i32(np.arange(200)), _i32([2])  # 20 rows need 60 ids at most
    step = CapturedStep(lambda: K.build_packed_layout(c, n, t, f, h, 16, 700))
    step.capture()
    for seed in range(3):
        rng = np.random.default_rng(100 + seed)
        cached, new, tables, _, _ = _case(rng, 20, 50, 30, 16)
        free = rng.permutation(200)
        c.copy_(_i32(cached)), n.copy_(_i32(new)), t.copy_(_i32(tables)), f.copy_(_i32(free)), h.fill_(seed)
        got = step.replay()
        for g, w in zip(got, _walk(cached, new, tables, free, seed, 16, 700)):
            assert np.array_equal(g.cpu().numpy(), w)
        assert np.array_equal(t.cpu().numpy(), tables)


def test_resident_rows_take_their_next_blocks_from_the_pool():
    meta = ResidentDecodeMetadata(3, 4, 16)
    meta.load(np.array([[5, 0], [6, 7], [0, 0]]), np.array([16, 20, 0]))
    pool = DeviceBlockPool([30, 31, 32], 16)
    meta.reserve(pool)
    assert meta.block_tables.tolist() == [[5, 30, 0, 0], [6, 7, 0, 0], [0, 0, 0, 0]] and pool.free_head.tolist() == [1]
    meta.reserve(pool)  # lengths as they were: the entry is the row's next block again
    assert meta.block_tables[0].tolist() == [5, 31, 0, 0]
    pool.reset([40])
    assert pool.free_head.tolist() == [0]


def test_captured_decode_steps_take_new_blocks_at_every_replay():
    bs = 4
    lens = np.array([5, 8, 0, 1, 16])
    meta = ResidentDecodeMetadata(5, 8, bs)
    tables = np.zeros((5, 8), np.int64)
    for r, n in enumerate(lens):
        tables[r, : -(-n // bs)] = 100 + 10 * r + np.arange(-(-n // bs))
    meta.load(tables, lens)
    pool = DeviceBlockPool(range(40, 60), bs)
    ids = iter(range(40, 60))

    def step():
        meta.reserve(pool)
        meta.advance()

    def walk(ids):
        for r in range(5):
            if lens[r] > 0:
                if lens[r] % bs == 0:
                    tables[r, lens[r] // bs] = next(ids)
                lens[r] += 1

    def same():
        return np.array_equal(meta.seq_lens.cpu().numpy(), lens) and np.array_equal(meta.block_tables.cpu().numpy(), tables)

    captured = CapturedStep(step)
    captured.capture()  # (runs it once)
    walk(ids)
    for _ in range(6):
        captured.replay()
        walk(ids)
    assert same() and pool.free_head.tolist() == [next(ids) - 40]
    pool.reset([70, 71, 72, 73, 74])  # the ids that are free now, into the list that the step was captured with
    ids = iter([70, 71, 72, 73, 74])
    for _ in range(4):
        captured.replay()
        walk(ids)
    assert same()
    K.check_device_status()


def test_a_pool_s_list_that_is_shorter_than_it_was_ends_where_it_ends(monkeypatch):
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")
    pool = DeviceBlockPool(range(10), 16)
    pool.reset([3, 4])
    tables = _i32(np.zeros((3, 2)))
    lay = pool.extend(tables, _i32([0, 0, 0]), _i32([1, 1, 1]), 3)
    assert tables.tolist() == [[3, 0], [4, 0], [-1, 0]] and lay.slot_mapping.tolist() == [[48, 64, -1]] and pool.free_head.tolist() == [3]
    with pytest.raises(K.DeviceStatusError, match="device status 2 "):
        K.check_device_status()
    pool.reset(list(range(20, 40)))  # more than there ever were
    assert pool.extend(tables, _i32([0, 0, 0]), _i32([1, 1, 1]), 3).slot_mapping.tolist() == [[320, 336, 352]]
    K.check_device_status()


# ------------------------------------------------------------------------------------------------ the operators in a run

@pytest.mark.parametrize("heads", [(8, 2, 256, 16), (8, 4, 64, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompts_in_chunks_and_then_decode_steps(heads, dtype):
    """Layout, append and attention through the backend, two layers: three prompts in two packed steps, a mixed step, decode steps and a
    verification of four tokens; every step's cache bit for bit and every output against 64-bit attention over what the cache holds."""
    hq, hkv, d, bs = heads
    layers, rows, width = 2, 4, 12
    rng = np.random.default_rng(7)
    backend = B200Backend()
    cache = backend.allocate_kv_cache(KVCacheSpec(layers, 60, bs, hkv, d, torch.float8_e4m3fn), rows, width)
    pool = DeviceBlockPool(rng.permutation(60), bs)
    tables = torch.zeros((rows, width), dtype=torch.int32, device="cuda")
    state = [[(t[i].view(torch.uint8).cpu().numpy().copy(), s[i].double().cpu().numpy()) for t, s in ((cache.k_cache, cache.k_scale), (cache.v_cache, cache.v_scale))]
             for i in range(layers)]
    lens = np.zeros(rows, np.int64)
    scale = d ** -0.5

    def normal(*shape):
        return torch.from_numpy(rng.standard_normal(shape)).to(dtype).cuda()

    def check(layer, out, q, before, new, table):
        q64, got = q.double().cpu().numpy().reshape(-1, hq, d), out.double().cpu().numpy().reshape(-1, hq, d)
        at = 0
        for r in range(rows):
            n = int(new[r])
            if n == 0:
                continue
            k, v = (R.gather(codes, s, table[r], before[r] + n) for codes, s in state[layer])
            seen = np.arange(before[r] + n)[None] <= (before[r] + np.arange(n))[:, None]
            want = R.attend(q64[at: at + n], k, v, seen, scale)
            assert np.abs(got[at: at + n] - want).max() <= R.tolerance(q64[at: at + n], k, v, scale, 16)
            at += n

    def remember(layer, k, v, slots):
        for (codes, s), x in zip(state[layer], (k, v)):
            R.append(codes, s, x.double().cpu().numpy().reshape(-1, hkv, d), [None if i < 0 else (int(i) // bs, int(i) % bs) for i in slots], bs)
        for (codes, s), numbers, scales in zip(state[layer], (cache.k_cache, cache.v_cache), (cache.k_scale, cache.v_scale)):
            assert np.array_equal(numbers[layer].view(torch.uint8).cpu().numpy(), codes) and np.array_equal(scales[layer].double().cpu().numpy(), s)

    for new in ([70, 33, 0, 100], [30, 0, 90, 1], [1, 1, 1, 1]):  # packed steps: chunks, a mixed one, a decode step as a packed batch
        bucket = sum(new) + 5
        lay = pool.extend(tables, _i32(lens), _i32(new), bucket)
        md = backend.build_attention_metadata(lay.positions, tables, lay.seq_lens, bs, True, query_start_loc=lay.query_start_loc,
                                              token_row_ids=lay.token_row_ids, query_lens_host=new)
        assert torch.equal(md.slot_mapping[0, : sum(new)], lay.slot_mapping[0, : sum(new)])
        for layer in range(layers):
            q, k, v = normal(1, bucket, hq, d), normal(1, bucket, hkv, d), normal(1, bucket, hkv, d)
            same, out = backend.write_kv_and_attention(layer, q, k, v, cache, md, bs, scale, hq // hkv, True)
            assert same is cache and not out[0, sum(new):].any()
            remember(layer, k, v, lay.slot_mapping[0].tolist())
            check(layer, out[0, : sum(new)], q[0, : sum(new)], lens, new, tables.cpu().numpy())
        lens += new
    for tokens in (1, 1, 4):  # decode steps, and a verification
        new = [tokens, tokens, tokens, 0]
        lay = pool.extend(tables, _i32(lens), _i32(new), 3 * tokens)
        table = tables[:3].contiguous()
        md = backend.build_attention_metadata(lay.positions.view(3, tokens), table, lay.seq_lens[:3].contiguous(), bs, False)
        if tokens > 1:
            md.query_start_loc = _i32(np.arange(4) * tokens)
        for layer in range(layers):
            q, k, v = normal(3, tokens, hq, d), normal(3, tokens, hkv, d), normal(3, tokens, hkv, d)
            _, out = backend.write_kv_and_attention(layer, q, k, v, cache, md, bs, scale, hq // hkv, False)
            remember(layer, k, v, lay.slot_mapping[0].tolist())
            check(layer, out, q, lens, new, tables.cpu().numpy())
        lens += new
    # a rectangular prefill: more query tokens than the decode kernel is for, over rows that are cached already
    md = AttentionMetadata(None, tables, _i32(lens), _i32(np.arange(5) * 20), 80, 0, _i32(lens[:, None] - 20 + np.arange(20)))
    q = normal(rows, 20, hq, d)
    out = backend.attention(0, q, cache, md, bs, scale, hq // hkv, True)
    check(0, out, q, lens - 20, [20] * 4, tables.cpu().numpy())
    K.check_device_status()


def test_the_backend_asks_for_positions():
    backend = B200Backend()
    cache = backend.allocate_kv_cache(KVCacheSpec(1, 4, 16, 2, 256, torch.float8_e4m3fn), 1, 1)
    md = AttentionMetadata(_i32([[0]]), _i32([[0]]), _i32([1]), _i32([0, 1]), 0, 1, None)
    x = torch.zeros(1, 1, 2, 256, device="cuda")
    with pytest.raises(ValueError, match="positions"):
        backend.write_kv(0, x, x, cache, md)
    with pytest.raises(ValueError, match="positions"):
        backend.attention(0, torch.zeros(1, 1, 8, 256, device="cuda"), cache, md, 16, 1.0, 4, False)
