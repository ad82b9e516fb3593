"""Attention over listed blocks: the accuracy of weights and queries, and keys of blocks that are not in the pool."""

import numpy as np
import pytest
import torch

import selective_reference as R
from nano_vllm_jax_b200.kernels import paged_kv as K
from nano_vllm_jax_b200.kernels import selective_kv as S
from test_gpu_selective_kv import BF16, F16, F32, MODEL, _f64, _gen, _i32, _normal
from test_gpu_selection_range import unread_status  # noqa: F401

pytestmark = pytest.mark.gpu

ATTENTION = [(MODEL, BF16), ((8, 1, 128, 16), BF16), ((12, 1, 64, 16), BF16), ((6, 3, 96, 16), BF16), (MODEL, F16), ((16, 1, 128, 16), F16), (MODEL, F32),
             ((8, 1, 64, 16), F32), ((4, 1, 40, 7), BF16)]


@pytest.mark.parametrize("layout,held", ATTENTION, ids=str)
def test_keys_of_blocks_outside_the_pool_are_left_out(layout, held, unread_status):
    hq, hkv, d, bs = layout
    g, rng = _gen(25), np.random.default_rng(25)
    k, v = _normal(g, held, 12, bs, hkv, d), _normal(g, held, 12, bs, hkv, d)
    q = _normal(g, held, 3, 1, hq, d)
    tables = np.tile(rng.permutation(12)[:10], (3, 1))
    tables[0, [0, 4]], tables[1, 7], tables[2] = [12, -1], 2 ** 31 - 1, -2 ** 31
    lens = np.array([10 * bs, 10 * bs + 1, 10 * bs])  # the second beyond its table: clipped
    chosen = np.tile(np.arange(10), (3, 1, hkv, 1))
    out = S.paged_decode_attention_selected(q, k, v, _i32(tables), _i32(lens), _i32(chosen), d ** -0.5, positions=_i32([[2 ** 31 - 1]] * 3))
    there = np.where((tables >= 0) & (tables < 12), np.arange(10), -1)[:, None, None].repeat(hkv, 2)
    want, tol = R.attend(_f64(q), _f64(k), _f64(v), np.clip(tables, 0, 11), np.minimum(lens, 10 * bs), None, there, d ** -0.5, bs, gamma=3 * d * 2.0 ** -23,
                         weight_bits=16)
    assert (np.abs(_f64(out).reshape(want.shape) - want) <= tol).all() and not out[2].any()
    with pytest.raises(K.DeviceStatusError, match="outside the pool|sequence length"):
        K.check_device_status()


def _cut_weights(w, terms):
    """Weights as the sum of `terms` bf16 numbers."""
    rest, total = w.astype(np.float32), np.zeros_like(w)
    for _ in range(terms):
        part = torch.from_numpy(rest).bfloat16().float().numpy()
        rest, total = rest - part, total + part
    return total


@pytest.mark.parametrize("layout,held", ATTENTION, ids=str)
def test_weights_are_as_accurate_as_stated(layout, held):
    """Sixteen keys (a block of seven: seven) whose scores are exact, V one-hot, so that every output is one weight over their sum.

    Scores are whole numbers up to 64 in size, times 2^-6: up to 1.45 in log2 units.  In units of 2^-22 of a weight: a score and the maximum are rounded once each,
    their factor once, their difference (up to 2.9) once, 0.95 in all, and the exponential is good to 1; both for the weight and for the sum, 3.9.  The sum of a
    lane's keys and over the lanes is four additions, 1; the terms of a weight are added with a place of 2^-23 each, 1.5; a shared column, the reciprocal
    and its product 0.75.  7.2 in all: 8.5 are allowed.  f16 weights stand 2^7 higher, so that the difference goes up to 9.9 (2.1 more), and end after 22 bits (1); on the CUDA
    cores two warps are joined by another exponential (2.7 more, without the terms' 1.5): 11.  Two bf16 terms instead of three leave up to 2^-18, 16.
    """
    hq, hkv, d, bs = layout
    n, rows, group = min(bs, 16), 40, hq // hkv
    rng = np.random.default_rng(26)
    q, k = rng.integers(-1, 2, (rows, hq, d)), rng.integers(-2, 3, (rows, bs, hkv, d))
    k[..., 32:] = 0
    v = np.zeros((rows, bs, hkv, d))
    for p in range(n):
        v[:, p, :, p] = 1.0
    act = BF16 if held != F16 else F16
    out = S.paged_decode_attention_selected(torch.from_numpy(q).cuda().to(act), torch.from_numpy(k).cuda().to(held), torch.from_numpy(v).cuda().to(held),
                                            _i32(np.arange(rows)[:, None]), _i32([n] * rows), _i32(np.zeros((rows, hkv, 1))), 2.0 ** -6)
    s = np.einsum("rhgd,rphd->rhgp", q.reshape(rows, hkv, group, d), k[:, :n]) * 2.0 ** -6
    assert np.abs(s).max() <= 1.0
    w = np.exp(s - s.max(-1, keepdims=True))
    want = w / w.sum(-1, keepdims=True)
    got = _f64(out).reshape(rows, hkv, group, d)
    tiles = held == BF16 and bs % 16 == 0
    tolerance = (8.5 if tiles else 11) * 2.0 ** -22
    assert not got[..., n:].any()
    assert (np.abs(got[..., :n] - want) <= tolerance * want).all()
    if tiles:  # the same with a term less would not pass
        lost, kept = (_cut_weights(w, terms) / w.sum(-1, keepdims=True) for terms in (2, 3))
        assert (np.abs(lost - want) > tolerance * want).any() and (np.abs(kept - want) <= tolerance * want).all()


@pytest.mark.parametrize("layout,held", [x for x in ATTENTION if x[1] != F32], ids=str)
def test_queries_of_24_bits_keep_them(layout, held):
    """f32 queries over 16-bit caches, K one-hot: a score is one number of the query, up to 8 in size.

    In units of 2^-22 of a weight: its terms are added with a place of 2^-23 of 8 each, 8, and so are the maximum's, 16; rounding of both in log2 units (up to 11.6) 2.8, their
    factor 2, their difference (up to 23) 2.8: 23.6, for the weight and for the sum, 47.  With what follows (8.5) 56; 58 are allowed.  Two terms for three
    leave 8 * 2^-15, 1024.  Weights over f16 caches end at 2^-24 where the largest is 2^7: 2^-31 of the largest besides.
    """
    hq, hkv, d, bs = layout
    n, rows = min(bs, 16), 20
    g = _gen(27)
    q = (torch.rand(rows, hq, d, generator=g, device="cuda") * 16 - 8).float()
    pages = torch.zeros(1, bs, hkv, d, device="cuda")
    for p in range(n):
        pages[0, p, :, p] = 1.0
    pages = pages.to(held)
    out = S.paged_decode_attention_selected(q, pages, pages, _i32(np.zeros((rows, 1))), _i32([n] * rows), _i32(np.zeros((rows, hkv, 1))), 1.0)
    want = torch.softmax(q[..., :n].double(), -1)
    got = out.double()[..., :n]
    assert ((got - want).abs() <= 58 * 2.0 ** -22 * want + (2.0 ** -31 if held == F16 else 0.0)).all()
