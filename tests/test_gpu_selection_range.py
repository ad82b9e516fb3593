"""Selection of blocks where scores leave fp32 or differ by less than it tells apart, or blocks of a row are not in the pool."""

import numpy as np
import pytest
import torch

import selective_reference as R
from nano_vllm_jax_b200.kernels import paged_kv as K
from nano_vllm_jax_b200.kernels import selective_kv as S
from test_gpu_selective_kv import BF16, F16, F32, MODEL, _f64, _gen, _i32, _normal, _selection

pytestmark = pytest.mark.gpu

# the forms of the selection: tensor-core tiles of one and two column tiles, two terms of the queries, and the CUDA cores (f32 bounds, many heads)
FORMS = [(MODEL, (BF16, BF16)), ((6, 3, 96, 16), (BF16, BF16)), ((12, 1, 128, 16), (F32, BF16)), ((6, 2, 64, 16), (F16, BF16)), (MODEL, (F32, F32)),
         ((6, 3, 96, 16), (F32, F32)), ((34, 2, 64, 16), (BF16, BF16))]


@pytest.fixture
def unread_status(monkeypatch):
    """The status word stays unread, so that a flagged call returns what it has made."""
    monkeypatch.setenv("NVJ_CHECK_STATUS", "0")
    yield
    try:
        K.check_device_status()
    except K.DeviceStatusError:
        pass


LENS = [16 * 25, 16 * 90, 16 * 300, 16 * 1100]  # blocks in doubt: few, and more than a warp ranks


def _beyond(q, bounds, tables):
    """Scores of both signs up to 1e41, of which f32 holds a part."""
    q *= 1e20
    bounds *= (10.0 ** (torch.arange(len(bounds), device="cuda") % 7 + 13.0)).to(bounds.dtype)[:, None, None, None]


def _below(q, bounds, tables):
    """Every score below what f32 holds: negative bounds under positive queries."""
    q[:] = q.abs() * 1e20
    bounds[:] = -(bounds.abs() + 1.0) * 1e20
    bounds[:] = bounds.sort(dim=2).values


def _partial(q, bounds, tables):
    """Sums that pass through numbers beyond f32 on their way to one that it holds: 1e39 and -1e39 beside numbers of 1e36."""
    q[:] = q.abs() * 1e18
    bounds *= 1e18
    q[..., ::8], q[..., 5::8] = 1e20, 1e20
    bounds[..., ::8], bounds[..., 5::8] = 1e19, -1e19


def _mixed(q, bounds, tables):
    """The same beside bounds that are not finite, which rank first."""
    _beyond(q, bounds, tables)
    bounds[tables[1, 7], :, 1, 3] = float("inf")
    bounds[tables[1, 50], :, 0, 2] = -float("inf")
    bounds[tables[2, 30], :, :, 1] = float("nan")


@pytest.mark.parametrize("layout,types", FORMS, ids=str)
@pytest.mark.parametrize("change", [_beyond, _below, _partial, _mixed])
def test_scores_that_f32_does_not_hold_rank_by_their_value(layout, types, change):
    if F16 in types:
        pytest.skip("queries of 1e18")
    _selection(21, layout, types, LENS, None, 20, 1, 2, change)


@pytest.mark.parametrize("layout,types", FORMS, ids=str)
@pytest.mark.parametrize("below", [False, True], ids=["scores of one size", "scores below f32"])
def test_blocks_outside_the_pool_rank_behind_every_other(layout, types, below, unread_status):
    if below and F16 in types:
        pytest.skip("queries of 1e20")
    hq, hkv, d, bs = layout
    g = _gen(22)
    k = _normal(g, types[1], 40, 4, hkv, d)
    k[0] *= 100.0  # (what a block that is not there must not be taken for)
    bounds = torch.stack((k.amin(1), k.amax(1)), 2).contiguous()
    q = _normal(g, types[0], 2, 1, hq, d)
    if below:
        _below(q, bounds, None)
    tables = np.tile(np.arange(40), (2, 1))
    held = tables.copy()
    tables[:, [5, 9, 22]] = [40, -1, 2 ** 31 - 1]
    lens = np.array([40 * bs, 40 * bs + 7])  # the second beyond its table: clipped
    for budget in (39, 38, 37, 20, 4):
        got = S.select_blocks(q, bounds, _i32(tables), _i32(lens), bs, budget, positions=_i32([[2 ** 31 - 1]] * 2), first=1, last=2).cpu().numpy()
        for b in range(2):
            for h in range(hkv):
                group = hq // hkv
                score = R.scores(_f64(q)[b, 0, h * group:(h + 1) * group], _f64(bounds)[held[b], h])
                score[[5, 9, 22]] = -np.inf
                assert np.array_equal(got[b, 0, h], R.choose(score, 40, budget, 1, 2)), (budget, b, h)
    with pytest.raises(K.DeviceStatusError, match="outside the pool|sequence length"):
        K.check_device_status()


@pytest.mark.parametrize("layout", [(4, 2, 64, 16), (8, 2, 128, 16), MODEL, (12, 1, 96, 16)], ids=str)
def test_queries_of_the_largest_rest_over_bf16_bounds(layout):
    """Queries of which two cut terms leave the most, 255 * 2^-23 of them, in half of the dims, exact ones in the others; blocks whose scores differ by less."""
    worst = torch.tensor([0x3F8080FF], dtype=torch.int32).view(F32).item()

    def near(q, bounds, tables):
        sign = torch.where(torch.rand_like(q) < 0.5, -1.0, 1.0)
        q[:] = sign * worst
        q[..., ::2] = sign[..., ::2]
        of = torch.arange(len(bounds), device="cuda")
        bounds[:] = 0.0
        bounds[of, :, 0, :], bounds[of, :, 1, :] = -1.0, 1.0  # every block the same, then one unit moved between a dim with a rest and one without
        where = 2 * (of % (layout[2] // 2))
        bounds[of, :, 0, where], bounds[of, :, 1, where] = -1.0 - 2.0 ** -7, 1.0 + 2.0 ** -7
        other = 2 * ((of // 7) % (layout[2] // 2)) + 1
        bounds[of, :, 0, other], bounds[of, :, 1, other] = -1.0 + 2.0 ** -7, 1.0 - 2.0 ** -7
    for budget in (5, 32, 100):
        _selection(23, layout, (F32, BF16), [16 * 110, 16 * 700], None, budget, 1, 2, near)


def test_the_largest_budget_lists_every_block():
    """2^31 - 1 places, 8.6 GB: the row's columns, then -1 to the last one."""
    bounds = torch.zeros(5, 1, 2, 8, dtype=BF16, device="cuda")
    out = S.select_blocks(torch.zeros(1, 1, 8, dtype=BF16, device="cuda"), bounds, _i32([[4, 0, 2, 1, 3]]), _i32([33]), 16, S.MOST_BUDGET)
    assert out.shape == (1, 1, S.MOST_BUDGET) and out[0, 0, :3].tolist() == [0, 1, 2]
    for part in out[0, 0, 3:].split(1 << 28):
        assert (part == -1).all()


@pytest.mark.parametrize("budget,block_size", [(2 ** 31, 16), (2 ** 32 + 4, 16), (4, 2 ** 16 + 1), (4, 2 ** 32 + 16)])
def test_numbers_that_a_call_cannot_hold_are_refused(budget, block_size):
    bounds = torch.zeros(5, 1, 2, 8, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="at most"):
        S.select_blocks(torch.zeros(1, 1, 8, dtype=BF16, device="cuda"), bounds, _i32([[4, 0, 2, 1, 3]]), _i32([33]), block_size, budget)
