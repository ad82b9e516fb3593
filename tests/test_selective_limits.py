"""Limits of the caches whose decode reads selected blocks that need no GPU."""

import pytest

from nano_vllm_jax_b200.kernels import selective_kv as S


@pytest.mark.parametrize("budget", [2 ** 31, 2 ** 32 + 4, 10 ** 12])
def test_budgets_that_a_call_cannot_hold_are_refused(budget):
    with pytest.raises(ValueError, match="at most"):
        S.check_budget(budget, 1, 1)
    S.check_budget(2 ** 31 - 1, 1, 1)
