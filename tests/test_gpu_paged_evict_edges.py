"""Eviction with as many moves as there can be, on both sides of every length where another form of the selection
takes over (1024, 4096, 16384 and 32768 slots)."""
import numpy as np
import pytest

from test_gpu_paged import Pool, check_evict, evict_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n", [1023, 1024, 1025, 4095, 4096, 4097, 16384, 16385, 32767, 32768, 32769])
def test_half_of_the_slots_move(n, in_place):
    budget = n // 2
    pool = Pool(2, n, 2, 64, 64, "bf16", seed=n)
    w, p = evict_inputs(2, 2, n, n)
    w[0, 0, :budget] = 0.5  # every slot below the budget goes, every one from there on stays but the last
    w[0, 0, budget:] = 1.0 + np.arange(n - budget)[::-1] / n
    w[1, 1] = 0.25          # ties all over
    check_evict(pool, w, p, [n, n - 5], n, budget, 0, 0, in_place=in_place)
    check_evict(pool, w, p, [n, n - 5], n, budget + 3, budget // 2, 3, in_place=in_place)
