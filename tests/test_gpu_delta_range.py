"""Prompts of the delta rule whose products of keys, queries, values and states pass f32's range before the norms are
applied, while everything in the recurrence stays within it.  Tolerances: test_gpu_delta.py's."""
import numpy as np
import pytest
import torch

import chpe_amd as ca
from test_gpu_delta import Layer, before, dev, pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("keys,queries,values,states", [
    (1e13, 1.0, 1.0, 1e27), (1.0, 1e13, 1.0, 1e27), (1e13, 1e13, 1e25, 1e25), (1e12, 1.0, 1e30, 1.0), (1e6, 1e6, 1e19, 1e24),
    (1e7, 1e-20, 1e20, 1e30), (1e-18, 1e7, 1e24, 1e-20), (1.0, 1.0, 1.0, 1e33)])
def test_products_past_the_range(keys, queries, values, states, hd, dtype):
    """The last chunk has few tokens; the values are large in the first one alone (the state's size stays)."""
    NK, NV, n = 2, 4, 150
    L = Layer(n, NK, NV, hd, dtype, False, seed=7)
    L.k *= keys
    L.q *= queries
    L.v[:64] *= values
    _, state = pool(2, NV, hd, 7)
    state *= states
    S0 = before(state, 0)
    out = ca.DeltaStates(state, NK).prompt(*L.args(), dev([0, n]), dev([0]), dev([1]))
    assert torch.isfinite(out).all() and torch.isfinite(state).all()
    L.check(0, n, out, state[1], S0, (keys, queries, values, states))
