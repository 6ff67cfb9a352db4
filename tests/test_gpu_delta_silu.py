"""SiLU behind the convolution and in the gated norm's gate, over all of its range.

x / (1 + e^-x) is off by at most 8 u of itself, u = 2^-24 (delta.hpp counts them), from x = -87 on; below, where 1 + e^-x passes
2^125.5 and its reciprocal leaves the normal numbers, by no more than it is: 87 e^-87 = 1.4319e-36.  An output of a 16-bit type
is off by half a step more; below the type's smallest normal number the step is a fixed one, half of which is 2^-25 for fp16
(2^-14 - 10 - 1), 2^-134 for bf16 (2^-126 - 7 - 1), 2^-150 for f32 (2^-126 - 23 - 1).  At -inf the formula itself is NaN."""
import math

import numpy as np
import pytest
import torch

import chpe_amd as ca
from test_gpu_delta import HALF, TYPES, U, dev

pytestmark = pytest.mark.gpu

TAIL = 1.432e-36
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def silu64(x):
    return x * np.where(x > 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def inputs(n, dtype):
    x = np.concatenate((np.linspace(-120, 120, n - 900), np.linspace(-104, -86, 400), np.geomspace(1e-38, 1e4, 250), -np.geomspace(1e-38, 1e4, 250)))
    x = torch.from_numpy(x).float().to(TYPES[dtype])
    x[:5] = torch.tensor([math.inf, 1e4, 0.0, -0.0, -6e4])
    return x


@pytest.mark.parametrize("dtype", list(TYPES))
def test_behind_the_convolution(dtype):
    n = 8192
    x = inputs(n, dtype)
    x[5:7] = torch.tensor([math.nan, -math.inf])
    w = torch.ones(n, 2, device="cuda")
    y = ca.DeltaConv(torch.zeros(1, n, 1, device="cuda"), w).apply(x[None].cuda(), None, dev([0]))[0].cpu().double().numpy()
    assert np.isnan(y[5:7]).all() and y[0] == math.inf and (y[2:4] == 0).all()
    ref = silu64(x.double().numpy()[7:])
    y = y[7:]
    tol = np.where(x.double().numpy()[7:] >= -87, 8 * U * np.abs(ref), TAIL)
    tol = tol + HALF[dtype] * (np.abs(ref) + tol) + 8 * LEAST["f32"] + LEAST[dtype]
    err = np.abs(y - ref)
    assert (err <= tol).all(), (x[7:][(err > tol)][:5], float((err / tol).max()))


@pytest.mark.parametrize("call", ["step", "prompt of few", "prompt"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_the_gate(dtype, call):
    """Outputs of one token that are the same in every dim have the root mean square 1 with eps 0: the gate is left.  (Two
    sums, a root, a reciprocal, three products: 8 + hd / 64 roundings more.)"""
    hd, heads, n = 64, 128, dict(step=1).get(call, 9 if call == "prompt of few" else 17)
    z = torch.zeros(n, heads, hd, dtype=TYPES[dtype])
    z[-1] = inputs(heads * hd, dtype).reshape(heads, hd)
    z[-1, 0, :5] = 1.0
    one = torch.ones(n, heads, hd, dtype=TYPES[dtype], device="cuda")
    gates = torch.full((n, heads), 20.0, device="cuda")
    args = (one, one, one, torch.full_like(gates, -60.0), gates, torch.zeros(heads, device="cuda"), torch.zeros(heads, device="cuda"))
    kw = dict(z=z.cuda(), norm_w=torch.ones(hd, device="cuda"), eps=0.0)
    h = ca.DeltaStates(torch.zeros(1, heads, hd, hd, device="cuda"), heads)
    out = h.step(*args, dev([-1]), dev([0]), **kw) if call == "step" else h.prompt(*args, dev([0, n]), dev([-1]), dev([0]), **kw)
    zz, y = z[-1].double().numpy(), out[-1].cpu().double().numpy()
    ref = silu64(zz)
    tol = np.where(zz >= -87, (8 + 8 + hd / 64) * U * np.abs(ref), TAIL * 1.001)
    tol = tol + HALF[dtype] * (np.abs(ref) + tol) + 16 * LEAST["f32"] + LEAST[dtype]
    err = np.abs(y - ref)
    assert (err <= tol).all(), (zz[err > tol][:5], float((err / tol).max()))
