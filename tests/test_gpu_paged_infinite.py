"""Infinite and NaN values in the paged cache: an infinite element of V makes its dim of the heads that read it
infinite, whatever the slot's weight and its place in a tile, a split or the row; with infinities of both
signs, or a NaN, the dim is NaN.  Everything else keeps its bits."""
import math

import numpy as np
import pytest
import torch

from test_gpu_paged import TYPES, Pool, dev

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def put(pool, row, head, slot, dim, x):
    pool.v[int(pool.table[row, slot // pool.ps]), head, slot % pool.ps, dim] = x


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H,KV,hd", [(16, 2, 128), (5, 5, 64), (40, 2, 64), (34, 2, 128), (16, 4, 256), (12, 2, 256)])
def test_infinite_values(H, KV, hd, dtype):
    lens = [1, 2, 37, 300, 2000, 1920, 0]
    pool = Pool(len(lens), 2003, KV, hd, 16, dtype, seed=H)
    rows = len(lens)
    q = (torch.randn(rows, H, hd, generator=torch.Generator().manual_seed(1)) * 2).cuda()
    dl, h = dev(np.array(lens, np.int32)), KV - 1
    w0, w1 = (torch.zeros(rows, KV, 2003, device="cuda") for _ in "ab")
    want = pool.p.attention(q, dl, 2003, weight_out=w0).reshape(rows, KV, H // KV, hd)
    for r, n in enumerate(lens):
        put(pool, r, h, n, 30, INF)  # behind the length
        if n == 0:
            continue
        last, mid = n - 1, n // 2
        special = {3: [(0, INF)], 7: [(last, -INF)], 8: [(last, INF)], hd - 1: [(mid, INF)], 20: [(0, NAN)], 33: [(last, NAN)],
                   34: [(mid, -INF), (min(127, last), -INF)], 40: [(0, INF), (last, NAN)], 41: [(0, INF), (last, -INF)]}
        for d, places in special.items():
            for slot, x in places:
                put(pool, r, h, slot, d, x)
            left = dict(places).values()  # (the last one at a slot)
            want[r, h, :, d] = sum(left)
    got = pool.p.attention(q, dl, 2003, weight_out=w1).reshape(rows, KV, H // KV, hd)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, 0.0, 1e38, -1e38), torch.nan_to_num(want, 0.0, 1e38, -1e38))
    assert torch.equal(w0, w1)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [50, 4000])
def test_infinite_values_of_slots_that_weigh_nothing(n, dtype):
    """Weights that 32 bits hold as 0, in the tile of the largest and in splits far from it; a window keeps its
    hands off the slots before it."""
    pool = Pool(1, n, 1, 64, 16, dtype, seed=13)
    at = torch.arange(n)
    pool.k[pool.table[0, at // 16].long().cuda(), 0, (at % 16).cuda(), 0] = (-at.float()).to(pool.k.dtype).cuda()
    q = torch.randn(1, 3, 64, generator=torch.Generator().manual_seed(13))
    q[0, :, 0] = torch.tensor([100.0, -100.0, 40.0])
    lens = dev(np.array([n], np.int32))
    want = pool.p.attention(q.cuda(), lens, n)
    before = pool.p.attention(q.cuda(), lens, n, window=n - 40)
    put(pool, 0, 0, 2, 5, INF)
    put(pool, 0, 0, n - 3, 6, -INF)
    put(pool, 0, 0, n // 2, 63, INF)
    got = pool.p.attention(q.cuda(), lens, n)
    want[..., 5], want[..., 6], want[..., 63] = INF, -INF, INF
    assert torch.equal(got, want)
    got = pool.p.attention(q.cuda(), lens, n, window=n - 40)
    before[..., 6] = -INF
    if n // 2 >= 40:
        before[..., 63] = INF
    assert torch.equal(got, before)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_nan_scores_and_bad_pages_stay_nan(dtype):
    """A head whose scores are NaN, a row with a bad page: NaN, infinite values or not."""
    pool = Pool(3, 300, 2, 128, 16, dtype, seed=14)
    for r in range(3):
        put(pool, r, 1, 17, 9, INF)
    pool.k[int(pool.table[0, 2]), 1, 3, 4] = NAN
    pool.p.table[1, 3] = -1
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(14)).cuda()
    for lens in ([300, 300, 300], [60, 64, 60]):
        got = pool.p.attention(q, dev(np.array(lens, np.int32)), 300)
        assert torch.isnan(got[0, 4:]).all() and torch.isfinite(got[0, :4]).all() and torch.isnan(got[1]).all()
        assert torch.isfinite(got[2, :4]).all() and (got[2, 4:, 9] == INF).all()
