"""The paged cache's calls at the largest launches that they make: nearly all rows are empty or share their pages."""
import numpy as np
import pytest
import torch

import chpe_amd as ca
from test_gpu_paged import Pool, attend64, dev

pytestmark = pytest.mark.gpu


def shared(rows, capacity, hd, ps, seed):
    """A cache of f32 rows that all have the same pages."""
    pool = Pool(1, capacity, 1, hd, ps, "f32", seed=seed)
    pool.p = ca.KvPages(pool.k, pool.v, pool.table.cuda().expand(rows, -1).contiguous())
    return pool


def test_attention_of_more_splits_than_a_launch_holds():
    """2^15 rows of 512 splits would be 2^24 workgroups: longer splits."""
    rows, n = 1 << 15, 512 << 10
    pool = shared(rows, n, 64, 4096, 1)
    lens = np.zeros(rows, np.int32)
    some = {0: n, 1: 5, 12345: 3000, rows - 2: n - 70001, rows - 1: 1}
    for r, m in some.items():
        lens[r] = m
    q = torch.randn(rows, 1, 64, generator=torch.Generator().manual_seed(1))
    out = pool.p.attention(q.cuda(), dev(lens), n).cpu().double()
    k, v = pool.rows64(0, n)
    for r, m in some.items():
        ref, _, tol, _ = attend64(q[r], k[:, :m], v[:, :m], 0.125)
        assert ((out[r] - ref).abs() <= tol).all(), r
        out[r] = 0
    assert not out.any()


def test_attention_with_weights_at_the_largest_join():
    """2^23 (row, query head) pairs in two splits and 2^20 workgroups of weights: one launch joins them all."""
    rows, H, n = 1 << 20, 8, 512
    pool = shared(rows, n, 256, 64, 2)
    lens = np.zeros(rows, np.int32)
    some = {0: n, 1: 5, 777777: 300, rows - 1: 511}
    for r, m in some.items():
        lens[r] = m
    q = torch.zeros(rows, H, 256, device="cuda")
    for r in some:
        q[r] = torch.randn(H, 256, generator=torch.Generator().manual_seed(r)).cuda()
    w = torch.zeros(rows, 1, n, device="cuda")
    out = pool.p.attention(q, dev(lens), n, weight_out=w)
    k, v = pool.rows64(0, n)
    for r, m in some.items():
        ref, p, tol, ptol = attend64(q[r].cpu(), k[:, :m], v[:, :m], 1 / 16)
        assert ((out[r].cpu().double() - ref).abs() <= tol).all(), r
        assert ((w[r, 0, :m].cpu().double() - p.sum(0)).abs() <= ptol.sum(0) + H * 2.0 ** -24 * p.sum(0)).all(), r
        out[r], w[r, :, :m] = 0, 0
    assert not out.any() and not w.any()


def test_eviction_of_the_most_rows():
    """2^22 - 1 rows, of which the first and the last two are over the budget."""
    rows, n = (1 << 22) - 1, 4
    pool = Pool(1, 16, 1, 64, 4, "f16", seed=3)
    pages = pool.table[0].tolist()
    table = torch.full((rows, 1), pages[3], dtype=torch.int32)
    cut = {0: pages[0], rows - 2: pages[1], rows - 1: pages[2]}
    lens = np.full(rows, 2, np.int32)
    w = torch.ones(rows, 1, n)
    for r, page in cut.items():
        table[r], lens[r], w[r, 0, 1] = page, n, 0.0
    p = ca.KvPages(pool.k, pool.v, table.cuda())
    k0, v0 = pool.k.clone(), pool.v.clone()
    for page in cut.values():  # slot 1 goes, slot 3 takes its place
        k0[page, 0, 1], v0[page, 0, 1] = k0[page, 0, 3], v0[page, 0, 3]
    dl, sp = dev(lens), torch.arange(n, dtype=torch.int32, device="cuda").expand(rows, 1, n).contiguous()
    sw = w.cuda()
    p.evict(dl, n, 3, sw, sp)
    assert torch.equal(pool.k, k0) and torch.equal(pool.v, v0)
    assert dl.cpu().tolist() == np.minimum(lens, 3).tolist()
    assert int((sp != torch.arange(n, dtype=torch.int32, device="cuda")).sum()) == 3 and int((sw != 1).sum()) == 0
    assert all(int(sp[r, 0, 1]) == 3 for r in cut)
