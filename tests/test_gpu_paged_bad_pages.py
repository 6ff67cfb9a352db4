"""Eviction over rows with page ids outside the pool: a kept slot that lies in such a page is lost, and the slot
that it would have filled holds NaN, so that the attention after the eviction still says so."""
import numpy as np
import pytest
import torch

from test_gpu_paged import TYPES, Pool, dev, evict_inputs, evict_ref

pytestmark = pytest.mark.gpu

BITS = {torch.float32: torch.int32, torch.float16: torch.int16, torch.bfloat16: torch.int16}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,budget", [(64, 20), (600, 300), (64, 61)])
@pytest.mark.parametrize("hd", [64, 256])
def test_slots_kept_in_a_bad_page_become_nan(hd, n, budget, dtype):
    rows, KV, H, ps = 4, 2, 4, 16
    pool = Pool(rows, n, KV, hd, ps, dtype, seed=n)
    w, p = evict_inputs(rows, KV, n, n)
    w[:, 0, n - ps:] += 1e3  # head 0 keeps what lies in the last page, head 1 nothing of it
    w[:, 1, n - ps:] = 0.0
    bad = torch.zeros(pool.table.shape, dtype=torch.bool)
    last = pool.table.shape[1] - 1
    for row, page, new in ((1, last, pool.k.shape[0]), (2, last, -1), (2, 0, 0x7fffffff), (3, 0, -2 ** 31)):
        pool.p.table[row, page] = new
        bad[row, page] = True
    k0, v0 = pool.k.cpu().clone(), pool.v.cpu().clone()
    nan = torch.zeros(k0.shape[:3], dtype=torch.bool)
    lost = np.zeros((rows, KV), bool)
    for r in range(rows):
        for h in range(KV):
            src = evict_ref(w[r, h], p[r, h], n, budget, 0, 0)
            for d in np.flatnonzero(src != np.arange(len(src))):
                pd, po, s, so = d // ps, d % ps, src[d] // ps, src[d] % ps
                to, frm = int(pool.table[r, pd]), int(pool.table[r, s])
                if bad[r, pd]:
                    continue
                if bad[r, s]:
                    nan[to, h, po] = True
                    lost[r, h] = True
                else:
                    k0[to, h, po], v0[to, h, po] = k0[frm, h, so], v0[frm, h, so]
    lens = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    pool.p.evict(lens, n, budget, dev(w), dev(p))
    for got, want in ((pool.k.cpu(), k0), (pool.v.cpu(), v0)):
        assert torch.isnan(got[nan]).all()
        b = BITS[got.dtype]
        assert torch.equal(got[~nan].contiguous().view(b), want[~nan].contiguous().view(b))
    # what the attention says of them
    assert lost[:, 0].tolist() == [False, True, n - budget < ps or lost[2, 0], False] and not lost[:, 1].any()
    q = torch.randn(rows, H, hd, generator=torch.Generator().manual_seed(1)).cuda()
    out = pool.p.attention(q, lens, n).cpu().reshape(rows, KV, H // KV, hd)
    for r in range(rows):
        for h in range(KV):
            here = lost[r, h] or bool(bad[r, :-(-budget // ps)].any())
            assert torch.isnan(out[r, h]).all() if here else torch.isfinite(out[r, h]).all(), (r, h)
