"""Attention over the paged cache, alone and behind a shared prefix, at scores far beyond what exponentials can tell apart: the
slots of the largest score have all the weight, equal shares of it where they tie.

A slot's key is a multiple of 1 / 8 in one dim, so that a query's scores differ by 1 / 128 of the largest or not at all, and tied
ones are the same number in 32 bits: with the largest from 2^17 on (in units of log2) all other weights are 0 (2^-1024).  The
weights of m tied slots are the same w, the output is a sum of m products with V, each rounded with the parts of w (2 u), m
additions (and of zeros), the sum of the weights (m u), a reciprocal or division and its product: (2 m + 8) u of the values'
mean magnitude, u = 2^-24.

A slot's weight is formed from its score, rounded (in units of log2: t), its row's sum from the score as the fma has it, which
differ by u |t|: 2^(u |t|) between the two, up to t = 2^22, from where on both take the rounded one."""
import numpy as np
import pytest
import torch

import chpe_amd as ca
from test_gpu_paged import TYPES, U, dev

pytestmark = pytest.mark.gpu

POWERS = [17, 21, 22, 23, 24, 25, 27, 31, 33, 40, 64, 100]


def make(rows, n, KV, hd, dtype, H, seed):
    g = torch.Generator().manual_seed(seed)
    pages = -(-n // 16)
    steps = torch.randint(-64, 65, (rows * pages, KV, 16), generator=g)
    steps[::2, :, 5], steps[::3, :, 7] = 64, -64  # ties, in several tiles and splits
    k = torch.zeros(rows * pages, KV, 16, hd)
    k[..., 3] = steps / 8.0
    v = torch.randn(rows * pages, KV, 16, hd, generator=g).to(TYPES[dtype])
    q = torch.zeros(rows, H, hd)
    q[..., 3] = (1 + torch.rand(rows, H, generator=g)) * 2.0 ** torch.tensor(POWERS, dtype=torch.float32)[torch.randint(0, len(POWERS), (rows, H), generator=g)]
    q[..., 3] *= torch.sign(torch.rand(rows, H, generator=g) - 0.5)
    return k.to(TYPES[dtype]).cuda(), v.cuda(), q


def check(out, q, steps, v, what):
    """One row: steps and v [KV][n], out [H][hd]."""
    H, KV = q.shape[0], steps.shape[0]
    for h in range(H):
        s = steps[h * KV // H] * (1 if q[h, 3] > 0 else -1)
        tied = v[h * KV // H][s == s.max()].double()
        tol = (2 * len(tied) + 8) * U * tied.abs().mean(0)
        err = (out[h].double() - tied.mean(0)).abs()
        assert (err <= tol).all(), (*what, h, float(q[h, 3]), len(tied), float((err / tol).max()))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H,KV,hd", [(16, 2, 64), (40, 2, 128), (7, 1, 256), (20, 1, 256), (6, 3, 128)])
def test_alone(H, KV, hd, dtype, sign):
    rows, n = 6, 330
    k, v, q = make(rows, n, KV, hd, dtype, H, H + hd)
    if sign < 0:  # all scores far below 0: the largest is -2^power / 8 or less
        k[..., 3] = -k[..., 3].abs() - 0.125
        q = q.abs()
    pages = -(-n // 16)
    p = ca.KvPages(k, v, torch.arange(rows * pages, dtype=torch.int32).reshape(rows, pages).cuda())
    lens = [n, 1, 17, 300, 64, 129]
    w = torch.zeros(rows, KV, n, device="cuda")
    out = p.attention(q.cuda(), dev(np.array(lens, np.int32)), n, scale=0.3, weight_out=w).cpu()
    flat = lambda t: t.cpu().float().reshape(rows, pages, KV, 16, -1).transpose(1, 2).reshape(rows, KV, pages * 16, -1)  # noqa: E731
    kk, vv = flat(k)[..., 3], flat(v)
    for r, m in enumerate(lens):
        check(out[r], q[r], kk[r, :, :m], vv[r, :, :m], (r,))
        s = kk[r, :, :m].repeat_interleave(H // KV, 0) * torch.sign(q[r, :, 3])[:, None]
        tied = (s == s.amax(-1, keepdim=True)).double()
        share = tied / tied.sum(-1, keepdim=True)
        t = (q[r, :, 3].abs() * 8 * 0.3 / np.log(2)).double().clamp(max=2.0 ** 22)[:, None]
        tol = share * ((2 * 64 + H) * U + torch.expm1(np.log(2) * U * t))
        want, tol = (x.reshape(KV, H // KV, m).sum(1) for x in (share, tol))
        err = (w[r, :, :m].cpu().double() - want).abs()
        assert (err <= tol).all(), (r, float((err - tol).max()))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,H,KV,hd", [(3, 4, 2, 64), (2, 12, 1, 128), (2, 6, 1, 256), (9, 40, 1, 64), (5, 96, 2, 128), (9, 40, 1, 256)])
def test_behind_a_prefix(rows, H, KV, hd, dtype):
    prefix, n = 500, 500 + 130
    k, v, q = make(rows, n, KV, hd, dtype, H, rows + hd)
    pages = -(-n // 16)
    table = torch.arange(rows * pages, dtype=torch.int32).reshape(rows, pages)
    p = ca.KvPages(k, v, table.cuda())
    lens = [prefix + 1 + (37 * r) % 130 for r in range(rows)]
    lens[-1] = 77  # shorter than the prefix
    out = p.prefix_attention(q.cuda(), dev(np.array(lens, np.int32)), dev(np.array([0, rows], np.int32)), dev(np.array([prefix], np.int32)),
                             prefix, 130, scale=0.3).cpu()
    flat = lambda t: t.cpu().float().reshape(rows, pages, KV, 16, -1).transpose(1, 2).reshape(rows, KV, pages * 16, -1)  # noqa: E731
    kk, vv = flat(k)[..., 3], flat(v)
    for r, m in enumerate(lens):
        of = [torch.cat((t[0, :, :prefix], t[r, :, prefix:]), 1)[:, :m] for t in (kk, vv)]
        check(out[r], q[r], *of, (r,))
