"""How many bits of the f32 queries and softmax weights the paged attention's products keep, with inputs whose
errors do not hide among many others: one-hot keys (a score is one product) and one-hot values (an output is
one weight).

Bounds, in roundings to f32 (u = 2^-24 relative).  A score s = q scale is exact but for what the products hold of
q: all 24 bits against f32 and bf16 caches (one product or three parts, whose sum is q itself), 22 bits in two
parts against fp16 (off by at most 2 u).  In units of log2 it is rounded three times: log2 e times the scale (1 u
of every score alike, so of their difference), the product (1 u of each of the two), and the same for the largest.
So the exponent is off by at most e = (2 + c) u (|t_j| + |t_max|) with c = 0 or 2, and a weight, which has the sum
of all below it, by 2 ln 2 e relative, plus 8 + n u for two exponentials (1 u each), n - 1 additions, the reciprocal
or division and its product, and, for an output, the parts' sum.  An output has the weight's parts too: 2 u more
for fp16.  Two bf16 parts instead of three leave an error of up to 64 u in a query's difference to the next, and in
a weight: the oracle's own test below shows that they would not pass."""
import numpy as np
import pytest
import torch

from test_gpu_paged import TYPES, U, Pool, dev

LN2 = float(np.log(2.0))


def inputs(H, KV, hd, rows, n, seed):
    """Queries between 4 and 8 or -8 and -4 with random low bits; slot j's key is 1 at dim j."""
    g = torch.Generator().manual_seed(seed)
    q = 4.0 + 4.0 * torch.rand(rows, H, hd, generator=g)
    near = torch.rand(rows, H, 1, generator=g) * 3 + 4  # (the row's scores within a quarter of each other)
    q[..., :n] = near + 0.25 * torch.rand(rows, H, n, generator=g)
    return q, 2.0 ** -2


def weights64(q, scale, n):
    s = q[..., :n].double() * scale
    t = s.abs() / LN2
    return s.softmax(-1), t + t.amax(-1, keepdim=True)


def bounds(p, t, n, dtype, output):
    c = 2 if dtype == "f16" else 0
    rel = (2 * LN2 * (2 + c) * t + 8 + n + (c if output else 0)) * U
    return p * rel


def parts(x, n):
    """x as the sum of its first n bf16 parts."""
    left, out = x.clone(), torch.zeros_like(x)
    for _ in range(n):
        hi = left.bfloat16().float()
        out, left = out + hi, left - hi
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (8, 2, 64), (8, 2, 256), (16, 2, 128), (14, 2, 64), (12, 2, 256), (32, 2, 128),
                                     (24, 2, 64), (20, 1, 256)])
@pytest.mark.parametrize("n", [2, 3])
def test_queries_and_weights_keep_their_bits(n, H, KV, hd, dtype):
    rows = 40
    q, scale = inputs(H, KV, hd, rows, n, H * hd + n)
    pool = Pool(rows, 16, KV, hd, 16, dtype, fill=False)
    for j in range(n):
        pool.k[:, :, j, j] = 1.0
        pool.v[:, :, j, 5 + j] = 1.0
    p, t = weights64(q, scale, n)
    w = torch.zeros(rows, KV, 16, device="cuda")
    out = pool.p.attention(q.cuda(), dev(np.full(rows, n, np.int32)), 16, scale=scale, weight_out=w).cpu().double()
    err, tol = (out[..., 5:5 + n] - p).abs(), bounds(p, t, n, dtype, True)
    assert (err <= tol).all(), float((err / tol).max())
    out[..., 5:5 + n] = 0
    assert (out == 0).all()
    # the weights of single heads: all other queries' scores are one 0 and one -200, whose weights are 1 and 2^-288
    g = H // KV
    for i in range(0, g, max(1, g // 4)):
        x = torch.zeros_like(q)
        x[..., 1], x[..., 0] = -800.0, 0.0
        x[..., 2] = -800.0
        x.view(rows, KV, g, hd)[:, :, i] = q.view(rows, KV, g, hd)[:, :, i]
        pool.p.attention(x.cuda(), dev(np.full(rows, n, np.int32)), 16, scale=scale, weight_out=w)
        want, tt = (y.view(rows, KV, g, n)[:, :, i, 1:] for y in (p, t))
        err, tol = (w[..., 1:n].cpu().double() - want).abs(), bounds(want, tt, n, dtype, False)
        assert (err <= tol).all(), (i, float((err / tol).max()))


@pytest.mark.parametrize("H,hd", [(8, 128), (32, 64)])
@pytest.mark.parametrize("n", [2, 3])
def test_two_bf16_parts_would_not_pass(n, H, hd):
    """The bounds above, against 64-bit weights of queries (and weights) cut to two bf16 parts."""
    q, scale = inputs(H, 1, hd, 40, n, H * hd + n)
    assert torch.equal(parts(q, 3), q)
    p, t = weights64(q, scale, n)
    cut, _ = weights64(parts(q, 2), scale, n)
    assert ((cut - p).abs() / bounds(p, t, n, "bf16", False)).max() > 1.5
    # a weight as it enters the product: relative to the row's largest
    rel = (p / p.amax(-1, keepdim=True)).float()
    assert torch.equal(parts(rel, 3), rel)
    assert ((parts(rel, 2) - rel).double().abs() / bounds(rel.double(), t, n, "bf16", True)).max() > 1.5
