"""The paged cache's operators (chpe_amd.KvPages) against plain computations in 64 bits on the CPU: layouts,
types, lengths from none to several splits, page ends inside a tile, windows, rows that share pages, bad
pages and lengths, eviction with ties and NaN, a run of all of them together, streams and graphs.

Tolerances count roundings to f32 (u = 2^-24 relative) in the worst case, no two cancelling:
* a score is a sum of hd products and the operands may be taken apart into parts that keep 22 bits: it is
  off by at most (hd u + 2^-21) scale sum |q k|, so a weight is off by twice that (its own and the sum's),
  plus (n + 16) u for the sum of n weights, the exponentials (|s - max| < 16 of the tests' scores would
  count 16 u) and the divisions, all relative; the output by that times sum p |v|.
* the norm of hd dims is off by (hd / 2 + 8) u relative, a rotation by 3 u of |x0| + |x1|; a cached key by
  half a step of its type more."""
import math

import numpy as np
import pytest
import torch

import chpe_amd as ca

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(a, dt=None):
    t = torch.as_tensor(np.ascontiguousarray(a) if isinstance(a, np.ndarray) else a)
    return t.to("cuda", dt) if dt else t.cuda()


class Pool:
    """A cache of `rows` sequences of up to `capacity` slots in shuffled pages, with room between them."""

    def __init__(self, rows, capacity, kv, hd, ps, dtype, seed=0, inner="slots", spare=3, fill=True):
        g = torch.Generator().manual_seed(seed)
        per = -(-capacity // ps)
        n = rows * per + spare
        shape = (n, kv, ps, hd) if inner == "slots" else (n, ps, kv, hd)
        mk = lambda: (torch.randn(shape, generator=g) if fill else torch.zeros(shape)).to(TYPES[dtype])  # noqa: E731
        k, v = mk(), mk()
        self.k, self.v = ((t if inner == "slots" else t.transpose(1, 2)) for t in (k.cuda(), v.cuda()))
        self.table = torch.randperm(n, generator=g)[:rows * per].reshape(rows, per).to(torch.int32)
        self.p = ca.KvPages(self.k, self.v, self.table.cuda())
        self.ps = ps

    def rows64(self, row, n):
        """K and V of a row's first n slots in 64 bits: [kv][n][hd]."""
        ids = self.table[row, :-(-n // self.ps)].long()
        take = lambda t: torch.cat([t[i] for i in ids.tolist()] or [t[0][:, :0]], 1)[:, :n].cpu().double()  # noqa: E731
        return take(self.k), take(self.v)


def attend64(q, k, v, scale, lo=0):
    """One row: out [H][hd], weights [H][n], and the bounds of their errors."""
    H, hd, (KV, n, _) = q.shape[0], q.shape[1], k.shape
    qq = q.double().reshape(KV, H // KV, hd)
    s = (qq @ k.transpose(1, 2)) * scale
    mag = (qq.abs() @ k.abs().transpose(1, 2)) * scale
    s[..., :lo] = -math.inf
    mag[..., :lo] = 0
    p = s.softmax(-1)
    off = 2 * (hd * U + 2.0 ** -21) * mag.amax(-1, keepdim=True) + (n + 16 + 16) * U
    return (p @ v).reshape(H, hd), p.reshape(H, n), ((p @ v.abs()) * off).reshape(H, hd), (p * off).reshape(H, n)


def check_attention(pool, q, lens, max_len, window=0, weights=False, scale=None, seed=0):
    rows, H, hd = q.shape
    KV = pool.k.shape[1]
    dq, dl = q.cuda(), dev(np.asarray(lens, np.int32))
    out = torch.full((rows, H, hd), 7.0, device="cuda")
    w_in = w_out = None
    if weights:
        g = torch.Generator().manual_seed(seed + 9)
        w_in = torch.rand(rows, KV, max_len + 5, generator=g)
        w_out = torch.full((rows, KV, max_len + 5), -3.0, device="cuda")
    pool.p.attention(dq, dl, max_len, scale=scale, window=window, out=out, weight_in=w_in.cuda() if weights else None,
                     weight_out=w_out)
    out, got_w = out.cpu().double(), w_out.cpu().double() if weights else None
    sc = hd ** -0.5 if scale is None else scale
    for r, n in enumerate(lens):
        if n == 0:
            assert (out[r] == 0).all(), r
            assert not weights or (got_w[r] == -3.0).all()
            continue
        lo = max(0, n - window) if window else 0
        ref, p, tol, ptol = attend64(q[r], *pool.rows64(r, n), sc, lo)
        err = (out[r] - ref).abs()
        assert (err <= tol + 1e-30).all(), (r, n, float((err / tol).max()))
        if weights:
            g = H // KV
            w = w_in[r, :, :n].double() + p.reshape(KV, g, n).sum(1)
            wt = ptol.reshape(KV, g, n).sum(1) + (g + 2) * U * w.abs()
            e = (got_w[r, :, :n] - w).abs()
            assert (e <= wt).all(), (r, n, float((e / wt).max()))
            assert (got_w[r, :, n:] == -3.0).all()  # behind the length: left as it was


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H,KV,hd", [(16, 2, 128), (16, 4, 256), (64, 8, 128), (5, 5, 64), (24, 8, 128), (12, 1, 64),
                                     (32, 2, 128), (40, 1, 256), (33, 3, 64), (17, 1, 128)])
def test_attention_layouts(H, KV, hd, dtype):
    lens = [77, 0, 1, 300, 31, 32, 33, 128, 129]
    pool = Pool(len(lens), 300, KV, hd, 16, dtype, seed=H)
    q = torch.randn(len(lens), H, hd, generator=torch.Generator().manual_seed(1)) * 2
    check_attention(pool, q, lens, 300)
    check_attention(pool, q, lens, 300, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_many_heads_a_kv_head(hd, dtype):
    """More query heads on one kv head than a workgroup serves, and than the weights' launch takes at a time."""
    pool = Pool(2, 400, 1, hd, 16, dtype, seed=14)
    q = torch.randn(2, 130, hd, generator=torch.Generator().manual_seed(14)) * 2
    check_attention(pool, q, [400, 63], 400, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_does_not_depend_on_the_other_rows(dtype):
    """A row's bits are the same whatever the other rows' lengths are."""
    pool = Pool(5, 3000, 2, 128, 16, dtype, seed=15)
    q = torch.randn(5, 16, 128, generator=torch.Generator().manual_seed(15)).cuda()
    got = [pool.p.attention(q, dev(np.array([1234, *rest], np.int32)), 3000)[0]
           for rest in ((0, 0, 0, 0), (3000, 3000, 3000, 3000), (1, 2999, 17, 640))]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ps", [1, 2, 8, 64, 256])
def test_attention_page_sizes_and_orders(ps, dtype):
    """Pages that end inside a tile, one slot a page, and heads as the inner dimension."""
    lens = [255, 13, 256, 100]
    q = torch.randn(4, 16, 128, generator=torch.Generator().manual_seed(2)) * 2
    for inner in ("slots", "heads"):
        pool = Pool(4, 256, 4, 128, ps, dtype, seed=ps, inner=inner)
        check_attention(pool, q, lens, 256, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 5000), (1, 20011), (3, 4097), (70, 130)])
def test_attention_lengths(rows, n, dtype):
    """From one slot to many splits, one row and many."""
    rng = np.random.default_rng(n)
    lens = [n] + [int(x) for x in rng.integers(0, n + 1, rows - 1)]
    pool = Pool(rows, n, 2, 128, 16, dtype, seed=n)
    q = torch.randn(rows, 16, 128, generator=torch.Generator().manual_seed(3)) * 2
    check_attention(pool, q, lens, n)
    check_attention(pool, q, lens, n, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("window", [1, 7, 32, 100, 999, 5000])
def test_attention_windows(window, dtype):
    lens = [1000, 999, 101, 100, 99, 1, 0]
    pool = Pool(7, 1000, 2, 64, 32, dtype, seed=window)
    q = torch.randn(7, 6, 64, generator=torch.Generator().manual_seed(4)) * 2
    check_attention(pool, q, lens, 1000, window=window)
    check_attention(pool, q, lens, 1000, window=window, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size,scale", [(1e-4, 1.0), (3e4, 1e-6), (1e7, 1e-9), (2.0, 0.0)])
def test_attention_query_ranges(size, scale, dtype):
    """Queries far from one (past fp16's range too), no scale at all: a plain mean."""
    pool = Pool(2, 200, 2, 128, 16, dtype, seed=5)
    q = torch.randn(2, 16, 128, generator=torch.Generator().manual_seed(5)) * size
    check_attention(pool, q, [200, 77], 200, scale=scale, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_small_keys_and_values(dtype):
    """Keys and values among fp16's subnormal numbers."""
    pool = Pool(2, 200, 2, 128, 16, dtype, seed=12)
    pool.k.mul_(2.0 ** -17)
    pool.v.mul_(2.0 ** -17)
    q = torch.randn(2, 16, 128, generator=torch.Generator().manual_seed(12)) * 1000
    check_attention(pool, q, [200, 77], 200, scale=3.0, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_splits_of_very_different_scores(dtype):
    """Scores that fall by hundreds from one split to the next: the join's maximum is the row's, however low."""
    n = 4000
    pool = Pool(1, n, 1, 64, 16, dtype, seed=13)
    at = torch.arange(n)
    pool.k[pool.table[0, at // 16].long().cuda(), 0, (at % 16).cuda(), 0] = (-at.float()).to(pool.k.dtype).cuda()
    q = torch.randn(1, 3, 64, generator=torch.Generator().manual_seed(13))
    q[0, :, 0] = torch.tensor([5.0, -5.0, 40.0])
    check_attention(pool, q, [n], n, weights=True)
    pool.k[:, :, :, 0] = -4000.0
    check_attention(pool, q, [n], n, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_sharp_and_flat_rows(dtype):
    """One slot that takes nearly everything, at the ends of tiles and splits; equal keys, whose weights are
    equal."""
    n = 700
    pool = Pool(1, n, 1, 128, 16, dtype, seed=6)
    q = torch.randn(1, 4, 128, generator=torch.Generator().manual_seed(6))
    for j in (0, 31, 32, 127, 128, n - 1):
        keep = pool.k.clone()
        page = int(pool.table[0, j // 16])
        pool.k[page, 0, j % 16] = (q[0, 1] * 3).to(pool.k.dtype).cuda()  # (score 3 |q|^2 / sqrt(128), about 34)
        check_attention(pool, q, [n], n, weights=True)
        pool.k.copy_(keep)
    pool.k[:] = pool.k[0, 0, 0].clone()
    check_attention(pool, q, [n], n, weights=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_ignores_what_lies_behind_the_length(dtype):
    """NaN and infinities in slots behind the length, in foreign pages and in table entries never read."""
    rows, n = 3, [45, 16, 130]
    pool = Pool(rows, 160, 2, 128, 16, dtype, seed=7)
    q = torch.randn(rows, 16, 128, generator=torch.Generator().manual_seed(7)) * 2
    want = pool.p.attention(q.cuda(), dev(np.array(n, np.int32)), 160)
    used = torch.zeros(pool.k.shape[0], pool.ps, dtype=torch.bool)
    for r in range(rows):
        for j in range(n[r]):
            used[int(pool.table[r, j // 16]), j % 16] = True
    gone = ~used[:, None, :, None].expand(pool.k.shape).cuda()
    for bad in (math.nan, math.inf, -math.inf):
        pool.k.masked_fill_(gone, bad)
        pool.v.masked_fill_(gone, bad)
        table = pool.p.table.clone()
        for r in range(rows):
            table[r, -(-n[r] // 16):] = 0x7fffffff if bad > 0 else -1
        p = ca.KvPages(pool.k, pool.v, table)
        got = p.attention(q.cuda(), dev(np.array(n, np.int32)), 160)
        assert torch.equal(got, want)


def test_attention_non_finite_values_stay_with_their_head():
    """A NaN or infinite value in one head's row of a used slot reaches that head's outputs and no others."""
    pool = Pool(2, 50, 2, 128, 16, "f16", seed=8)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(8))
    lens = dev(np.array([50, 40], np.int32))
    want = pool.p.attention(q.cuda(), lens, 50)
    page = int(pool.table[0, 1])
    for cache, bad in ((pool.v, math.nan), (pool.v, math.inf), (pool.k, math.nan)):
        old = cache[page, 1, 3, 5].clone()
        cache[page, 1, 3, 5] = bad
        got = pool.p.attention(q.cuda(), lens, 50)
        assert torch.equal(got[1], want[1]) and torch.equal(got[0, :4], want[0, :4])
        assert not torch.isfinite(got[0, 4:, 5]).any()
        if cache is pool.v:
            assert torch.equal(got[0, 4:, :5], want[0, 4:, :5]) and torch.equal(got[0, 4:, 6:], want[0, 4:, 6:])
        cache[page, 1, 3, 5] = old


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_bad_lengths_and_pages_give_nan(dtype):
    pool = Pool(5, 64, 2, 64, 16, dtype, seed=9)
    q = torch.randn(5, 4, 64, generator=torch.Generator().manual_seed(9))
    good = pool.p.attention(q.cuda(), dev(np.array([64, 64, 64, 64, 64], np.int32)), 64)
    pool.p.table[1, 2] = pool.k.shape[0]
    pool.p.table[3, 0] = -1
    got = pool.p.attention(q.cuda(), dev(np.array([64, 64, -1, 64, 65], np.int32)), 64)
    assert torch.equal(got[0], good[0]) and torch.isnan(got[1:]).all()


def test_attention_rows_that_share_pages():
    """A common prefix, and one sequence's drafts as rows of growing length, weights per row."""
    pool = Pool(4, 200, 2, 128, 16, "f16", seed=10)
    pool.table[1, :5] = pool.table[0, :5]
    pool.table[2] = pool.table[0]
    pool.table[3] = pool.table[0]
    pool.p.table.copy_(pool.table)
    q = torch.randn(4, 16, 128, generator=torch.Generator().manual_seed(10))
    check_attention(pool, q, [150, 120, 151, 152], 200, weights=True)


def test_attention_offsets_past_32_bits():
    """Pages behind element 2^32 of the pool (8.6 GB of keys), and behind byte 2^32 of one head's stride."""
    n = (1 << 32) // (2 * 16 * 128) + 4
    k = torch.empty(n, 2, 16, 128, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(11)
    table = torch.tensor([[n - 1, 0, n - 3, n // 2 + 1]], dtype=torch.int32)
    for i in table[0].tolist():
        k[i], v[i] = torch.randn(2, 16, 128, generator=g).half().cuda(), torch.randn(2, 16, 128, generator=g).half().cuda()
    pool = Pool.__new__(Pool)
    pool.k, pool.v, pool.table, pool.ps, pool.p = k, v, table, 16, ca.KvPages(k, v, table.cuda())
    check_attention(pool, torch.randn(1, 16, 128, generator=g), [61], 64, weights=True)
    # the same memory with heads far apart
    heads = [t.view(2, n, 16, 128).transpose(0, 1) for t in (k, v)]
    for i in table[0].tolist():
        for t in heads:
            t[i] = torch.randn(2, 16, 128, generator=g).half().cuda()
    pool.k, pool.v = heads
    pool.p = ca.KvPages(*heads, table.cuda())
    check_attention(pool, torch.randn(1, 16, 128, generator=g), [61], 64, weights=True)
    # and written there
    x = torch.randn(3, 2, 128, generator=g).cuda()
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    slots = dev(np.array([1, 35, 63], np.int32))
    pool.p.append(x, 2 * x, z, slots, slots)
    pool.p.evict(dev(np.array([64], np.int32)), 64, 63, torch.arange(128.0, device="cuda").reshape(1, 2, 64),
                 torch.zeros(1, 2, 64, dtype=torch.int32, device="cuda"), lens_out=torch.zeros(1, dtype=torch.int32, device="cuda"),
                 weight_out=torch.zeros(1, 2, 64, device="cuda"), pos_out=torch.zeros(1, 2, 64, dtype=torch.int32, device="cuda"))
    kk, vv = pool.rows64(0, 64)
    want = x.half().cpu().double()
    assert torch.equal(kk[:, [1, 35, 63]].transpose(0, 1), want)
    assert torch.equal(kk[:, 0], want[2]) and torch.equal(vv[:, 0], (2 * x).half().cpu().double()[2])


# ------------------------------------------------------------------ append
def rope_tables(n, rot, theta=1e6):
    a = np.arange(n)[:, None] * theta ** (-2.0 * np.arange(rot // 2) / rot)[None]
    return torch.from_numpy(np.cos(a)).float(), torch.from_numpy(np.sin(a)).float()


def embed64(x, gain, eps, cos, sin, inter):
    """x [t][h][hd] normalised and rotated by cos, sin [t][rot / 2]; the bound of the error."""
    hd, half = x.shape[-1], cos.shape[-1]
    x = x.double()
    rel = 3 * U
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
        rel += (hd / 2 + 8) * U
    y, tol = x.clone(), x.abs() * rel
    c, s = cos.double()[:, None], sin.double()[:, None]
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if inter else (slice(0, half), slice(half, 2 * half))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    tol[..., i] = tol[..., j] = (x[..., i].abs() + x[..., j].abs()) * rel
    return y, tol


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H,KV,hd,rot,norm,inter,gate", [
    (16, 2, 128, 128, False, False, False), (16, 4, 256, 64, True, False, True), (64, 8, 128, 128, True, False, False),
    (5, 5, 64, 64, True, True, False), (24, 8, 128, 96, False, False, True), (7, 1, 256, 8, True, True, False),
    (0, 3, 64, 0, True, False, False), (3, 3, 128, 0, False, False, False), (33, 3, 64, 40, True, False, False),
    (1, 1, 256, 256, True, True, True), (9, 3, 128, 24, True, True, True)])
@pytest.mark.parametrize("tokens", [1, 3, 97])
def test_append(H, KV, hd, rot, norm, inter, gate, tokens, dtype):
    g = torch.Generator().manual_seed(H * 7 + tokens)
    rows, cap = 4, 48
    pool = Pool(rows, cap, KV, hd, 16, dtype, seed=tokens, spare=2, inner="heads" if inter else "slots")
    k0, v0 = pool.k.clone(), pool.v.clone()
    q = torch.randn(tokens, max(H, 1), 2 * hd if gate else hd, generator=g) * 3
    wide = torch.randn(tokens, 2 * KV + 1, hd, generator=g)  # keys and values next to each other, and something else
    k, v = wide[:, :KV], wide[:, KV + 1:]
    at = torch.randperm(rows * cap, generator=g)[:tokens]
    row, slot = at // cap, at % cap
    pos = torch.randint(0, 400, (tokens,), generator=g)
    row[tokens // 2] = -1 if tokens > 1 else row[0]  # a padded place of the batch
    gq, gk = (torch.randn(hd, generator=g) + 1 for _ in "qk") if norm else (None, None)
    cos, sin = rope_tables(400, rot) if rot else (torch.zeros(1, 0), torch.zeros(1, 0))
    sp = torch.full((rows, KV, cap + 3), -7, dtype=torch.int32, device="cuda")
    sw = torch.full((rows, KV, cap + 3), 2.5, device="cuda")
    dw, dq = wide.cuda(), q.cuda()
    i32 = lambda t: t.to(torch.int32).cuda()  # noqa: E731
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    out = pool.p.append(dw[:, :KV], dw[:, KV + 1:], i32(row), i32(slot), i32(pos), q=dq[..., :hd] if H else None,
                        q_norm=c(gq), k_norm=c(gk), eps=1e-5, rope=(cos.cuda(), sin.cuda()) if rot else None,
                        interleaved=inter, slot_pos=sp, slot_weight=sw)
    cs, sn = (cos[pos], sin[pos]) if rot else (torch.zeros(tokens, 0), torch.zeros(tokens, 0))
    if H:
        ref, tol = embed64(q[..., :hd], gq, 1e-5, cs, sn, inter)
        assert ((out.cpu().double() - ref).abs() <= tol).all()
    else:
        assert out is None
    ref, tol = embed64(k, gk, 1e-5, cs, sn, inter)
    half_step = torch.finfo(TYPES[dtype]).eps / 2 if dtype != "f32" else 0.0
    low = 2.0 ** -25 if dtype == "f16" else 0.0  # (half of fp16's smallest step)
    want_sp, want_sw = torch.full_like(sp, -7).cpu(), torch.full_like(sw, 2.5).cpu()
    for t in range(tokens):
        if row[t] < 0:
            continue
        page, off = int(pool.table[row[t], slot[t] // 16]), int(slot[t] % 16)
        err = (pool.k[page, :, off].cpu().double() - ref[t]).abs()
        assert (err <= tol[t] * (1 + half_step) + ref[t].abs() * half_step + low).all()
        assert torch.equal(pool.v[page, :, off].cpu(), v[t].to(TYPES[dtype]))
        k0[page, :, off], v0[page, :, off] = pool.k[page, :, off], pool.v[page, :, off]
        want_sp[row[t], :, slot[t]], want_sw[row[t], :, slot[t]] = int(pos[t]), 0.0
    assert torch.equal(pool.k, k0) and torch.equal(pool.v, v0)  # nothing else was written
    assert torch.equal(sp.cpu(), want_sp) and torch.equal(sw.cpu(), want_sw)


def test_append_queries_in_place():
    pool = Pool(2, 32, 2, 128, 16, "f16", seed=4)
    g = torch.Generator().manual_seed(4)
    x, q = torch.randn(50, 2, 128, generator=g).cuda(), torch.randn(50, 7, 128, generator=g).cuda()
    z = torch.zeros(50, dtype=torch.int32, device="cuda")
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    rope = tuple(t.cuda() for t in rope_tables(64, 96))
    want = pool.p.append(x, x, z - 1, z, pos, q=q, q_norm=q[0, 0] * 1, rope=rope)
    gain = q[0, 0] * 1
    assert pool.p.append(x, x, z - 1, z, pos, q=q, q_norm=gain, rope=rope, q_out=q) is q and torch.equal(q, want)


def test_append_roundings_and_special_values():
    """Values, infinities and NaN in the cache's types as torch rounds them; keys unrotated."""
    x = torch.tensor([0.0, -0.0, 1.0, 65504.0, 65519.9, 65520.0, 1e30, -1e30, 3.4e38, 1e-8, 2.98e-8, 6e-8, 1e-40, math.inf,
                      -math.inf, math.nan, 1.00390625, 1.01171875, 0.33333334])
    x = torch.cat((x, torch.randn(64 - len(x), generator=torch.Generator().manual_seed(1)))).reshape(1, 1, 64)
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    for dtype in TYPES:
        pool = Pool(1, 16, 1, 64, 16, dtype, fill=False)
        pool.p.append(x.cuda(), -x.cuda(), z, z, z)
        page = int(pool.table[0, 0])
        for got, want in ((pool.k[page, 0, 0], x[0, 0]), (pool.v[page, 0, 0], -x[0, 0])):
            want = want.to(TYPES[dtype])
            assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(got.cpu().float(), 5.0), torch.nan_to_num(want.float(), 5.0))


def test_append_bad_places_write_nothing():
    """Rows, slots, positions and pages outside: nothing is written; a position outside the tables gives NaN
    queries and leaves the other tokens alone."""
    pool = Pool(2, 32, 2, 64, 16, "f32", seed=3)
    k0, v0 = pool.k.clone(), pool.v.clone()
    pool.p.table[1, 1] = 0x40000000
    row, slot, pos = [-1, 2, 0, 0, 0, 0, 1, 0], [0, 0, -1, 32, 1, 2, 17, 4], [0, 1, 2, 3, 8, -1, 5, 7]
    g = torch.Generator().manual_seed(3)
    x = torch.randn(8, 2, 64, generator=g).cuda()
    q = torch.randn(8, 3, 64, generator=g).cuda()
    cos, sin = (t.cuda() for t in rope_tables(8, 64))
    sp = torch.full((2, 2, 32), -7, dtype=torch.int32, device="cuda")
    sw = torch.full((2, 2, 32), 2.5, device="cuda")
    i32 = lambda a: dev(np.array(a, np.int32))  # noqa: E731
    out = pool.p.append(x, x, i32(row), i32(slot), i32(pos), q=q, rope=(cos, sin), slot_pos=sp, slot_weight=sw)
    assert torch.isnan(out[[4, 5]]).all() and torch.isfinite(out[[0, 1, 2, 3, 6, 7]]).all()
    page = int(pool.table[0, 0])
    assert torch.equal(pool.v[page, :, 4], x[7])
    k0[page, :, 4], v0[page, :, 4] = pool.k[page, :, 4], x[7]
    assert torch.equal(pool.k, k0) and torch.equal(pool.v, v0)
    assert int((sp != -7).sum()) == 2 and (sp[0, :, 4] == 7).all() and int((sw != 2.5).sum()) == 2


# ------------------------------------------------------------------ evict
def evict_ref(w, p, n, budget, recent, sinks):
    """One head: the slot that each new slot held, as the header states it."""
    keep_n = min(n, budget)
    w, p, at = w[:n].astype(np.float64), p[:n].astype(np.int64), np.arange(n)
    safe = (p > p.max() - recent) | (p < sinks) if n else np.zeros(0, bool)
    nan = np.isnan(w) & ~safe
    order = sorted(at, key=lambda j: (not safe[j], nan[j], 0.0 if safe[j] or nan[j] else -w[j], j))
    keep = np.zeros(n, bool)
    keep[order[:keep_n]] = True
    src = at[:keep_n].copy()
    src[~keep[:keep_n]] = at[keep_n:][keep[keep_n:]]
    return src


def check_evict(pool, w, p, lens, max_len, budget, recent, sinks, in_place=False, src=True):
    rows, KV, stride = w.shape
    k0, v0 = pool.k.clone(), pool.v.clone()
    dl, dw, dp = dev(np.asarray(lens, np.int32)), dev(w), dev(p)
    if in_place:
        lo, wo, po = dl, dw, dp
    else:
        lo, wo, po = torch.full_like(dl, -9), torch.full_like(dw, -9.0), torch.full_like(dp, -9)
    w1, p1 = wo.cpu().numpy().copy(), po.cpu().numpy().copy()
    ss = torch.full_like(dp, -5) if src else None
    s1 = np.full(p.shape, -5, np.int32)
    pool.p.evict(dl, max_len, budget, dw, dp, recent=recent, sinks=sinks, lens_out=None if in_place else lo,
                 weight_out=None if in_place else wo, pos_out=None if in_place else po, slot_src=ss)
    for r, n in enumerate(lens):
        if n < 0 or n > max_len:
            continue
        for h in range(KV):
            s = evict_ref(w[r, h], p[r, h], n, budget, recent, sinks)
            m = len(s)
            w1[r, h, :m], p1[r, h, :m], s1[r, h, :m] = w[r, h, s], p[r, h, s], s
            for d in np.flatnonzero(s != np.arange(m)):
                pd, ps = int(pool.table[r, d // pool.ps]), int(pool.table[r, s[d] // pool.ps])
                k0[pd, h, d % pool.ps], v0[pd, h, d % pool.ps] = k0[ps, h, s[d] % pool.ps], v0[ps, h, s[d] % pool.ps]
    want = [n if n < 0 or n > max_len else min(n, budget) for n in lens]
    assert lo.cpu().tolist() == want
    assert np.array_equal(wo.cpu().numpy(), w1, equal_nan=True) and np.array_equal(po.cpu().numpy(), p1)
    assert not src or np.array_equal(ss.cpu().numpy(), s1)
    assert torch.equal(pool.k, k0) and torch.equal(pool.v, v0)


def evict_inputs(rows, KV, n, seed, zeros=0.1):
    r = np.random.default_rng(seed)
    w = np.exp(2 * r.standard_normal((rows, KV, n)) - 3).astype(np.float32)
    w[r.random(w.shape) < zeros] = 0.0
    p = np.argsort(r.random((rows, KV, n)), -1).astype(np.int32)
    return w, p


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("KV,hd,n,budget,recent,sinks", [
    (2, 128, 100, 50, 10, 4), (4, 256, 65, 64, 8, 0), (8, 64, 300, 1, 0, 1), (1, 128, 1000, 999, 100, 4), (3, 64, 257, 0, 0, 0),
    (2, 128, 256, 256, 0, 0), (2, 128, 40, 4000, 2000, 9), (1, 64, 1, 0, 0, 0), (1, 64, 1, 1, 1, 0), (2, 64, 520, 260, 260, 0),
    (2, 64, 4500, 1111, 99, 3)])
def test_evict(KV, hd, n, budget, recent, sinks, dtype):
    rows = 3
    pool = Pool(rows, n, KV, hd, 16, dtype, seed=n)
    w, p = evict_inputs(rows, KV, n, n + budget)
    lens = [n, 0, (n + 1) // 2]
    check_evict(pool, w, p, lens, n, budget, recent, sinks)
    check_evict(pool, w, p, lens, n, budget, recent, sinks, in_place=True, src=False)


@pytest.mark.parametrize("ps,inner", [(1, "slots"), (8, "heads"), (256, "slots")])
def test_evict_page_sizes(ps, inner):
    w, p = evict_inputs(2, 3, 300, ps)
    check_evict(Pool(2, 300, 3, 64, ps, "bf16", seed=ps, inner=inner), w, p, [300, 133], 300, 90, 20, 2)


def test_evict_ties_and_special_weights():
    """All equal; few values; negative, infinite, NaN weights and both zeros; every position alike."""
    n = 700
    pool = Pool(1, n, 4, 64, 16, "f16", seed=4)
    _, p = evict_inputs(1, 4, n, 4)
    r = np.random.default_rng(4)
    for vals in ([1.0], [0.0, -0.0], [0.0, 1.0, 2.0], [math.nan, 1.0, -1.0, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45],
                 [math.nan], [-math.inf], [math.inf, 1.0]):
        w = r.choice(np.array(vals, np.float32), (1, 4, n))
        for budget in (1, 350, 699):
            check_evict(pool, w, p, [n], n, budget, 0, 0)
            check_evict(pool, w, p, [n], n, budget, budget // 2, budget // 4)
    w, _ = evict_inputs(1, 4, n, 5)
    check_evict(pool, w, np.zeros_like(p), [n], n, 350, 0, 0)
    check_evict(pool, w, np.full_like(p, 5), [n], n, 350, 1, 0)  # (all of them are the newest: the lowest slots stay)
    check_evict(pool, w, np.full_like(p, -2 ** 31), [n], n, 350, 0, 1)
    check_evict(pool, w, np.where(p % 2, 2 ** 31 - 1, -2 ** 31).astype(np.int32), [n], n, 350, 300, 1)


@pytest.mark.parametrize("n,budget", [(70, 66), (300, 150)])
def test_evict_in_place_over_many_workgroups(n, budget):
    """lens_out is lens, and a row's heads are spread over more workgroups than the chip holds at once: all of
    them see the length before the call."""
    rows, KV = 700, 3
    pool = Pool(rows, n, KV, 64, 16, "f16", seed=8)
    w, p = evict_inputs(rows, KV, n, 8)
    check_evict(pool, w, p, [n] * rows, n, budget, 5, 1, in_place=True)


def test_evict_to_nothing_in_place():
    pool = Pool(300, 33, 2, 64, 16, "bf16", seed=9)
    w, p = evict_inputs(300, 2, 33, 9)
    check_evict(pool, w, p, [33] * 299 + [-4], 33, 0, 0, 0, in_place=True)


@pytest.mark.parametrize("n", [9, 64, 1000, 1024, 1025, 4097, 17000])
def test_evict_a_few(n):
    """One to ten slots go: the smallest weights, their ties from the highest slot on, protected ones last."""
    pool = Pool(2, n, 3, 64, 16, "bf16", seed=n)
    w, p = evict_inputs(2, 3, n, n, zeros=0.3)
    w[:, 1] = np.random.default_rng(n).choice(np.array([math.nan, -1.0, -0.0, 0.0, math.inf, -math.inf], np.float32), (2, n))
    w[1, 2] = 1.0
    for drop in range(1, 11):
        if drop < n:
            check_evict(pool, w, p, [n, max(0, n - 3)], n, n - drop, min(3, n - drop), 0)
    check_evict(pool, w, np.full_like(p, 7), [n, n], n, n - 4, 1, 0)  # (every position the newest: the highest slots go)
    check_evict(pool, w, np.full_like(p, 7), [n, n - 1], n, n - 8, 0, 0)


def test_evict_one_slot_of_many():
    """Every step of a full cache: the one that goes, wherever it is."""
    n = 2049
    pool = Pool(1, n, 2, 128, 16, "f32", seed=5)
    for at in (0, 5, 1023, 2047, 2048):
        w, p = evict_inputs(1, 2, n, at, zeros=0.0)
        w[:, :, at] = 1e-9
        check_evict(pool, w, p, [n], n, n - 1, 0, 0)


def test_evict_long_rows():
    n = 70000
    pool = Pool(2, n, 1, 64, 64, "f16", seed=6)
    w, p = evict_inputs(2, 1, n, 6, zeros=0.4)
    check_evict(pool, w, p, [n, 65537], n, 30011, 500, 4)


def test_evict_bad_lengths_and_pages():
    pool = Pool(4, 64, 2, 64, 16, "f32", seed=7)
    w, p = evict_inputs(4, 2, 64, 7)
    check_evict(pool, w, p, [64, -1, 65, 2 ** 31 - 1], 64, 20, 5, 1)
    check_evict(pool, w, p, [64, -1, 65, 60], 64, 20, 5, 1, in_place=True)
    k0, v0 = pool.k.clone(), pool.v.clone()
    pool.p.table[:] = pool.k.shape[0]
    lens = torch.full((4,), 64, dtype=torch.int32, device="cuda")
    pool.p.evict(lens, 64, 20, dev(w), dev(p))
    assert torch.equal(pool.k, k0) and torch.equal(pool.v, v0) and (lens == 20).all()


# ------------------------------------------------------------------ together
def generate(pool, H, steps, budget, stream=None, seed=0, prompt=(40, 23, 1)):
    """A serving loop: prompts, then steps of append, attention and, where a row is over the budget, eviction.
    Yields each step's inputs and outputs after everything was enqueued."""
    rows, KV, hd = len(prompt), pool.k.shape[1], pool.k.shape[3]
    cap = pool.p.capacity
    g = torch.Generator().manual_seed(seed)
    cos, sin = (t.cuda() for t in rope_tables(4096, hd))
    sp = torch.zeros(rows, KV, cap, dtype=torch.int32, device="cuda")
    sw = torch.zeros(rows, KV, cap, device="cuda")
    lens = np.array(prompt, np.int32)
    at = np.array(prompt, np.int32)
    row = np.concatenate([np.full(n, r) for r, n in enumerate(prompt)]).astype(np.int32)
    slot = np.concatenate([np.arange(n) for n in prompt]).astype(np.int32)
    x = torch.randn(len(row), 2, KV, hd, generator=g)
    pool.p.append(x[:, 0].contiguous().cuda(), x[:, 1].contiguous().cuda(), dev(row), dev(slot), dev(slot), rope=(cos, sin),
                  slot_pos=sp, slot_weight=sw)
    for _ in range(steps):
        x = torch.randn(rows, 2, KV, hd, generator=g)
        q = torch.randn(rows, H, hd, generator=g)
        qr = pool.p.append(x[:, 0].contiguous().cuda(), x[:, 1].contiguous().cuda(), dev(np.arange(rows, dtype=np.int32)),
                           dev(lens), dev(at), q=q.cuda(), rope=(cos, sin), slot_pos=sp, slot_weight=sw)
        lens, at = lens + 1, at + 1
        out = pool.p.attention(qr, dev(lens), cap, weight_in=sw, weight_out=sw)
        yield x, q, qr, out, lens.copy(), at.copy(), sw, sp
        if lens.max() > budget:
            d = dev(lens)
            pool.p.evict(d, cap, budget, sw, sp, recent=8, sinks=2)
            lens = np.minimum(lens, budget)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_run_of_all_three(dtype):
    """Prompt, steps, weights, evictions every step once full: the cache holds exactly the tokens that the
    weights keep, each with its own rotation, and the attention reads them."""
    H, KV, hd, budget = 16, 2, 128, 32
    pool = Pool(3, 48, KV, hd, 16, dtype, fill=False)
    rope = rope_tables(4096, hd)
    for step, (x, q, qr, out, lens, at, sw, sp) in enumerate(generate(pool, H, 20, budget)):
        pos = sp.cpu().numpy()
        for r in range(3):
            n = int(lens[r])
            for h in range(KV):  # every position at most once, the newest and the first ones there
                held = set(pos[r, h, :n].tolist())
                first, newest = set(range(min(2, int(at[r])))), set(range(max(0, int(at[r]) - 8), int(at[r])))
                assert len(held) == n and first <= held and newest <= held
            k, v = pool.rows64(r, n)
            ref, _, tol, _ = attend64(qr[r].cpu(), k, v, hd ** -0.5)
            assert ((out[r].cpu().double() - ref).abs() <= tol).all()
            c, s = (t[at[r] - 1:at[r]] for t in rope)
            want, wtol = embed64(x[r:r + 1, 0], None, 0, c, s, False)
            half_step = torch.finfo(TYPES[dtype]).eps / 2
            assert ((k[:, n - 1] - want[0]).abs() <= wtol[0] * 2 + want[0].abs() * half_step + 2.0 ** -25).all()
        # a sequence's weights: each step gives every query head 1 in all
        if step == 0:
            assert torch.allclose(sw[:, :, :48].sum(-1).cpu(), torch.full((3, KV), H / KV), rtol=128 * U)  # (41 weights and their sum)


def test_streams_two_at_once():
    """Two caches on two streams at once, each with a workspace of its own, as alone."""
    pools = [Pool(4, 3000, 2, 128, 16, "f16", seed=s) for s in (1, 2)]
    q = [torch.randn(4, 16, 128, generator=torch.Generator().manual_seed(s)).cuda() for s in (1, 2)]
    lens = dev(np.array([3000, 1, 2222, 700], np.int32))
    want = [p.p.attention(x, lens, 3000) for p, x in zip(pools, q)]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for p, x, s in zip(pools, q, streams):
            with torch.cuda.stream(s):
                got.append(p.p.attention(x, lens, 3000))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


def test_graph_of_a_step():
    """A step captured once and replayed with other inputs, lengths and tables, eager work between: each
    replay as the eager calls on a copy."""
    H, KV, hd, cap = 16, 2, 128, 64
    a, b = Pool(3, cap, KV, hd, 16, "f16", seed=3), Pool(3, cap, KV, hd, 16, "f16", seed=3)
    g = torch.Generator().manual_seed(3)
    cos, sin = (t.cuda() for t in rope_tables(256, hd))

    def state(pool):
        return dict(p=pool.p, x=torch.zeros(3, KV, hd, device="cuda"), q=torch.zeros(3, H, hd, device="cuda"),
                    rows=torch.arange(3, dtype=torch.int32, device="cuda"), at=torch.zeros(3, dtype=torch.int32, device="cuda"),
                    pos=torch.zeros(3, dtype=torch.int32, device="cuda"), lens=torch.zeros(3, dtype=torch.int32, device="cuda"),
                    sp=torch.randint(0, 99, (3, KV, cap), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda(),
                    sw=torch.rand(3, KV, cap, generator=torch.Generator().manual_seed(2)).cuda(),
                    out=torch.zeros(3, H, hd, device="cuda"), qo=torch.zeros(3, H, hd, device="cuda"),
                    lo=torch.zeros(3, dtype=torch.int32, device="cuda"), src=torch.zeros(3, KV, cap, dtype=torch.int32, device="cuda"),
                    w1=torch.zeros(pool.p.attention_workspace(H, cap, True), dtype=torch.uint8, device="cuda"),
                    w2=torch.zeros(pool.p.evict_workspace(cap), dtype=torch.uint8, device="cuda"))

    def step(s):
        s["p"].append(s["x"], s["x"], s["rows"], s["at"], s["pos"], q=s["q"], rope=(cos, sin), q_out=s["qo"], slot_pos=s["sp"],
                      slot_weight=s["sw"])
        s["p"].attention(s["qo"], s["lens"], cap, out=s["out"], weight_in=s["sw"], weight_out=s["sw"], workspace=s["w1"])
        s["p"].evict(s["lens"], cap, 40, s["sw"], s["sp"], recent=4, sinks=1, lens_out=s["lo"], slot_src=s["src"],
                     workspace=s["w2"])

    sa, sb = state(a), state(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(sa)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(5):
        lens = np.array([[64, 40, 1], [41, 0, 64], [30, 64, 50], [64, 64, 64], [1, 2, 3]][i], np.int32)
        x, q = torch.randn(3, KV, hd, generator=g), torch.randn(3, H, hd, generator=g)
        for s in (sa, sb):
            s["x"].copy_(x)
            s["q"].copy_(q)
            s["lens"].copy_(torch.from_numpy(lens))
            s["at"].copy_(torch.from_numpy(np.maximum(lens, 1) - 1))
            s["pos"].copy_(torch.from_numpy(lens + 10 * i))
        for pool in (a, b):
            pool.p.table.copy_(pool.table.roll(i, 0))
        torch.cuda.synchronize()
        graph.replay()
        step(sb)
        torch.cuda.synchronize()
        for name in ("out", "qo", "lo", "src", "sp", "sw"):
            assert torch.equal(sa[name], sb[name]), (i, name)
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
        junk = torch.randn(1 << 20, device="cuda").sum()  # eager work between the replays
        assert torch.isfinite(junk)


def test_two_graphs_one_workspace():
    """Graphs of other sizes that use one workspace, replayed in turn."""
    pools = [Pool(4, 2000, 2, 128, 16, "f16", seed=21), Pool(1, 700, 4, 64, 32, "bf16", seed=22)]
    qs = [torch.randn(4, 16, 128, generator=torch.Generator().manual_seed(21)).cuda(),
          torch.randn(1, 12, 64, generator=torch.Generator().manual_seed(22)).cuda()]
    lens = [dev(np.array([2000, 3, 0, 1111], np.int32)), dev(np.array([700], np.int32))]
    tops = (2000, 700)
    ws = torch.zeros(max(p.p.attention_workspace(q.shape[1], n, True) for p, q, n in zip(pools, qs, tops)),
                     dtype=torch.uint8, device="cuda")
    outs = [torch.zeros_like(q) for q in qs]
    gots = [torch.zeros(p.p.rows, p.p.kv_heads, n, device="cuda") for p, n in zip(pools, tops)]
    wants = [torch.zeros_like(w) for w in gots]
    want = [p.p.attention(q, n, t, weight_out=w) for p, q, n, t, w in zip(pools, qs, lens, tops, wants)]
    graphs = []
    for p, q, n, t, o, w in zip(pools, qs, lens, tops, outs, gots):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            p.p.attention(q, n, t, out=o, weight_out=w, workspace=ws)
    for i in (0, 1, 0, 0, 1, 1, 0):
        outs[i].fill_(5.0)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i]) and torch.equal(gots[i], wants[i])


def test_stream_handles():
    """The default stream by its handles, and a stream that is none of torch's current ones."""
    lib, pool = ca.load_engine_lib(), Pool(2, 64, 2, 64, 16, "f32", seed=23)
    x = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(23)).cuda()
    row, slot = dev(np.array([0, 1], np.int32)), dev(np.array([5, 60], np.int32))
    for i, stream in enumerate((None, 1, 2, torch.cuda.Stream().cuda_stream)):
        torch.cuda.synchronize()
        y = x * (i + 2)
        torch.cuda.synchronize()
        rc = lib.chpe_paged_append(pool.p._c, 2, 0, None, 0, 0, y.data_ptr(), 128, y.data_ptr(), 128, None, None, 1e-6, None,
                                   None, 0, 0, 0, row.data_ptr(), slot.data_ptr(), slot.data_ptr(), None, None, None, 0, stream)
        assert rc == 0
        torch.cuda.synchronize()
        for r, s in ((0, 5), (1, 60)):
            assert torch.equal(pool.k[int(pool.table[r, s // 16]), :, s % 16], y[r])


def test_workspace_content_does_not_matter():
    pool = Pool(3, 2000, 2, 128, 16, "bf16", seed=4)
    q = torch.randn(3, 16, 128, generator=torch.Generator().manual_seed(4)).cuda()
    lens = dev(np.array([2000, 0, 77], np.int32))
    need = pool.p.attention_workspace(16, 2000)
    got = [pool.p.attention(q, lens, 2000, workspace=torch.full((need,), fill, dtype=torch.uint8, device="cuda"))
           for fill in (0, 255, 127)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2]) and (got[0][1] == 0).all()


def test_windows_fit_the_workspace():
    """The bytes do not depend on the window: no window's launch needs more."""
    lib = ca.load_engine_lib()
    pool = Pool(2, 4096, 2, 64, 16, "f16", seed=5)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)).cuda()
    lens = dev(np.array([4096, 1000], np.int32))
    need = pool.p.attention_workspace(4, 4096)
    buf = torch.full((need + 256,), 77, dtype=torch.uint8, device="cuda")
    for window in (0, 1, 31, 33, 100, 511, 1024, 2047, 4095, 4096):
        pool.p.attention(q, lens, 4096, window=window, workspace=buf[:need])
        assert (buf[need:] == 77).all()
    assert lib.chpe_paged_attention_workspace(pool.p._c, 4, 4096, 0) == need


def test_python_refusals():
    pool = Pool(2, 32, 2, 64, 16, "f16")
    p = pool.p
    q, lens = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    w, s = torch.zeros(2, 2, 32, device="cuda"), torch.zeros(2, 2, 32, dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 2, 64, device="cuda")
    for call in (lambda: p.attention(q.half(), lens, 32), lambda: p.attention(q, lens.long(), 32),
                 lambda: p.attention(q[:1], lens, 32), lambda: p.attention(q.cpu(), lens, 32),
                 lambda: p.attention(q, lens, 32, weight_in=w), lambda: p.attention(q, lens, 32, weight_out=w[..., :31]),
                 lambda: p.attention(q.transpose(0, 1), lens, 32), lambda: p.attention(q[:, :3], lens, 32),
                 lambda: p.append(x, x[:1], lens, lens, lens), lambda: p.append(x.half(), x, lens, lens, lens),
                 lambda: p.append(x, x, lens, lens, lens[:1]), lambda: p.append(x, x, lens, lens, lens, q=q.transpose(1, 2)),
                 lambda: p.append(x, x, lens, lens, lens, q_norm=q[0, 0, :32]),
                 lambda: p.evict(lens, 32, 16, w[..., :31].contiguous(), s), lambda: p.evict(lens, 32, 16, w, s.long()),
                 lambda: p.evict(lens, 32, 16, w, s, lens_out=lens[:1]), lambda: p.evict(lens, 32, -1, w, s),
                 lambda: p.evict(lens, 32, 16, w, s, recent=-1), lambda: p.attention(q, lens, 32, window=-1),
                 lambda: p.attention(q, lens, -1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ca.EngineError):
        p.attention(q, lens, 33, workspace=torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ca.EngineError):
        p.attention(q, lens, 32, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ca.EngineError):
        p.evict(lens, 32, 4, w, s, recent=4, sinks=1)
