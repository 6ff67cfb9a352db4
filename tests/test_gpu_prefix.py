"""The attention behind shared prefixes (chpe_amd.KvPages.prefix_attention) against softmax attention in 64 bits on the CPU,
and the operators of a serving loop of the hybrid model together: convolution, delta rule, append and both attentions.

Tolerances: test_gpu_paged.py's, which count the roundings of a softmax joined from parts."""
import numpy as np
import pytest
import torch

import chpe_amd as ca
from test_gpu_paged import TYPES, U, attend64

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.as_tensor(np.asarray(a)).to("cuda", torch.int32)


class Groups:
    """Groups of rows over one pool: (rows, prefix, lengths); rows of no group have prefix None."""

    def __init__(self, groups, KV, hd, ps, dtype, seed=0, inner="slots", own_tables=False):
        g = torch.Generator().manual_seed(seed)
        self.lens = [n for _, ls in groups for n in ls]
        self.prefix = [p or 0 for p, ls in groups for _ in ls]
        rows = len(self.lens)
        self.first_of = []
        self.max_prefix = max([p for p, _ in groups if p] + [0])
        self.max_rest = max([n - p for n, p in zip(self.lens, self.prefix)] + [0])
        per = max(1, -(-(self.max_prefix + self.max_rest) // ps), -(-max(self.lens) // ps))
        n = rows * per + 5
        shape = (n, KV, ps, hd) if inner == "slots" else (n, ps, KV, hd)
        k, v = (torch.randn(shape, generator=g).to(TYPES[dtype]).cuda() for _ in "kv")
        self.k, self.v = (t if inner == "slots" else t.transpose(1, 2) for t in (k, v))
        table = torch.randperm(n, generator=g)[:rows * per].reshape(rows, per).to(torch.int32)
        starts, at = [], 0
        for p, ls in groups:
            if p is not None:
                starts.append((at, at + len(ls), p))
            for i in range(len(ls)):
                self.first_of.append(at if p is not None else at + i)
                if p is not None and not own_tables:  # whole pages shared, as a server has them
                    table[at + i, :p // ps] = table[at, :p // ps]
            at += len(ls)
        self.table, self.ps = table, ps
        self.group_rows = dev(np.array([s[0] for s in starts] + [starts[-1][1] if starts else 0], np.int32))
        self.prefix_lens = dev(np.array([s[2] for s in starts], np.int32))
        self.p = ca.KvPages(self.k, self.v, table.cuda())

    def rows64(self, r, n):
        at = np.arange(n)
        head = self.table[self.first_of[r]].numpy()
        page = np.where(at < self.prefix[r], head[at // self.ps], self.table[r].numpy()[at // self.ps])
        take = lambda t: t[torch.from_numpy(page.astype(np.int64)).cuda(), :, torch.from_numpy(at % self.ps).cuda()].cpu().double().transpose(0, 1)  # noqa: E731
        return take(self.k), take(self.v)

    def run(self, q, lens=None, **kw):
        out = torch.full(q.shape, 7.0, device="cuda")
        work = torch.full((self.p.prefix_workspace(q.shape[1], self.prefix_lens.numel(), self.max_prefix, self.max_rest),), 255,
                          dtype=torch.uint8, device="cuda")
        return self.p.prefix_attention(q.cuda(), dev(np.asarray(self.lens if lens is None else lens, np.int32)), self.group_rows,
                                       self.prefix_lens, self.max_prefix, self.max_rest, out=out, workspace=work, **kw)

    def check(self, q, out, scale=None, rows=None):
        for r in range(len(self.lens)) if rows is None else rows:
            n = self.lens[r]
            if n == 0:
                assert (out[r] == 0).all(), r
                continue
            ref, _, tol, _ = attend64(q[r], *self.rows64(r, n), q.shape[2] ** -0.5 if scale is None else scale)
            err = (out[r].cpu().double() - ref).abs()
            assert (err <= tol + 1e-30).all(), (r, n, float((err / tol).max()))


def queries(rows, H, hd, seed=1):
    return torch.randn(rows, H, hd, generator=torch.Generator().manual_seed(seed)) * 2


MIXED = [(100, [101, 150, 100, 99, 1, 0]), (None, [77, 0, 5]), (64, [65]), (33, [40, 34, 160]), (0, [3, 31]), (257, [300, 258, 380])]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H,KV,hd", [(16, 2, 128), (16, 4, 256), (64, 8, 128), (5, 5, 64), (24, 8, 128), (12, 1, 64), (40, 1, 256),
                                     (33, 3, 64), (17, 1, 128)])
def test_layouts(H, KV, hd, dtype):
    """Groups of several rows, of one, without a prefix, rows of no group between them, rows shorter than their prefix."""
    g = Groups(MIXED[:1] + MIXED[2:], KV, hd, 16, dtype, seed=H)
    q = queries(len(g.lens), H, hd)
    g.check(q, g.run(q))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ps", [1, 8, 64, 512])
def test_pages_and_rows_of_no_group(dtype, ps):
    before = [(None, [77, 0, 5])] + [(100, [101, 150, 100, 99]), (64, [65])] + [(None, [130])]
    g = Groups(before, 2, 64, ps, dtype, seed=ps, inner="heads")
    q = queries(len(g.lens), 6, 64)
    g.check(q, g.run(q))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_the_prefix_lies_in_the_first_rows_pages(dtype):
    g = Groups([(48, [60, 49, 90])], 2, 64, 16, dtype, own_tables=True)
    q = queries(3, 4, 64)
    g.check(q, g.run(q))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,prefix", [(70, 1300), (3, 9000), (1, 5), (130, 40)])
def test_sizes(rows, prefix, dtype):
    """More queries than a workgroup's, more splits than one, both."""
    lens = [prefix + 1 + (7 * i) % 90 for i in range(rows)]
    g = Groups([(prefix, lens)], 2, 128, 32, dtype, seed=rows)
    q = queries(rows, 10, 128)
    out = g.run(q)
    g.check(q, out, rows=range(0, rows, 9))
    assert torch.equal(out, g.run(q))


def test_many_groups():
    """More groups than a wave's lanes, some of them empty."""
    groups = [(16 + i % 5, [20 + i % 7] * (i % 3)) for i in range(150)]
    g = Groups(groups, 1, 64, 8, "f16", seed=3)
    q = queries(len(g.lens), 2, 64)
    g.check(q, g.run(q))


def test_scale_and_no_rest():
    g = Groups([(40, [40, 33, 40])], 2, 64, 8, "bf16")
    assert g.max_rest == 0
    q = queries(3, 8, 64)
    g.check(q, g.run(q, scale=0.3), scale=0.3)


def test_lengths_and_groups_that_are_not_valid():
    """NaN for the rows that they concern, and what is read stays in bounds."""
    g = Groups([(100, [101, 150, 120]), (50, [60, 80]), (None, [40])], 2, 64, 16, "f16")
    q = queries(6, 4, 64)
    nan = lambda out: torch.isnan(out).flatten(1).all(1).tolist()  # noqa: E731
    lens = list(g.lens)
    lens[1], lens[4] = 100 + g.max_rest + 1, -5
    out = g.run(q, lens)
    assert nan(out) == [False, True, False, False, True, False]
    g.check(q, out, rows=[0, 2, 3, 5])
    for bad, which in ((101, [0, 1, 2]), (-1, [0, 1, 2])):
        keep = g.prefix_lens.clone()
        g.prefix_lens[0] = bad
        out = g.run(q)
        g.prefix_lens.copy_(keep)
        assert nan(out) == [i in which for i in range(6)]
        g.check(q, out, rows=[3, 4, 5])
    for rows in ([0, 7, 5], [0, 3, 2], [-2, 3, 5], [0, 3, 2 ** 31 - 1], [5, 4, 3]):
        keep = g.group_rows.clone()
        g.group_rows.copy_(dev(rows))
        g.run(q)
        torch.cuda.synchronize()
        g.group_rows.copy_(keep)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_pages_outside_the_pool(dtype):
    g = Groups([(64, [65, 90]), (64, [70, 20])], 2, 64, 16, dtype, own_tables=True)
    q = queries(4, 4, 64)
    table = g.table.clone()
    table[0, 2], table[1, 5], table[3, :] = -1, 10 ** 6, 99999  # a prefix's; a row's own; never looked at but its slots 64 ..
    g.p = ca.KvPages(g.k, g.v, table.cuda())
    out = g.run(q)
    assert torch.isnan(out).flatten(1).all(1).tolist() == [True, True, False, False]
    g.check(q, out, rows=[2, 3])
    g.p = ca.KvPages(g.k, g.v, torch.where(torch.arange(4)[:, None] == 0, g.table, table).cuda())
    out = g.run(q)
    assert torch.isnan(out).flatten(1).all(1).tolist() == [False, True, False, False]
    g.check(q, out, rows=[0, 2, 3])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_that_are_not_finite(hd, dtype):
    """Slots that a row does not see are never used; an infinite element of V that it sees makes its dim infinite."""
    g = Groups([(100, [104, 90, 130, 101])], 1, hd, 16, dtype)
    put = lambda t, r, slot, x: t.select(0, int(g.table[r, slot // 16])).select(1, slot % 16).copy_(x)  # noqa: E731
    for r in range(4):
        for slot in range(g.lens[r] if g.lens[r] >= 100 else 100, g.table.shape[1] * 16):
            put(g.k, r, slot, torch.full((1, hd), float("nan")))
            put(g.v, r, slot, torch.full((1, hd), float("inf")))
    q = queries(4, 3, hd)
    g.check(q, g.run(q))
    g.v[int(g.table[0, 95 // 16]), :, 95 % 16, 3] = float("inf")   # in the prefix: not row 1's, whose length is 90
    g.v[int(g.table[2, 120 // 16]), :, 120 % 16, 5] = -float("inf")
    out = g.run(q).cpu()
    inf = torch.isinf(out)
    assert inf[[0, 2, 3], :, 3].all() and (out[[0, 2, 3], :, 3] > 0).all() and (out[2, :, 5] == -float("inf")).all()
    inf[[0, 2, 3], :, 3] = False
    inf[2, :, 5] = False
    assert torch.isfinite(out[~inf & ~torch.isinf(out)]).all() and not inf.any() and not torch.isnan(out).any()
    g.check(q, out, rows=[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_queries_bad_pages_and_infinities(hd, dtype):
    """As the two tests above, with as many queries a group as share their K and V in LDS."""
    lens = [201, 200, 90, 240, 300, 0, 217, 299]
    g = Groups([(200, lens), (70, [71, 80])], 1, hd, 16, dtype, seed=hd, own_tables=True)
    put = lambda t, r, slot, x: t.select(0, int(g.table[r, slot // 16])).select(1, slot % 16).copy_(x)  # noqa: E731
    for r, n in enumerate(g.lens):  # what no row sees
        for slot in range(max(n, 200 if r == 0 else 70 if r == 8 else 0), g.table.shape[1] * 16):
            put(g.k, r, slot, torch.full((1, hd), float("nan")))
            put(g.v, r, slot, torch.full((1, hd), float("inf")))
    q = queries(10, 40, hd)
    out = g.run(q)
    g.check(q, out)
    # a page of the prefix: every row but those that end before it; a row's own
    table = g.table.clone()
    table[0, 9], table[8, 4] = -1, 1 << 30
    table[4, 15] = 10 ** 6
    g.p = ca.KvPages(g.k, g.v, table.cuda())
    nan = torch.isnan(g.run(q)).flatten(1).all(1).tolist()
    assert nan == [n > 144 for n in lens] + [True, True]
    table[0, 9], table[8, 4] = g.table[0, 9], g.table[8, 4]
    g.p = ca.KvPages(g.k, g.v, table.cuda())
    again = g.run(q)
    assert torch.isnan(again).flatten(1).all(1).tolist() == [r == 4 for r in range(10)]
    rest = [r for r in range(10) if r != 4]
    assert torch.equal(again[rest], out[rest])
    # an infinity in the prefix, past row 2's end
    g.p = ca.KvPages(g.k, g.v, g.table.cuda())
    g.v[int(g.table[0, 150 // 16]), :, 150 % 16, 7] = -float("inf")
    inf = g.run(q)
    sees = [r for r in range(8) if g.lens[r] > 150]
    assert (inf[sees, :, 7] == -float("inf")).all()
    inf[sees, :, 7] = out[sees, :, 7]
    assert torch.equal(inf, out)


def test_offsets_past_32_bits():
    """Pages whose offsets pass 2^32 bytes and 2^31 elements, for few queries a group and for many."""
    for rows, H in ((2, 4), (9, 32)):
        g = Groups([(64, [66 + i for i in range(rows)])], 1, 64, 16, "f16")
        n, page = g.k.shape[0], 16 * 64
        step = (1 << 32) // n // 8 * 8  # the last page's begins behind 3 * 2^30 elements
        far = [torch.empty(step * (n - 1) + page, dtype=torch.float16, device="cuda").as_strided(g.k.shape, (step, page, 64, 1))
               for _ in "kv"]
        for to, t in zip(far, (g.k, g.v)):
            to.copy_(t)
        q = queries(rows, H, 64)
        near = g.run(q)
        g.check(q, near)
        g.p = ca.KvPages(*far, g.table.cuda())
        assert torch.equal(g.run(q), near)
        del far, g


def test_many_queries_captured():
    """Groups that change between replays; a second graph with a workspace of its own at the same time."""
    g = Groups([(200, [201 + 7 * i for i in range(9)])], 2, 128, 16, "bf16", seed=6)
    q = queries(9, 64, 128).cuda()
    lens, runs = dev(np.asarray(g.lens, np.int32)), []
    for _ in range(2):
        out = torch.empty_like(q)
        work = torch.empty(g.p.prefix_workspace(64, 1, g.max_prefix, g.max_rest), dtype=torch.uint8, device="cuda")
        run = lambda out=out, work=work: g.p.prefix_attention(q, lens, g.group_rows, g.prefix_lens, g.max_prefix, g.max_rest,  # noqa: E731
                                                              out=out, workspace=work)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        runs.append((graph, out, run))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for groups, prefix in (([0, 9], 200), ([0, 4], 150), ([3, 9], 199), ([9, 9], 200), ([0, 9], 201)):
        g.group_rows.copy_(dev(groups))
        g.prefix_lens.fill_(prefix)
        runs[0][2]()
        want = runs[0][1].clone()
        for _, out, _ in runs:
            out.fill_(0)
        torch.cuda.synchronize()
        for (graph, _, _), s in zip(runs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, _ in runs:
            assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)), groups


def test_as_without_groups():
    """No groups: chpe_paged_attention's results up to the order of the joins."""
    g = Groups([(None, [300, 1, 77, 0])], 4, 128, 16, "bf16")
    q = queries(4, 16, 128)
    out = g.run(q)
    g.check(q, out)
    one = g.p.attention(q.cuda(), dev(np.asarray(g.lens, np.int32)), 300)
    scale = max(1.0, float(one.abs().max()))
    assert (out - one).abs().max() <= 2 * (2 * (128 * U + 2.0 ** -21) * 40 + 332 * U) * scale


def test_streams_and_graphs():
    g = Groups([(200, [201, 250, 230]), (64, [90])], 2, 128, 16, "f16", seed=5)
    q = queries(4, 8, 128).cuda()
    lens = dev(np.asarray(g.lens, np.int32))
    out = torch.empty_like(q)
    work = torch.empty(g.p.prefix_workspace(8, 2, g.max_prefix, g.max_rest), dtype=torch.uint8, device="cuda")
    run = lambda: g.p.prefix_attention(q, lens, g.group_rows, g.prefix_lens, g.max_prefix, g.max_rest, out=out, workspace=work)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for groups, prefixes, ls in (([0, 3, 4], [200, 64], g.lens), ([0, 1, 4], [5, 64], [6, 80, 64, 90]), ([2, 2, 4], [9, 200], [20, 50, 201, 250])):
        g.group_rows.copy_(dev(groups))
        g.prefix_lens.copy_(dev(prefixes))
        lens.copy_(dev(ls))
        q.normal_()
        run()
        want = out.clone()
        out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(out).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = g.p.prefix_attention(q, lens, g.group_rows, g.prefix_lens, g.max_prefix, g.max_rest)
    s.synchronize()
    assert torch.equal(other, want)


def test_what_python_refuses():
    g = Groups([(16, [20, 30])], 2, 64, 8, "f32")
    q, lens = queries(2, 4, 64).cuda(), dev(np.asarray(g.lens, np.int32))
    call = lambda **kw: g.p.prefix_attention(**{**dict(q=q, lens=lens, group_rows=g.group_rows, prefix_lens=g.prefix_lens,  # noqa: E731
                                                       max_prefix=16, max_rest=14), **kw})
    call()
    for bad in (dict(q=q[0]), dict(q=q.half()), dict(q=q.cpu()), dict(lens=lens[:1]), dict(lens=lens.long()), dict(group_rows=lens[:1]),
                dict(prefix_lens=lens), dict(max_prefix=-1), dict(max_rest=2 ** 32), dict(max_rest=10 ** 6), dict(out=q[:1])):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ca.EngineError):
        call(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


# ------------------------------------------------------------------ as a serving loop has them
def test_a_prompt_forked_into_samples():
    """One prompt through a linear-attention layer and a full-attention layer, then three samples of it for four steps: the
    layers' state and pages are shared from the prompt on.  Every sample has the results of a run of its own, token by
    token from nothing."""
    NK, NV, hd, H, KV, n, samples, steps = 2, 4, 64, 4, 2, 75, 3, 4
    C = (2 * NK + NV) * hd
    rng = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=rng).cuda()  # noqa: E731
    w, A_log, bias, norm = rand(C, 4), rand(NV), rand(NV), 1 + 0.1 * rand(hd)
    total = n + samples * steps
    x, ab, z = rand(total, C), rand(total, 2 * NV), rand(total, NV, hd)          # the projections' outputs: the prompt's tokens,
    q, k, v = rand(total, H, hd), rand(total, KV, hd), rand(total, KV, hd)       # then the samples', step by step
    cos, sin = (f(torch.outer(torch.arange(n + steps).float(), 1e4 ** (-torch.arange(hd // 2) / (hd // 2)))).cuda() for f in (torch.cos, torch.sin))

    def layer(conv, states, at, starts, src, dst):
        y = conv.apply(x[at], None if starts is None else dev(starts), dev(src), dev(dst))
        qq, kk, vv = (t.unflatten(1, (-1, hd)) for t in y.split([NK * hd, NK * hd, NV * hd], 1))
        args = (qq, kk, vv, ab[at][:, :NV], ab[at][:, NV:], A_log, bias)
        kw = dict(z=z[at], norm_w=norm)
        return states.step(*args, dev(src), dev(dst), **kw) if starts is None else states.prompt(*args, dev(starts), dev(src), dev(dst), **kw)

    def pools(slots, pages, rows, per):
        return (ca.DeltaConv(torch.zeros(slots, C, 3, device="cuda"), w), ca.DeltaStates(torch.zeros(slots, NV, hd, hd, device="cuda"), NK),
                torch.zeros(pages, KV, 16, hd, device="cuda", dtype=torch.float16), torch.zeros(pages, KV, 16, hd, device="cuda", dtype=torch.float16))

    # together
    conv, states, pk, pv = pools(samples + 1, 40, samples, 6)
    tok = torch.arange(n, device="cuda")
    shared = n // 16  # whole pages; the samples' next page gets a copy of what the prompt left in its last one
    table = torch.tensor([[*range(shared), 10 + 2 * s, 11 + 2 * s] for s in range(samples)], dtype=torch.int32).cuda()
    cache = ca.KvPages(pk, pv, table)
    got_d = [layer(conv, states, tok, [0, n], [-1], [samples])]
    pos = tok.to(torch.int32)
    cache.append(k[:n], v[:n], torch.zeros_like(pos), pos, pos, q=q[:n], rope=(cos, sin))
    for s in range(1, samples):
        pk[10 + 2 * s], pv[10 + 2 * s] = pk[10], pv[10]
    got_a = []
    src = [samples] * samples
    for i in range(steps):
        at = n + samples * i + torch.arange(samples, device="cuda")
        got_d.append(layer(conv, states, at, None, src, range(samples)))
        src = list(range(samples))
        here = torch.full((samples,), n + i, dtype=torch.int32, device="cuda")
        qr = cache.append(k[at], v[at], dev(src), here, here, q=q[at], rope=(cos, sin))
        got_a.append(cache.prefix_attention(qr, here + 1, dev([0, samples]), dev([16 * shared]), 16 * shared, 16 + steps))

    # each sample alone, token by token
    for s in range(samples):
        conv, states, pk, pv = pools(1, 8, 1, 8)
        cache = ca.KvPages(pk, pv, torch.arange(8, dtype=torch.int32, device="cuda")[None])
        for t in range(n + steps):
            at = torch.tensor([t if t < n else n + samples * (t - n) + s], device="cuda")
            d = layer(conv, states, at, None, [-1] if t == 0 else [0], [0])
            here = torch.tensor([t], dtype=torch.int32, device="cuda")
            qr = cache.append(k[at], v[at], dev([0]), here, here, q=q[at], rope=(cos, sin))
            mine = got_d[0][t:t + 1] if t < n else got_d[1 + t - n][s:s + 1]
            # both are within the recurrence's bound (8 sqrt(D T) + 64) u of its largest value, 4 at most here, and the norm divides
            # by the root mean square of the outputs, which is above 1 / 8 of that
            assert (mine - d).abs().max() <= 2 * (8 * (hd * (t + 1)) ** 0.5 + 64) * U * 4 * 8 * 4, (s, t)
            if t >= n:
                a = cache.attention(qr, here + 1, n + steps)
                # 2 (hd u + 2^-21) of scores below 64, and the sums' (n + 16) u, of outputs below 4; twice
                assert (got_a[t - n][s] - a[0]).abs().max() <= 2 * 4 * (2 * (hd * U + 2.0 ** -21) * 64 + (n + 32) * U), (s, t)
