"""The gated delta rule over a pool of states (chpe_amd.DeltaStates) and its convolution (chpe_amd.DeltaConv) against
plain recurrences in 64 bits on the CPU: types, head layouts, strides, lengths from none to several chunks, slots that are
read, left, shared, new, not kept or outside the pool, rows that are left out, values that are not finite, streams
and graphs.

Tolerances.  u = 2^-24.  Every stored value of a head (an output, a state's element) is a sum whose terms are bounded by
the head's largest |value| M, and a token's update adds sums of D products to it; the factors I - b k k^T and the decays
are contractions, so errors of earlier tokens do not grow.  Roundings are off by up to u relative, in either direction, a sum
of D products over T tokens by c u sqrt(D T) M with c = 8 for the largest of a few thousand; what is not a sum of
products (norms, exponentials, gates: up to 40 roundings, and up to 20 u of a log decay of -20) is in the 64 u M that
come on top.  An output of a 16-bit type is off by half a step more.  The gated norm divides by the head's root mean
square r: an error e becomes |w silu(z)| e (1 + |o| / r) / r, and 64 u of the result."""
import numpy as np
import pytest
import torch

import chpe_amd as ca

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
EPS = 1e-5


def dev(a, dt=torch.int32):
    return torch.as_tensor(np.asarray(a)).to("cuda", dt)


class Layer:
    """Inputs of `n` tokens, on the GPU as parts of wider rows, on the CPU in 64 bits."""

    def __init__(self, n, NK, NV, hd, dtype, gate, seed, pad=0, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.n, self.NK, self.NV, self.hd, self.dtype, self.gate = n, NK, NV, hd, dtype, gate
        dt, width = TYPES[dtype], (2 * NK + NV) * hd
        wide = (torch.randn(n, width + pad, generator=g) * scale).to(dt).cuda()
        self.q, self.k = (wide[:, i * NK * hd:(i + 1) * NK * hd].unflatten(1, (NK, hd)) for i in range(2))
        self.v = wide[:, 2 * NK * hd:width].unflatten(1, (NV, hd))
        ab = torch.randn(n, 2 * NV + 3, generator=g).cuda()
        self.a, self.b = ab[:, :NV], ab[:, NV:2 * NV]
        self.A_log = (torch.rand(NV, generator=g) * 6 - 4).cuda()
        self.dt_bias = torch.randn(NV, generator=g).cuda()
        self.z = torch.randn(n, NV, hd, generator=g).to(dt).cuda() if gate else None
        self.norm_w = (1 + 0.2 * torch.randn(hd, generator=g)).cuda() if gate else None

    def args(self):
        return self.q, self.k, self.v, self.a, self.b, self.A_log, self.dt_bias

    def kw(self):
        return dict(z=self.z, norm_w=self.norm_w, eps=EPS)

    def row64(self, lo, hi, S):
        """The recurrence over tokens lo .. hi - 1 from S [NV][hd][hd]: outputs before the norm, the state."""
        cpu = lambda t: t[lo:hi].cpu().double().numpy()  # noqa: E731
        q, k, v, a, b = (cpu(t) for t in (self.q, self.k, self.v, self.a, self.b))
        A, bias = np.exp(self.A_log.cpu().double().numpy()), self.dt_bias.cpu().double().numpy()
        with np.errstate(all="ignore"):
            k, q = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (k, q))
            k, q = (x.repeat(self.NV // self.NK, 1) for x in (k, q / np.sqrt(self.hd)))
            decay, beta = np.exp(-A * np.logaddexp(0.0, a + bias)), 1 / (1 + np.exp(-b))
            S, out = S.copy(), np.zeros((hi - lo, self.NV, self.hd))
            for t in range(hi - lo):
                S *= decay[t][:, None, None]
                d = (v[t] - np.einsum("hij,hi->hj", S, k[t])) * beta[t][:, None]
                S += k[t][:, :, None] * d[:, None]
                out[t] = np.einsum("hij,hi->hj", S, q[t])
        return out, S

    def check(self, lo, hi, out, got_S, S0, what):
        ref, S = self.row64(lo, hi, S0)
        T = hi - lo
        each = lambda M: (8 * np.sqrt(self.hd * max(T, 1)) + 64) * U * M  # noqa: E731
        tol_S = each(np.maximum(np.abs(S).max((1, 2)), np.abs(S0).max((1, 2))))
        if got_S is not None:
            err = np.abs(got_S.cpu().double().numpy() - S)
            assert (err <= tol_S[:, None, None]).all(), (what, "state", float((err / tol_S[:, None, None]).max()))
        if T == 0:
            return
        # an output is a sum of D of the state's elements times a query of length 1 / sqrt(D)
        tol = np.broadcast_to(np.maximum(each(np.abs(ref).max((0, 2))), tol_S)[None, :, None], ref.shape).copy()
        if self.gate:
            w, z = self.norm_w.cpu().double().numpy(), self.z[lo:hi].cpu().double().numpy()
            gate, rms = w * z / (1 + np.exp(-z)), np.sqrt((ref * ref).mean(-1, keepdims=True) + EPS)
            tol = np.abs(gate) * tol / rms * (1 + np.abs(ref) / rms) + 64 * U * np.abs(ref / rms * gate)
            ref = ref / rms * gate
        tol = tol + HALF[self.dtype] * (np.abs(ref) + tol) + 2.0 ** -25 * (self.dtype == "f16")
        err = np.abs(out[lo:hi].cpu().double().numpy() - ref)
        assert (err <= tol).all(), (what, "out", float((err / tol).max()))


def pool(n, NV, hd, seed, room=0):
    g = torch.Generator().manual_seed(seed + 100)
    wide = torch.randn(n, NV * hd * hd + room, generator=g).cuda() * 0.5
    return wide, wide[:, :NV * hd * hd].unflatten(1, (NV, hd, hd))


def before(state, slot):
    x = state[max(slot, 0)].cpu().double().numpy()
    return x if slot >= 0 else np.zeros_like(x)


LAYOUTS = [(16, 32, 128), (3, 9, 128), (1, 6, 128), (2, 2, 64), (4, 16, 64), (5, 5, 64)]


# ------------------------------------------------------------------ one token per row
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("NK,NV,hd", LAYOUTS)
def test_step(NK, NV, hd, dtype, gate):
    L = Layer(6, NK, NV, hd, dtype, gate, seed=NV, pad=16)
    wide, state = pool(9, NV, hd, NV, room=8)
    old = wide.clone()
    slots, to = [4, -1, 0, 8, 4, 2], [4 + 1, 1, 0, 3, 6, -1]  # another, new, its own, two from one, not kept
    h = ca.DeltaStates(state, NK)
    out = h.step(*L.args(), dev(slots), dev(to), **L.kw())
    assert out.dtype is TYPES[dtype]
    for r, (s, t) in enumerate(zip(slots, to)):
        L.check(r, r + 1, out, state[t] if t >= 0 else None, before(old[:, :NV * hd * hd].unflatten(1, (NV, hd, hd)), s), r)
    kept = [i for i in range(9) if i not in to]
    assert torch.equal(wide[kept], old[kept])  # no other slot, and nothing between the slots, is touched
    assert torch.equal(wide[:, NV * hd * hd:], old[:, NV * hd * hd:])


def test_step_is_the_engines_step():
    """The same arithmetic as the decode step's kernels on one layer of the hybrid model's layout."""
    L = Layer(1, 16, 32, 128, "f32", True, seed=3)
    _, state = pool(1, 32, 128, 3)
    S0 = state[0].cpu().numpy()
    out = ca.DeltaStates(state, 16).step(*L.args(), dev([0]), **L.kw())
    args = [t[0].cpu().numpy() for t in L.args()[:5]] + [t.cpu().numpy() for t in L.args()[5:]]
    ref, S = ca.gpu_deltanet_step(*args, S0, z=L.z[0].cpu().numpy(), norm_w=L.norm_w.cpu().numpy(), eps=EPS)
    # both within the bound of the recurrence's roundings: 8 sqrt(128) + 64 of u, twice, of the largest value
    bound = 2 * (8 * np.sqrt(128) + 64) * U
    assert np.abs(state[0].cpu().numpy() - S).max() <= bound * np.abs(S).max()
    assert np.abs(out[0].cpu().numpy() - ref).max() <= 16 * bound * np.abs(ref).max()


def test_slots_outside_the_pool():
    """A state before that is none: NaN, in what comes of it alone; a state after that has no slot: not kept."""
    NK, NV, hd = 2, 4, 64
    for n in (1, 3, 70):  # step, token by token, chunks
        L = Layer(3 * n, NK, NV, hd, "f32", False, seed=n)
        wide, state = pool(3, NV, hd, 1)
        old = state.clone()
        h = ca.DeltaStates(state, NK)
        starts = dev([0, n, 2 * n, 3 * n])
        slot_in, slot_out = dev([0, 3, -2]), dev([2, 1, 7])
        out = (h.step(*L.args(), slot_in, slot_out) if n == 1 else h.prompt(*L.args(), starts, slot_in, slot_out))
        L.check(0, n, out, state[2], before(old, 0), n)
        assert torch.isnan(out[n:]).all() and torch.isnan(state[1]).all() and torch.equal(state[0], old[0])


# ------------------------------------------------------------------ prompts
LENGTHS = [65, 1, 0, 8, 9, 63, 64, 2, 129, 16, 17, 200, 48, 127]


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("NK,NV,hd", LAYOUTS)
def test_prompt(NK, NV, hd, dtype, gate):
    lens = LENGTHS if NV < 32 else LENGTHS[::2]
    skip = 5  # tokens of no row, before the first and behind the last
    starts = skip + np.concatenate(([0], np.cumsum(lens)))
    n = int(starts[-1]) + skip
    L = Layer(n, NK, NV, hd, dtype, gate, seed=NV + 1, pad=8)
    rows = len(lens)
    wide, state = pool(2 * rows, NV, hd, NV, room=4)
    old = wide.clone()
    old_state = old[:, :NV * hd * hd].unflatten(1, (NV, hd, hd))
    order = np.random.default_rng(NV).permutation(2 * rows)
    slots, to = order[:rows].copy(), order[rows:].copy()
    slots[1] = -1
    slots[3] = slots[0]  # two from one
    to[4] = slots[4]     # its own
    to[5] = -1           # not kept
    h = ca.DeltaStates(state, NK)
    out = torch.full((n, NV, hd), 3.0, dtype=TYPES[dtype], device="cuda")
    ws = torch.full((h.prompt_workspace(n, rows, gate),), 255, dtype=torch.uint8, device="cuda")
    h.prompt(*L.args(), dev(starts), dev(slots), dev(to), out=out, workspace=ws, **L.kw())
    for r in range(rows):
        L.check(int(starts[r]), int(starts[r + 1]), out, state[to[r]] if to[r] >= 0 else None, before(old_state, slots[r]), (r, lens[r]))
    assert (out[:skip] == 3.0).all() and (out[n - skip:] == 3.0).all()
    kept = [i for i in range(2 * rows) if i not in to]
    assert torch.equal(wide[kept], old[kept]) and torch.equal(wide[:, NV * hd * hd:], old[:, NV * hd * hd:])


@pytest.mark.parametrize("rows", [1, 5, 9])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_prompt_columns(dtype, rows):
    """Every number of columns a workgroup: by the rows, at the widest layout."""
    NK, NV, hd = 8, 32, 128
    lens = [100] * rows
    starts = np.concatenate(([0], np.cumsum(lens)))
    L = Layer(int(starts[-1]), NK, NV, hd, dtype, False, seed=rows)
    _, state = pool(rows, NV, hd, rows)
    old = state.clone()
    out = ca.DeltaStates(state, NK).prompt(*L.args(), dev(starts), dev(np.arange(rows)))
    for r in range(0, rows, 4):
        L.check(int(starts[r]), int(starts[r + 1]), out, state[r], before(old, r), r)


@pytest.mark.parametrize("NK,NV,hd,dtype", [(16, 32, 128, "f32"), (16, 32, 128, "bf16"), (8, 64, 64, "f16"), (2, 4, 64, "f32")])
def test_prompt_of_short_rows(NK, NV, hd, dtype):
    """Lengths about those from which on a row runs in chunks, in few rows and in many."""
    for lens in ([8, 9, 16, 17, 1, 0, 7, 15, 18, 64, 65, 8, 16, 17, 2, 9], [17, 8], [9], [8], [16]):
        starts = np.concatenate([[0], np.cumsum(lens)])
        L = Layer(int(starts[-1]), NK, NV, hd, dtype, True, seed=len(lens))
        _, state = pool(len(lens), NV, hd, 5)
        old = state.clone()
        out = ca.DeltaStates(state, NK).prompt(*L.args(), dev(starts), dev(np.arange(len(lens))), **L.kw())
        for r, n in enumerate(lens):
            L.check(starts[r], starts[r + 1], out, state[r], before(old, r), (lens, r))


@pytest.mark.parametrize("rows", [64, 69])
def test_prompt_of_many_rows(rows):
    """As many rows as are taken by their lengths, and more."""
    lens = ([20, 3, 70, 64, 0, 129] * 12)[:rows]
    starts = np.concatenate([[0], np.cumsum(lens)])
    L = Layer(int(starts[-1]), 8, 16, 64, "bf16", False, seed=rows)
    _, state = pool(rows, 16, 64, 5)
    old = state.clone()
    out = ca.DeltaStates(state, 8).prompt(*L.args(), dev(starts), dev(np.arange(rows)))
    for r in range(rows):
        L.check(starts[r], starts[r + 1], out, state[r], before(old, r), r)


def test_prompt_in_pieces_and_again():
    """A prompt in one call, in two, and the same call again: the last bit for bit, the pieces within the roundings."""
    NK, NV, hd, n = 4, 8, 128, 150
    L = Layer(n, NK, NV, hd, "f32", False, seed=5)
    _, state = pool(4, NV, hd, 5)
    S0 = before(state, 0)
    h = ca.DeltaStates(state, NK)
    a = h.prompt(*L.args(), dev([0, n]), dev([0]), dev([1])).clone()
    b = h.prompt(*L.args(), dev([0, n]), dev([0]), dev([2]))
    assert torch.equal(a, b) and torch.equal(state[1], state[2])
    out = torch.empty_like(a)
    for lo, hi, s in ((0, 77, 0), (77, 85, 3), (85, n, 3)):
        part = tuple(t[lo:hi] for t in L.args()[:5]) + L.args()[5:]
        out[lo:hi] = h.prompt(*part, dev([0, hi - lo]), dev([s]), dev([3]))
    L.check(0, n, out, state[3], S0, "pieces")
    L.check(0, n, a, state[1], S0, "whole")


def test_rows_that_are_left_out():
    """A range that does not lie in the tokens: nothing of it is read or written; the other rows are what they are."""
    NK, NV, hd = 1, 2, 64
    for starts in ([0, 70, 60, 100], [0, 40, 101, 100], [-3, 5, 5, 90], [0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], [100, 0, -1, -2]):
        L = Layer(100, NK, NV, hd, "f32", False, seed=1)
        _, state = pool(6, NV, hd, 1)
        old = state.clone()
        out = torch.full((100, NV, hd), 3.0, device="cuda")
        ca.DeltaStates(state, NK).prompt(*L.args(), dev(starts), dev([0, 1, 2]), dev([3, 4, 5]), out=out)
        conv = torch.zeros(6, 8, 3, device="cuda")
        ca.DeltaConv(conv, torch.ones(8, 4, device="cuda")).apply(torch.ones(100, 8, device="cuda"), dev(starts), dev([0, 1, 2]), dev([3, 4, 5]))
        torch.cuda.synchronize()
        for r in range(3):
            lo, hi = starts[r], starts[r + 1]
            if not 0 <= lo <= hi <= 100:
                assert torch.equal(state[3 + r], old[3 + r]), (starts, r)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hd", [64, 128])
def test_equal_keys_and_full_gates(hd, dtype):
    """The worst triangular systems: the same key all the time, b near 1, no decay; and keys that alternate."""
    NK, NV, n = 1, 3, 130
    for kind in ("same", "two", "tiny"):
        L = Layer(n, NK, NV, hd, dtype, False, seed=2)
        if kind == "same":
            L.k[:] = L.k[:1].clone()
        elif kind == "two":
            L.k[::2], L.k[1::2] = L.k[:1].clone(), -L.k[1:2].clone()
        else:
            L.k *= 2.0 ** -12
        L.b[:] = 12.0
        L.A_log[:] = -30.0
        _, state = pool(1, NV, hd, 2)
        S0 = before(state, 0)
        out = ca.DeltaStates(state, NK).prompt(*L.args(), dev([0, n]), dev([0]))
        L.check(0, n, out, state[0], S0, kind)


def test_decays():
    """Decays from one to none within a chunk: sums of logs in the thousands leave their differences alone."""
    NK, NV, hd, n = 1, 4, 64, 140
    L = Layer(n, NK, NV, hd, "f32", False, seed=9)
    L.A_log[:] = torch.tensor([-20.0, 3.0, 6.0, 40.0])
    L.a[:] = torch.where(torch.rand(n, NV, generator=torch.Generator().manual_seed(1)) < 0.2, 5.0, -30.0).cuda()
    L.a[7, 2], L.a[8, 2], L.b[9, 1], L.b[10, 1] = np.inf, -np.inf, np.inf, -np.inf
    _, state = pool(1, NV, hd, 9)
    S0 = before(state, 0)
    out = ca.DeltaStates(state, NK).prompt(*L.args(), dev([0, n]), dev([0]))
    L.check(0, n, out, state[0], S0, "decays")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("what", ["v", "k", "q", "a", "b"])
def test_values_that_are_not_finite(what, bad, dtype):
    """They reach what the recurrence lets them reach: not an earlier token, a value's not another column."""
    NK, NV, hd, n, at = 2, 4, 64, 150, 100
    clean, L = (Layer(n, NK, NV, hd, dtype, False, seed=4) for _ in range(2))
    if what in "vkq":
        getattr(L, what)[at, 1, 5] = bad
    else:
        getattr(L, what)[at, 1] = bad
    _, state = pool(2, NV, hd, 4)
    S0, h = before(state, 0), ca.DeltaStates(state, NK)
    out = h.prompt(*L.args(), dev([0, n]), dev([0]), dev([1]))
    ref, S = L.row64(0, n, S0)
    assert np.isfinite(ref[:at]).all()
    fine = np.isfinite(ref)
    got = out.cpu().double().numpy()
    assert (np.isfinite(got) | ~fine).all(), "a value that the recurrence leaves finite is not"
    assert (~np.isfinite(got) | fine).all(), "a value that the recurrence does not leave finite is"
    assert (np.isfinite(state[1].cpu().numpy()) == np.isfinite(S)).all()
    M = np.abs(np.where(fine, ref, 0)).max()
    tol = (8 * np.sqrt(hd * n) + 64) * U * max(M, np.abs(S0).max()) + HALF[dtype] * np.abs(np.where(fine, ref, 0))
    assert (np.where(fine, np.abs(got - ref), 0) <= tol + 2.0 ** -25).all()


@pytest.mark.parametrize("scale", [1e-20, 1e17])
def test_large_and_small_keys(scale):
    """Keys whose squares leave f32's range, or the products': as the recurrence in f32 has them."""
    NK, NV, hd, n = 1, 2, 128, 70
    L = Layer(n, NK, NV, hd, "f32", False, seed=6)
    L.k *= scale
    _, state = pool(1, NV, hd, 6)
    S0 = before(state, 0)
    out = ca.DeltaStates(state, NK).prompt(*L.args(), dev([0, n]), dev([0]))
    L.check(0, n, out, state[0], S0, scale)


def test_strides_past_32_bits():
    """Slots and tokens whose offsets pass 2^32 bytes and 2^31 elements."""
    NK, NV, hd = 1, 1, 64
    big = torch.empty(1 << 30, device="cuda")  # 4 GiB of floats, three times
    slots = big.as_strided((3, NV, hd, hd), ((1 << 29) - 4096, hd * hd, hd, 1))
    slots.normal_()
    L = Layer(3, NK, NV, hd, "f32", False, seed=8)
    rows = torch.empty((1 << 30) + 4096, device="cuda")
    L.k = rows.as_strided((3, NK, hd), (1 << 29, hd, 1)).normal_()
    old = slots.clone()
    h = ca.DeltaStates(slots, NK)
    out = h.step(*L.args(), dev([2, 1, 0]), dev([2, 1, 0]))
    for r, s in enumerate((2, 1, 0)):
        L.check(r, r + 1, out, slots[s], before(old, s), r)
    now = slots.clone()
    out = h.prompt(*L.args(), dev([0, 0, 0, 3]), dev([0, 1, 2]))
    L.check(0, 3, out, slots[2], before(now, 2), "prompt")


# ------------------------------------------------------------------ the convolution
@pytest.mark.parametrize("taps", range(2, 9))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv(dtype, taps):
    """u sqrt(taps) at most of the sum of |w x|, and of SiLU 8 u; half a step of the type on top."""
    C, P, lens = 1032, taps - 1, [5, 0, 1, 2, 16, 17, 33, 64, 3, 100]
    g = torch.Generator().manual_seed(taps)
    starts = 2 + np.concatenate(([0], np.cumsum(lens)))
    n = int(starts[-1]) + 3
    wide = torch.randn(n, C + 24, generator=g).to(TYPES[dtype]).cuda()
    x, w = wide[:, 8:C + 8], torch.randn(C, taps, generator=g).cuda()
    rows = len(lens)
    state = torch.randn(2 * rows, C, P, generator=g).cuda()
    old = state.clone()
    slots, to = np.arange(rows), rows + np.arange(rows)
    slots[3], to[4], to[5], slots[6] = -1, 4, -1, 0
    y = torch.full((n, C + 8), 3.0, dtype=TYPES[dtype], device="cuda")
    out = ca.DeltaConv(state, w).apply(x, dev(starts), dev(slots), dev(to), out=y[:, :C])
    xd, wd = x.cpu().double().numpy(), w.cpu().double().numpy()
    for r, m in enumerate(lens):
        lo = int(starts[r])
        seq = np.concatenate((before(old, int(slots[r])), xd[lo:lo + m].T), 1)
        s = sum(wd[:, j, None] * seq[:, j:j + m] for j in range(taps))
        mag = sum(np.abs(wd[:, j, None] * seq[:, j:j + m]) for j in range(taps))
        ref = s / (1 + np.exp(-s))
        tol = 1.1 * taps * U * mag + 8 * U * np.abs(ref)
        tol = tol + HALF[dtype] * (np.abs(ref) + tol) + 2.0 ** -25 * (dtype == "f16")
        err = np.abs(out[lo:lo + m].cpu().double().numpy().T - ref)
        assert (err <= tol).all(), (r, m, float((err / tol).max()))
        if to[r] >= 0:
            assert np.array_equal(state[int(to[r])].cpu().double().numpy(), seq[:, m:]), r
    assert (y[:2] == 3.0).all() and (y[n - 3:] == 3.0).all() and (y[:, C:] == 3.0).all()
    kept = [i for i in range(2 * rows) if i not in to]
    assert torch.equal(state[kept], old[kept])


def test_conv_one_token_a_row():
    C = 256
    state, w = torch.randn(5, C, 3).cuda(), torch.randn(C, 4).cuda()
    x, old = torch.randn(4, C).cuda(), state.clone()
    h = ca.DeltaConv(state, w)
    a = h.apply(x, None, dev([0, 1, 2, 9]), dev([0, 1, 4, 3]))
    b_state = old.clone()
    b = ca.DeltaConv(b_state, w).apply(x, dev([0, 1, 2, 3, 4]), dev([0, 1, 2, 9]), dev([0, 1, 4, 3]))
    assert torch.equal(a[:3], b[:3]) and torch.equal(state[[0, 1, 2, 4]], b_state[[0, 1, 2, 4]])
    assert torch.isnan(a[3]).all() and torch.isnan(state[3][:, :2]).all() and torch.equal(state[3][:, 2], x[3])


# ------------------------------------------------------------------ streams, graphs, devices
def test_calls_on_other_streams_and_at_once():
    NK, NV, hd, n = 4, 8, 128, 90
    L = Layer(n, NK, NV, hd, "bf16", True, seed=11)
    _, state = pool(6, NV, hd, 11)
    h = ca.DeltaStates(state, NK)
    want = h.prompt(*L.args(), dev([0, n]), dev([0]), dev([1]), **L.kw()).clone()
    torch.cuda.synchronize()
    outs = [torch.zeros_like(want) for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    work = [torch.empty(h.prompt_workspace(n, 1, True), dtype=torch.uint8, device="cuda") for _ in range(4)]
    starts, src, dst = dev([0, n]), dev([0]), [dev([2 + i]) for i in range(4)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, o, w, d in zip(streams, outs, work, dst):
            with torch.cuda.stream(s):
                h.prompt(*L.args(), starts, src, d, out=o, workspace=w, **L.kw())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert all(torch.equal(state[1], state[2 + i]) for i in range(4))


def test_captured_and_replayed_with_other_rows():
    """A captured step, prompt and convolution go by what the device arrays hold when they are replayed."""
    NK, NV, hd, n, rows = 2, 4, 128, 96, 3
    C = (2 * NK + NV) * hd
    L = Layer(n, NK, NV, hd, "f32", True, seed=12)
    _, state = pool(8, NV, hd, 12)
    conv, w = torch.randn(8, C, 3).cuda(), torch.randn(C, 4).cuda()
    h, cv = ca.DeltaStates(state, NK), ca.DeltaConv(conv, w)
    x = torch.randn(n, C).cuda()
    starts, src, dst = dev([0, 30, 31, n]), dev([0, 1, 2]), dev([3, 4, 5])
    out, y, so = torch.empty(n, NV, hd, device="cuda"), torch.empty(n, C, device="cuda"), torch.empty(rows, NV, hd, device="cuda")
    ws = torch.empty(h.prompt_workspace(n, rows, True), dtype=torch.uint8, device="cuda")
    one = tuple(t[:rows] for t in L.args()[:5]) + L.args()[5:]

    def run():
        cv.apply(x, starts, src, dst, out=y)
        h.prompt(*L.args(), starts, src, dst, out=out, workspace=ws, **L.kw())
        h.step(*one, dst, dst, z=L.z[:rows], norm_w=L.norm_w, eps=EPS, out=so)

    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for i, s in enumerate(([0, 30, 31, n], [0, 0, 96, 96], [5, 20, 84, 90], [0, 64, 66, 67])):
        starts.copy_(dev(s))
        x.normal_()
        L.v.normal_()
        keep, keep_conv = state.clone(), conv.clone()
        run()
        want = [t.clone() for t in (out, y, so, state, conv)]
        state.copy_(keep)
        conv.copy_(keep_conv)
        for t in (out, y, so):
            t.fill_(0)
        want[0][:s[0]] = want[0][s[3]:] = 0
        want[1][:s[0]] = want[1][s[3]:] = 0
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((out, y, so, state, conv), want):
            assert torch.equal(a, b), i


def test_nothing_to_do():
    NK, NV, hd = 2, 4, 64
    _, state = pool(3, NV, hd, 1)
    old, L = state.clone(), Layer(0, NK, NV, hd, "f32", False, seed=1)
    h = ca.DeltaStates(state, NK)
    assert h.step(*L.args(), dev([]), dev([])).shape == (0, NV, hd)
    h.prompt(*L.args(), dev([0, 0, 0]), dev([0, -1]), dev([1, 2]))  # rows of no token: copied, cleared
    assert torch.equal(state[0], old[0]) and torch.equal(state[1], old[0]) and (state[2] == 0).all()
    assert h.prompt(*L.args(), dev([0]), dev([]), dev([])).shape == (0, NV, hd)


def test_rows_without_tokens_need_no_inputs():
    _, state = pool(3, 4, 64, 1)
    old = state.clone()
    s = ca._DeltaStates(state.data_ptr(), state.stride(0), 3, 4, 2, 64)
    t = ca._DeltaTokens(*(0 if n in ("type", "eps") or n.endswith("_stride") else None for n, _ in ca._DeltaTokens._fields_))
    starts, slots, to = dev([0, 0, 0, 0]), dev([0, -1, 2]), dev([1, 2, -1])
    work = torch.empty(ca.load_engine_lib().chpe_delta_prompt_workspace(s, 0, 2, 0), dtype=torch.uint8, device="cuda")
    assert ca.load_engine_lib().chpe_delta_prompt(s, t, 0, 2, starts.data_ptr(), slots.data_ptr(), to.data_ptr(), work.data_ptr(),
                                                  work.numel(), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(state[0], old[0]) and torch.equal(state[1], old[0]) and (state[2] == 0).all()


def test_what_python_refuses():
    NK, NV, hd, n = 2, 4, 64, 3
    L = Layer(n, NK, NV, hd, "f32", False, seed=1)
    _, state = pool(3, NV, hd, 1)
    h = ca.DeltaStates(state, NK)
    s = dev([0, 1, 2])
    q, k, v, a, b, A, d = L.args()
    for bad in ((q[:2], k, v, a, b, A, d), (q.half(), k, v, a, b, A, d), (q, k, v.transpose(1, 2).contiguous().transpose(1, 2), a, b, A, d),
                (q, k, v, a.half(), b, A, d), (q, k, v, a, b[:, :2], A, d), (q, k, v, a, b, A.cpu(), d), (q.cpu(), k, v, a, b, A, d)):
        with pytest.raises(ValueError):
            h.step(*bad, s)
    for kw in (dict(z=v), dict(norm_w=A), dict(out=v.half())):
        with pytest.raises(ValueError):
            h.step(*L.args(), s, **kw)
    for bad in (s.long(), s[:2], s.cpu(), dev([0, 1, 2, 3])):
        with pytest.raises(ValueError):
            h.step(*L.args(), bad)
    with pytest.raises(ValueError):
        h.prompt(*L.args(), dev([0, 3]), s)
    with pytest.raises(ca.EngineError):
        h.prompt(*L.args(), dev([0, 3]), dev([0]), workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ca.EngineError):
        ca.DeltaStates(state, 3).step(torch.zeros(n, 3, hd, device="cuda"), torch.zeros(n, 3, hd, device="cuda"), v, a, b, A, d, s)
    with pytest.raises(ValueError):
        ca.DeltaStates(state.half(), NK)
    with pytest.raises(ValueError):
        ca.DeltaConv(torch.zeros(2, 8, 3, device="cuda"), torch.zeros(8, 3, device="cuda"))
    with pytest.raises(ca.EngineError):
        ca.DeltaConv(torch.zeros(2, 12, 3, device="cuda"), torch.zeros(12, 4, device="cuda")).apply(torch.zeros(1, 12, device="cuda"), None, dev([0]))
