"""How many bits the products of the delta rule's chunks keep, with inputs whose errors do not hide among many others: keys and
queries that are one number at one dim and 0 elsewhere, no decay, so that every sum has one term, or one per earlier token at
the same dim.

Bounds, in roundings to f32 (u = 2^-24 relative, in the worst case), of one chunk.  A product of two values in bf16 parts leaves out
less than 1 u and rounds once (2).  1 / |k|: the square, 1e-6 and the sum, half of them by the root, the root, the division (4);
1 / |q| over sqrt(D) two more (6); b: an exponential (2), a sum, a division (4).  A_ij: b, both norms, the product, 3 factors (17);
T_ij: the substitution, two f32 products of blocks (5), b and its product (5), so 27; v - K S: the product, its factor (5), its
product, the difference (9).  An update u: T, x and their product (38); a state's element: the factor and its product (6), the
product with the key, the sum: 47.  An output: both norms, the product and 3 factors (15), then with u (38) their product and the
sum: 56.  All of it relative to the same sums of magnitudes.  Two bf16 parts instead of three leave errors of up to 128 u in every
operand: the 64-bit oracle's own test below shows that no operand cut to two would pass."""
import numpy as np
import pytest
import torch

import chpe_amd as ca
from test_gpu_delta import HALF, TYPES, U, dev

STATE, OUT = 47, 56


class Sparse:
    """Inputs of one row: n tokens, heads of hd dims, keys of token t at dim t % period."""

    def __init__(self, kind, NK, NV, hd, n, dtype, seed):
        g = np.random.default_rng(seed)
        some = lambda *s: (1 + g.random(s)) * g.choice([-1.0, 1.0], s)  # noqa: E731
        put = lambda x, t: torch.from_numpy(x).to(TYPES[t])  # noqa: E731
        # queries look at their own token's dim, so at what it and an earlier token left there
        at = np.arange(n) % {"twice": (n + 1) // 2}.get(kind, n)
        self.at = at = at % hd
        k, q = np.zeros((n, NK, hd)), np.zeros((n, NK, hd))
        k[np.arange(n), :, at], q[np.arange(n), :, at] = some(n, NK), some(n, NK)
        v, S0, b = some(n, NV, hd), some(NV, hd, hd), g.random((n, NV)) * 2 + 1.0  # (b: 0.73 to 0.95)
        if kind == "queries":    # outputs of the state before alone
            b[:] = -200.0
        elif kind in ("values", "twice", "short"):   # of the tokens alone
            S0[:] = 0
        elif kind == "states":   # what the tokens take off the state
            v[:] = 0
        if kind == "short":      # keys beside which 1e-6 counts: K's and Q's products with them have bits of their own
            k *= g.choice([2.0 ** -10, 2.0 ** -11], (n, 1, 1))
        if kind == "twice":
            v[(n + 1) // 2:] = 0  # the second token takes off what the first left
        self.k, self.q, self.v = put(k, dtype), put(q, dtype), put(v, dtype)
        self.S0, self.b = put(S0, "f32"), put(b, "f32")

    def f64(self):
        NV, NK = self.v.shape[1], self.k.shape[1]
        k, q = (x.double().numpy().repeat(NV // NK, 1) for x in (self.k, self.q))
        return k, q, self.v.double().numpy(), 1 / (1 + np.exp(-self.b.double().numpy())), self.S0.double().numpy()

    def exact(self):
        """Outputs, state, and the sums of the magnitudes of their terms."""
        k, q, v, b, S = self.f64()
        hd, M, out, mag = S.shape[1], np.abs(S), np.zeros_like(v), np.zeros_like(v)
        for t, d in enumerate(self.at):
            kk, qq = (x[t, :, d] / np.sqrt(x[t, :, d] ** 2 + 1e-6) for x in (k, q))
            kk, qq = kk[:, None], qq[:, None] / np.sqrt(hd)
            M[:, d] += np.abs(kk) * b[t][:, None] * (np.abs(v[t]) + np.abs(kk) * M[:, d])
            S = S.copy()
            S[:, d] += kk * b[t][:, None] * (v[t] - kk * S[:, d])
            out[t], mag[t] = qq * S[:, d], np.abs(qq) * M[:, d]
        return out, S, mag, M

    def chunk(self, cut):
        """The chunk's products with the operand `cut` (a name) in two bf16 parts, all else exact."""
        k, q, v, b, S = (np.moveaxis(x, 1, 0) if i < 4 else x for i, x in enumerate(self.f64()))
        c = lambda name, x: two_parts(x) if name == cut else x  # noqa: E731
        T = lambda x: np.swapaxes(x, 1, 2)  # noqa: E731
        rk, rq = (1 / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (k, q))
        rq = rq / np.sqrt(k.shape[2])
        b = b[..., None]
        n = k.shape[1]
        x = v - rk * (c("k of K S", k) @ c("S of K S", S))
        A = np.tril(b * rk * (c("k of K K", k) @ T(c("k of K K", k))) * T(rk), -1)
        W = np.linalg.inv(np.eye(n) + A) * T(b)
        O = np.tril(rq * (c("q of Q K", q) @ T(c("k of Q K", k))) * T(rk))  # noqa: E741
        u = c("T", W) @ c("x", x)
        out = rq * (c("q of Q S", q) @ c("S of Q S", S)) + c("Q K", O) @ c("u", u)
        S = S + T(c("k of K u", k)) @ c("u of K u", u * rk)
        return np.moveaxis(out, 0, 1), S


def two_parts(x):
    x = torch.from_numpy(x).float()
    hi = x.bfloat16().float()
    return (hi + (x - hi).bfloat16().float()).double().numpy()


KINDS = ["queries", "values", "states", "twice", "short", "all"]
OPERANDS = ["k of K S", "S of K S", "k of K K", "q of Q K", "k of Q K", "T", "x", "q of Q S", "S of Q S", "Q K", "u", "k of K u", "u of K u"]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [64, 50])
@pytest.mark.parametrize("NK,NV,hd,dtype", [
    (1, 3, 128, "f32"), (8, 48, 128, "f32"), (2, 6, 64, "f32"), (16, 48, 64, "f32"), (1, 3, 128, "f16"), (8, 48, 128, "f16"), (5, 5, 64, "f16"),
    (1, 3, 128, "bf16"), (8, 48, 128, "bf16"), (16, 256, 128, "bf16"), (2, 6, 64, "bf16")])
def test_chunks_keep_their_bits(NK, NV, hd, dtype, n, kind):
    x = Sparse(kind, NK, NV, hd, n, dtype, seed=NV + n)
    out64, S64, mag, M = x.exact()
    state = x.S0[None].cuda()
    zero = torch.zeros(NV, device="cuda")
    out = ca.DeltaStates(state, NK).prompt(x.q.cuda(), x.k.cuda(), x.v.cuda(), torch.zeros(n, NV, device="cuda"), x.b.cuda(), zero - 60.0, zero,
                                           dev([0, n]), dev([0]))
    err, tol = np.abs(state[0].cpu().double().numpy() - S64), STATE * U * M
    assert (err <= tol).all(), ("state", float((err / np.maximum(tol, 1e-300)).max()))
    err, tol = np.abs(out.cpu().double().numpy() - out64), OUT * U * mag
    tol = tol + HALF[dtype] * (np.abs(out64) + tol) + 2.0 ** -25 * (dtype == "f16")
    assert (err <= tol).all(), ("out", float((err / np.maximum(tol, 1e-300)).max()))


@pytest.mark.parametrize("hd", [64, 128])
def test_the_oracles_chunk_is_the_recurrence(hd):
    for kind in KINDS:
        x = Sparse(kind, 1, 3, hd, 64, "f32", seed=1)
        out, S, mag, M = x.exact()
        got, got_S = x.chunk(None)
        assert (np.abs(got - out) <= 1e-13 * mag).all() and (np.abs(got_S - S) <= 1e-13 * M).all(), kind


@pytest.mark.parametrize("operand", OPERANDS)
@pytest.mark.parametrize("NK,NV,hd", [(8, 48, 128), (16, 48, 64)])
def test_two_bf16_parts_would_not_pass(NK, NV, hd, operand):
    """The bounds above, of the same f32 inputs, against 64-bit chunks with one operand cut to two bf16 parts."""
    worst = 0.0
    for kind in KINDS:
        x = Sparse(kind, NK, NV, hd, 64, "f32", seed=NV + 64)
        out, S, mag, M = x.exact()
        got, got_S = x.chunk(operand)
        for e, t in ((np.abs(got - out), OUT * U * mag), (np.abs(got_S - S), STATE * U * M)):
            worst = max(worst, float((e[t > 0] / t[t > 0]).max(initial=0)))
    assert worst > 1.1, worst
