"""Slots and tokens of the delta rule's operators whose offsets pass 2^32 elements, in every kernel: the same bits as from the same
inputs close together, which are checked against the recurrence in 64 bits."""
import pytest
import torch

import chpe_amd as ca
from test_gpu_delta import TYPES, Layer, before, dev

pytestmark = pytest.mark.gpu

SLOT = (1 << 31) + 4096  # floats between slots: the third begins behind 2^32


@pytest.fixture
def memory():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("80 GiB of free device memory")
    yield
    torch.cuda.empty_cache()


def spread(tensors, stride):
    """Copies of [tokens, ..] tensors, side by side in rows `stride` elements apart."""
    n, dt = tensors[0].shape[0], tensors[0].dtype
    widths = [t[0].numel() for t in tensors]
    mem, out, at = torch.empty((n - 1) * stride + sum(widths), dtype=dt, device="cuda"), [], 0
    for t, w in zip(tensors, widths):
        inner = [1]
        for s in reversed(t.shape[2:]):
            inner.insert(0, inner[0] * s)
        view = mem.as_strided(t.shape, (stride, *inner), at)
        out.append(view.copy_(t))
        at += w
    assert (n - 1) * stride >= 1 << 32
    return out


def far_layer(L):
    """Replaces the layer's token tensors; returns rows for the outputs."""
    stride = -(-(1 << 32) // (L.n - 1) // 8) * 8 + 8
    L.q, L.k, L.v, L.z, out = spread([L.q, L.k, L.v, L.z, torch.zeros_like(L.v)], stride)
    L.a, L.b = spread([L.a, L.b], stride)
    return out


def far_state(state):
    return spread([state], SLOT)[0]


@pytest.mark.parametrize("dtype,NV,hd", [("bf16", 4, 64), ("f16", 32, 128), ("bf16", 130, 128), ("f32", 2, 128)])
def test_prompts_and_steps(memory, dtype, NV, hd):
    NK = NV // 2
    L = Layer(95, NK, NV, hd, dtype, True, seed=NV)
    near = torch.randn(3, NV, hd, hd, generator=torch.Generator().manual_seed(NV)).cuda()
    S0 = near.clone()
    args, kw = L.args(), L.kw()
    calls = [(slots, to, torch.empty_like(L.v)) for slots, to in (([2, 0], [2, 1]), ([0, 2], [1, 2]))]
    starts, h = dev([0, 90, 95]), ca.DeltaStates(near, NK)  # in chunks; token by token
    for slots, to, want in calls:
        old = near.clone()
        h.prompt(*args, starts, dev(slots), dev(to), out=want, **kw)
        for r, (lo, hi) in enumerate(((0, 90), (90, 95))):
            L.check(lo, hi, want, near[to[r]], before(old, slots[r]), (slots, r))
    out, state = far_layer(L), far_state(S0)
    h = ca.DeltaStates(state, NK)
    for slots, to, want in calls:
        h.prompt(*L.args(), starts, dev(slots), dev(to), out=out, **L.kw())
        assert torch.equal(out, want)
    assert torch.equal(state, near)
    out.zero_()
    h.prompt(*L.args(), dev([0, 95]), dev([2]), dev([2]), out=out, **L.kw())  # (one row: other sizes of workgroups)
    near_h = ca.DeltaStates(near, NK)
    assert torch.equal(out, near_h.prompt(*args, dev([0, 95]), dev([2]), dev([2]), **kw)) and torch.equal(state, near)
    # one token a row: tokens 0, 47 and 94
    pick = slice(0, 95, 47)
    three = lambda a: tuple(t[pick] for t in a[:5]) + a[5:]  # noqa: E731
    S1 = near.clone()
    got = h.step(*three(L.args()), dev([2, 1, 0]), z=L.z[pick], norm_w=L.norm_w, eps=kw["eps"], out=out[pick])
    want = near_h.step(*three(args), dev([2, 1, 0]), z=kw["z"][pick], norm_w=kw["norm_w"], eps=kw["eps"])
    assert torch.equal(got, want) and torch.equal(state, near)
    for r, (t, s) in enumerate(((0, 2), (47, 1), (94, 0))):
        L.check(t, t + 1, out, state[s], before(S1, s), ("step", r))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_convolution(memory, dtype):
    C, n = 1024, 95
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(n, C, generator=g).to(TYPES[dtype]).cuda(), torch.randn(C, 4, generator=g).cuda()
    near = torch.randn(3, C, 3, generator=g).cuda()
    stride = -(-(1 << 32) // (n - 1) // 8) * 8 + 8
    state = far_state(near)
    far_x, far_y = spread([x, torch.zeros_like(x)], stride)
    a, b = ca.DeltaConv(near, w), ca.DeltaConv(state, w)
    for starts, slots, to in ((dev([0, 90, 95]), dev([2, 0]), dev([2, 1])), (dev([0, 90, 95]), dev([0, 2]), dev([1, 2]))):
        want = a.apply(x, starts, slots, to)
        b.apply(far_x, starts, slots, to, out=far_y)
        assert torch.equal(far_y, want) and torch.equal(state, near)
    want = a.apply(x[::47], None, dev([2, 1, 0]))
    assert torch.equal(b.apply(far_x[::47], None, dev([2, 1, 0]), out=far_y[::47]), want) and torch.equal(state, near)
