"""What the delta rule's calls and the prefix attention refuse (include/chpe.h, chpe_delta_*, chpe_paged_prefix_*), on the
host: every check comes before the first launch, so nothing here needs a GPU.  The addresses are never followed."""
import pytest

import chpe_amd as ca
from test_paged_refusals import A, BAD_PAGES, pages

BIG = 1 << 40


def states(**kw):
    c = dict(state=A, slot_stride=4 * 64 * 64, n_slots=9, v_heads=4, k_heads=2, head_dim=64)
    c.update(kw)
    return ca._DeltaStates(*(c[n] for n, _ in ca._DeltaStates._fields_))


def tokens(**kw):
    c = dict(type=0, q=A, k=A, v=A, z=None, out=A, q_stride=512, k_stride=512, v_stride=512, z_stride=0, out_stride=256, a=A, b=A,
             a_stride=4, b_stride=4, A_log=A, dt_bias=A, norm_w=None, eps=1e-6)
    c.update(kw)
    return ca._DeltaTokens(*(c[n] for n, _ in ca._DeltaTokens._fields_))


def step(s, t, rows=3, slot_in=A, slot_out=A):
    return ca.load_engine_lib().chpe_delta_step(s, t, rows, slot_in, slot_out, None)


def prompt(s, t, n=70, rows=3, starts=A, slot_in=A, slot_out=A, work=A, size=BIG):
    return ca.load_engine_lib().chpe_delta_prompt(s, t, n, rows, starts, slot_in, slot_out, work, size, None)


def conv(**kw):
    a = dict(state=A, stride=64 * 3, n_slots=5, channels=64, taps=4, w=A, type=0, x=A, xs=64, y=A, ys=64, n=70, rows=3,
             starts=A, slot_in=A, slot_out=A)
    a.update(kw)
    return ca.load_engine_lib().chpe_delta_conv(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(state=None), dict(state=A + 8), dict(slot_stride=4 * 64 * 64 - 4), dict(slot_stride=4 * 64 * 64 + 2), dict(n_slots=0),
    dict(n_slots=1 << 31), dict(v_heads=0), dict(k_heads=0), dict(k_heads=3), dict(k_heads=8), dict(head_dim=96), dict(head_dim=256),
    dict(slot_stride=1 << 60),
], ids=str)
def test_states(bad):
    s = states(**bad)
    assert step(s, tokens()) == prompt(s, tokens()) == -1
    assert ca.load_engine_lib().chpe_delta_prompt_workspace(s, 70, 3, 0) == 0


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(type=-1), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=A + 4), dict(k=A + 8), dict(v=A + 12),
    dict(out=A + 4), dict(a=None), dict(b=None), dict(A_log=None), dict(dt_bias=None), dict(z=A, z_stride=256), dict(norm_w=A),
    dict(z=A + 4, z_stride=256, norm_w=A), dict(z=A, z_stride=252, norm_w=A), dict(z=A, z_stride=256, norm_w=A + 4), dict(q_stride=124),
    dict(q_stride=130), dict(k_stride=127), dict(v_stride=252), dict(out_stride=255), dict(out_stride=258), dict(a_stride=3), dict(b_stride=0),
    dict(q_stride=1 << 60), dict(a_stride=1 << 61), dict(type=1, q_stride=516), dict(type=2, out_stride=260),
], ids=str)
def test_tokens(bad):
    assert step(states(), tokens(**bad)) == prompt(states(), tokens(**bad)) == -1


def test_calls():
    lib, s, t = ca.load_engine_lib(), states(), tokens()
    assert step(None, t) == step(s, None) == prompt(None, t) == prompt(s, None) == -1
    assert step(s, t, slot_in=None) == step(s, t, slot_out=None) == step(s, t, rows=1 << 31) == step(s, t, rows=1 << 22) == -1
    for bad in (dict(starts=None), dict(slot_in=None), dict(slot_out=None), dict(work=None), dict(work=A + 8), dict(n=1 << 31),
                dict(rows=1 << 31), dict(rows=1 << 21)):
        assert prompt(s, t, **bad) == -1, bad
    need = lib.chpe_delta_prompt_workspace(s, 70, 3, 0)
    assert need > 0 and prompt(s, t, size=need - 1) == -2
    z = tokens(z=A, z_stride=256, norm_w=A)
    more = lib.chpe_delta_prompt_workspace(s, 70, 3, 1)
    assert more == need + 70 * 4 * 64 * 4 and prompt(s, z, size=more - 1) == -2
    assert lib.chpe_delta_prompt_workspace(None, 70, 3, 0) == 0 and lib.chpe_delta_prompt_workspace(s, 1 << 31, 3, 0) == 0
    assert lib.chpe_delta_prompt_workspace(s, 70, 1 << 21, 0) == 0
    # nothing to do: before any launch
    assert step(s, t, rows=0) == prompt(s, t, rows=0) == 0


@pytest.mark.parametrize("bad", [
    dict(state=None), dict(state=A + 4), dict(stride=188), dict(stride=194), dict(n_slots=0), dict(channels=0), dict(channels=60),
    dict(taps=1), dict(taps=9), dict(w=None), dict(w=A + 8), dict(type=3), dict(x=None), dict(x=A + 4), dict(xs=60), dict(xs=66), dict(y=None),
    dict(y=A + 8), dict(ys=32), dict(type=2, xs=68), dict(n=1 << 31), dict(rows=1 << 31), dict(starts=None), dict(slot_in=None),
    dict(slot_out=None), dict(rows=1 << 27),
], ids=str)
def test_conv(bad):
    assert conv(**bad) == -1


def test_conv_without_rows():
    assert conv(rows=0) == 0 and conv(rows=0, n=0, starts=None, x=None, y=None) == 0


def prefix(c, **kw):
    a = dict(heads=64, lens=A, groups=2, group_rows=A, prefix_lens=A, max_prefix=48, max_rest=32, q=A, qs=64 * 128, scale=0.1, out=A,
             os=64 * 128, work=A, size=BIG)
    a.update(kw)
    return ca.load_engine_lib().chpe_paged_prefix_attention(c, *a.values(), None)


@pytest.mark.parametrize("bad", BAD_PAGES, ids=lambda b: "-".join(b))
def test_prefix_descriptions(bad):
    assert prefix(pages(**bad)) == -1
    assert ca.load_engine_lib().chpe_paged_prefix_workspace(pages(**bad), 64, 2, 48, 32) == 0


@pytest.mark.parametrize("bad", [
    dict(heads=0), dict(heads=63), dict(heads=65544), dict(lens=None), dict(group_rows=None), dict(prefix_lens=None), dict(groups=1 << 31),
    dict(max_prefix=49), dict(max_rest=33), dict(max_prefix=0xffffffff), dict(q=None), dict(q=A + 4), dict(out=None), dict(out=A + 8),
    dict(work=None), dict(work=A + 4), dict(qs=64 * 128 - 4), dict(qs=64 * 128 + 2), dict(os=64 * 128 + 1), dict(qs=1 << 60),
], ids=str)
def test_prefix_arguments(bad):
    assert prefix(pages(), **bad) == -1


def test_prefix_workspace():
    lib = ca.load_engine_lib()
    need = lib.chpe_paged_prefix_workspace(pages(), 64, 2, 48, 32)
    assert need > 0 and prefix(pages(), size=need - 1) == -2 and prefix(None) == -1
    assert prefix(pages(rows=0), size=0) == 0
    assert lib.chpe_paged_prefix_workspace(pages(), 64, 2, 49, 32) == 0 and lib.chpe_paged_prefix_workspace(None, 64, 2, 1, 1) == 0
    # the two kinds of workgroups in one launch: together within what a launch can have
    many, groups = pages(rows=1 << 20), (1 << 20) - (1 << 17)
    assert lib.chpe_paged_prefix_workspace(many, 8, groups - 1, 16, 16) > 0 and lib.chpe_paged_prefix_workspace(many, 8, groups, 16, 16) == 0
