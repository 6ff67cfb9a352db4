"""What the paged cache's calls refuse (include/chpe.h, chpe_paged_*), on the host: every check comes before
the first launch, so nothing here needs a GPU.  The addresses are never followed."""
import ctypes

import pytest

import chpe_amd as ca

A = 0x10000  # an address at a 16-byte boundary


def pages(**kw):
    c = dict(k=A, v=A, type=1, kv_heads=8, head_dim=128, page_size=16, n_pages=64, page_stride=16384, head_stride=2048,
             slot_stride=128, table=A, rows=3, pages_per_row=5, table_stride=5)
    c.update(kw)
    return ca._KvPages(*(c[n] for n, _ in ca._KvPages._fields_))


BAD_PAGES = [
    dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 2), dict(type=3), dict(type=-1), dict(kv_heads=0),
    dict(head_dim=96), dict(head_dim=0), dict(page_size=0), dict(page_size=24), dict(n_pages=0), dict(table=None),
    dict(pages_per_row=0), dict(table_stride=4),
    dict(slot_stride=64),                      # slots in each other
    dict(slot_stride=0),                       # one slot for all
    dict(head_stride=1024),                    # heads in each other's slots
    dict(page_stride=8192),                    # pages in each other
    dict(slot_stride=132, head_stride=132 * 16, page_stride=132 * 128),  # rows that start between 16-byte boundaries
    dict(page_stride=1 << 62), dict(head_stride=(1 << 64) - 8, page_stride=2048),
    dict(page_size=1 << 20, pages_per_row=4096, table_stride=4096, head_stride=128 << 20, page_stride=1024 << 20),
]


def append(c, **kw):
    a = dict(tokens=2, heads=64, q=A, qs=64 * 128, qh=128, k=A, ks=1024, v=A, vs=1024, qn=None, kn=None, eps=1e-6, cos=A,
             sin=A, rot=128, rows=100, inter=0, row=A, slot=A, pos=A, out=A, sp=None, sw=None, ts=0)
    a.update(kw)
    return ca.load_engine_lib().chpe_paged_append(c, *a.values(), None)


def attention(c, **kw):
    a = dict(heads=64, lens=A, max_len=80, q=A, qs=64 * 128, scale=0.1, window=0, out=A, os=64 * 128, wi=None, wo=None,
             ws=0, work=A, bytes=1 << 40)
    a.update(kw)
    return ca.load_engine_lib().chpe_paged_attention(c, *a.values(), None)


def evict(c, **kw):
    a = dict(lens=A, max_len=80, budget=40, recent=8, sinks=2, w=A, p=A, stride=80, lo=A, wo=A, po=A, src=None, work=A,
             bytes=1 << 40)
    a.update(kw)
    return ca.load_engine_lib().chpe_paged_evict(c, *a.values(), None)


@pytest.mark.parametrize("bad", BAD_PAGES, ids=lambda b: "-".join(b))
def test_descriptions_are_checked_by_every_call(bad):
    c, lib = pages(**bad), ca.load_engine_lib()
    assert append(c) == attention(c) == evict(c) == -1
    assert lib.chpe_paged_attention_workspace(c, 64, 80, 0) == 0 and lib.chpe_paged_evict_workspace(c, 80) == 0


def test_null_description():
    assert append(None) == attention(None) == evict(None) == -1


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(row=None), dict(slot=None), dict(pos=None), dict(q=None), dict(out=None),
    dict(q=A + 4), dict(k=A + 4), dict(v=A + 8), dict(out=A + 4), dict(qn=A + 4), dict(kn=A + 4), dict(cos=A + 4),
    dict(sin=A + 8), dict(ks=1020), dict(vs=1023), dict(ks=1026), dict(qh=124), dict(qs=64 * 128 - 4), dict(qs=64 * 128 + 2),
    dict(rot=136), dict(rot=12), dict(cos=None), dict(sin=None), dict(rows=0), dict(sp=A), dict(sw=A),
    dict(tokens=1 << 31),
], ids=lambda b: "-".join(f"{k}{v}" for k, v in b.items()))
def test_append_arguments(bad):
    assert append(pages(), **bad) == -1


@pytest.mark.parametrize("bad", [
    dict(lens=None), dict(q=None), dict(out=None), dict(work=None), dict(q=A + 4), dict(out=A + 8), dict(work=A + 4),
    dict(heads=0), dict(heads=63), dict(max_len=81), dict(qs=64 * 128 - 4), dict(os=64 * 128 + 1), dict(wi=A),
    dict(wo=A, ws=79),
], ids=lambda b: "-".join(f"{k}{v}" for k, v in b.items()))
def test_attention_arguments(bad):
    assert attention(pages(), **bad) == -1


@pytest.mark.parametrize("bad", [
    dict(lens=None), dict(w=None), dict(p=None), dict(lo=None), dict(wo=None), dict(po=None), dict(work=None),
    dict(work=A + 8), dict(max_len=81), dict(stride=79), dict(budget=9), dict(budget=0), dict(recent=0xffffffff),
], ids=lambda b: "-".join(f"{k}{v}" for k, v in b.items()))
def test_evict_arguments(bad):
    assert evict(pages(), **bad) == -1


def test_workspaces():
    lib = ca.load_engine_lib()
    for rows, heads, n, weights in ((3, 64, 80, 0), (1, 8, 1, 1), (3, 8, 80, 1)):
        c = pages(rows=rows)
        need = lib.chpe_paged_attention_workspace(c, heads, n, weights)
        assert need > 0
        more = dict(wo=A, ws=80) if weights else {}
        assert attention(c, heads=heads, max_len=n, qs=heads * 128, os=heads * 128, bytes=need - 1, **more) == -2
    need = lib.chpe_paged_evict_workspace(pages(), 80)
    assert need > 0 and evict(pages(), bytes=need - 1) == -2


def test_nothing_to_do_is_no_error():
    none = pages(rows=0, table=None, pages_per_row=0, table_stride=0)
    assert append(pages(), tokens=0, q=None, k=None, v=None) == 0
    assert attention(none, max_len=0) == 0 and evict(none, max_len=0) == 0


def test_description_layout():
    """The ctypes structure and the header's."""
    assert ctypes.sizeof(ca._KvPages) == 88 and ca._KvPages.page_stride.offset == 40 and ca._KvPages.table.offset == 64


def test_tensor_checks():
    """KvPages refuses tensors before it calls: types, shapes, strides, CPU tensors."""
    torch = pytest.importorskip("torch")
    k, table = torch.zeros(4, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32)
    for kk, vv, tt in ((k, k[:3], table), (k, k.half(), table), (k.double(), k.double(), table), (k, k, table.long()),
                       (k, k, table[0]), (k, k.transpose(1, 2).contiguous().transpose(1, 2), table),
                       (k.transpose(2, 3), k.transpose(2, 3), table), (k, k, table[:1].expand(2, 2)), (k, k, table)):
        with pytest.raises(ValueError):
            ca.KvPages(kk, vv, tt)
