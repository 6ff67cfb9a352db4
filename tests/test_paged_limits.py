"""The paged cache's limits, on the host: what the workspace calls answer agrees with what the calls refuse, up to
sizes where products of the arguments pass 32 and 64 bits.  Nothing is launched: the workspaces given are too
small, or the arguments bad."""
import pytest

import chpe_amd as ca
from test_paged_refusals import A, append, attention, evict, pages


@pytest.mark.parametrize("rows,kv,ok", [
    ((1 << 22) - 1, 1, True), (1 << 22, 1, False), (1 << 21, 2, False), (1 << 23, 1, False), ((1 << 21) - 1, 2, True),
    ((1 << 32) - 1, 1, False)])
def test_eviction_counts_its_own_workgroups(rows, kv, ok):
    """1024 threads a (row, kv head): fewer than 2^32 in all."""
    c = pages(rows=rows, kv_heads=kv)
    assert (ca.load_engine_lib().chpe_paged_evict_workspace(c, 80) > 0) == ok
    assert evict(c, bytes=0) == (-2 if ok else -1)


@pytest.mark.parametrize("rows,kv,heads,max_len,window,weights,ok", [
    (131072, 1, 64, 80, 0, 0, True), (131073, 1, 64, 80, 0, 0, False), (200000, 8, 64, 80, 0, 0, False),
    (200000, 8, 64, 80, 1, 0, False), ((1 << 32) - 1, 8, 65536, 80, 0, 0, False),
    ((1 << 32) - 1, 8, 65536, 0x7ffffff0, 0, 1, False),
    (1 << 20, 1, 1, 0x7ffffff0, 0, 0, True), (1 << 20, 1, 1, 0x7ffffff0, 99, 0, True),
    (1 << 20, 8, 8, 0x7ffffff0, 0, 0, True),
    (1 << 20, 1, 1, 8 * 1024, 0, 1, True), (1 << 20, 1, 1, 8 * 1024 + 1, 0, 1, False), (1 << 20, 1, 1, 8 * 1024 + 1, 1, 1, False),
    (1 << 20, 1, 8, 8 * 1024, 0, 0, True)])
def test_attention_workspace_is_0_where_the_call_refuses(rows, kv, heads, max_len, window, weights, ok):
    per = (max_len + 15) // 16
    c = pages(rows=rows, kv_heads=kv, pages_per_row=per, table_stride=per)
    assert (ca.load_engine_lib().chpe_paged_attention_workspace(c, heads, max_len, weights) > 0) == ok
    more = dict(wo=A, ws=max_len) if weights else {}
    got = attention(c, heads=heads, max_len=max_len, window=window, qs=heads * 128, os=heads * 128, bytes=0, **more)
    assert got == (-2 if ok else -1)


@pytest.mark.parametrize("heads,head_stride", [(5, 1 << 62), (65, 1 << 58), (64, 0x0410410410410414), (2, (1 << 64) - 128)])
def test_append_strides_whose_extent_wraps(heads, head_stride):
    """(heads - 1) * q_head_stride past 64 bits does not pass for a small extent; nor without a second token."""
    assert append(pages(), heads=heads, qh=head_stride, qs=64 * 128) == -1
    assert append(pages(), heads=heads, qh=head_stride, qs=64 * 128, tokens=1) == -1
