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
