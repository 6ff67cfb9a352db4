"""Sizes past 32 bits given to KvPages: refused, not cut to their low bits."""
import pytest
import torch

import chpe_amd as ca
from test_gpu_paged import Pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("high", [1 << 32, (1 << 32) + 5, 1 << 64])
def test_sizes_past_32_bits_are_refused(high):
    pool = Pool(2, 32, 2, 64, 16, "f16")
    p = pool.p
    q, lens = torch.zeros(2, 4, 64, device="cuda"), torch.full((2,), 20, dtype=torch.int32, device="cuda")
    w, s = torch.zeros(2, 2, 32, device="cuda"), torch.zeros(2, 2, 32, dtype=torch.int32, device="cuda")
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    for call in (lambda: p.attention(q, lens, high + 32, workspace=ws), lambda: p.attention(q, lens, 32, window=high + 3, workspace=ws),
                 lambda: p.attention_workspace(4, high + 32), lambda: p.attention_workspace(high + 4, 32),
                 lambda: p.evict_workspace(high + 32), lambda: p.evict(lens, 32, high, w, s, workspace=ws),
                 lambda: p.evict(lens, high + 32, 16, w, s, workspace=ws),
                 lambda: p.evict(lens, 32, 16, w, s, recent=high, workspace=ws),
                 lambda: p.evict(lens, 32, 16, w, s, sinks=high, workspace=ws)):
        with pytest.raises(ValueError):
            call()
    assert (lens == 20).all()
    with pytest.raises(ValueError):
        p.attention_workspace(4, -1)
    with pytest.raises(ValueError):
        p.evict_workspace(-1)


def test_descriptions_past_32_bits_are_refused():
    """A pool of more pages than 32 bits count (one page repeated: its stride is 0)."""
    k = torch.zeros(1, 2, 16, 64, device="cuda", dtype=torch.float16)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    many = k.expand((1 << 32) + 1, 2, 16, 64)
    with pytest.raises(ValueError):
        ca.KvPages(many, many, table)


def test_the_largest_sizes_are_taken():
    """A budget and a window of 2^32 - 1 mean no limit; nothing is dropped."""
    pool = Pool(2, 32, 2, 64, 16, "f16")
    p = pool.p
    q, lens = torch.randn(2, 4, 64, device="cuda"), torch.full((2,), 20, dtype=torch.int32, device="cuda")
    w, s = torch.zeros(2, 2, 32, device="cuda"), torch.zeros(2, 2, 32, dtype=torch.int32, device="cuda")
    p.evict(lens, 32, (1 << 32) - 1, w, s)
    assert (lens == 20).all()
    assert torch.equal(p.attention(q, lens, 32, window=(1 << 32) - 1), p.attention(q, lens, 32))
