"""Tables of groups that are not valid, or padded: only the rows of a group that is not valid give NaN.  The workspace holds NaN
before the call, so that a part that nobody forms shows.  Tolerances: test_gpu_paged.py's."""
import numpy as np
import pytest
import torch

from test_gpu_prefix import Groups, dev, queries

pytestmark = pytest.mark.gpu


def nan_rows(out):
    return [r for r, x in enumerate(torch.isnan(out).flatten(1).all(1).tolist()) if x]


def run(g, q, group_rows, prefix_lens):
    g.group_rows, g.prefix_lens = dev(np.array(group_rows, np.int64)), dev(np.array(prefix_lens, np.int64))
    return g.run(q)


# query heads, head dim, queries of a workgroup: more heads on the kv head than those, so that a group's first tile of queries has
# a number above its first row
@pytest.mark.parametrize("H,hd,dtype,tile", [
    (64, 64, "f32", 16), (48, 128, "f32", 16), (40, 256, "f32", 16), (40, 256, "bf16", 8), (24, 256, "f16", 8),
    (40, 64, "f16", 16), (130, 256, "bf16", 64), (300, 64, "f16", 128), (256, 128, "bf16", 128)])
@pytest.mark.parametrize("more", [0, 1, 3])
def test_groups_that_start_behind_the_rows(H, hd, dtype, tile, more):
    """Starts whose tiles' numbers, a product with the heads, pass 32 bits: small again when cut to them."""
    many = tile > 16
    prefix, rest = (400, 30) if many else (100, 60)  # (long rests keep a group's many queries from sharing a workgroup of 64 or 128)
    good = [prefix + 1, prefix + rest, prefix, prefix + 7, prefix + 20]
    g = Groups([(prefix, good), (None, [30, 20, 0])], 1, hd, 16, dtype, seed=H)
    q = queries(8, H, hd)
    start = min(-(-((1 << 32) + more) * tile // H), (1 << 31) - 1)
    for groups, bad in (([0, 5, start, start], [5, 6, 7]), ([0, 5, 6, start], [6, 7]), ([0, 5, 8, start], []), ([0, 5, start, (1 << 31) - 1], [5, 6, 7])):
        out = run(g, q, groups, [prefix, 0, 0])
        assert nan_rows(out) == bad, groups
        g.check(q, out, rows=[r for r in range(8) if r not in bad])
