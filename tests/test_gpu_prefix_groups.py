"""Tables of groups that are not valid, or padded: only the rows of a group that is not valid give NaN.  The workspace holds NaN
before the call, so that a part that nobody forms shows.  Tolerances: test_gpu_paged.py's."""
import numpy as np
import pytest
import torch

from test_gpu_paged import TYPES
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


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H", [4, 40])  # few queries a group, many
def test_rows_behind_a_group_that_is_not_valid(H, dtype):
    """A row in no group has no prefix, whatever the last group ahead of it holds."""
    g = Groups([(100, [101, 140, 100]), (100, [120, 130]), (None, [40, 0, 35])], 2, 64, 16, dtype, seed=H)
    q = queries(8, H, 64)
    want = run(g, q, [0, 3, 5], [100, 100])
    g.check(q, want)
    for prefixes, bad in (([100, 101], [3, 4]), ([100, -1], [3, 4]), ([-5, 2 ** 31 - 1], [0, 1, 2, 3, 4])):
        out = run(g, q, [0, 3, 5], prefixes)
        assert nan_rows(out) == bad, prefixes
        g.check(q, out, rows=[r for r in range(8) if r not in bad])
    for groups in ([-2, 5], [-7, -2]):  # (rows 0 to 4 in a group that is not valid; in none, but longer than max_rest)
        out = run(g, q, groups, [100])
        assert nan_rows(out) == [0, 1, 2, 3, 4], groups
        g.check(q, out, rows=[5, 6, 7])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H", [4, 40])
def test_empty_groups_pad_a_table(H, dtype):
    """A table of a fixed number of groups, the last ones empty, whatever their prefixes' lengths are."""
    g = Groups([(100, [101, 140, 100, 120, 130]), (None, [40, 0, 35])], 2, 64, 16, dtype, seed=H + 1)
    q = queries(8, H, 64)
    for pad in (0, -1, 101, 2 ** 31 - 1, 50):
        for groups, prefixes in (([0, 5, 5, 5], [100, pad, pad]), ([0, 5, 5, 8, 8], [100, pad, 0, pad]), ([0, 0, 5], [pad, 100])):
            out = run(g, q, groups, prefixes)
            assert nan_rows(out) == [], (groups, prefixes)
            g.check(q, out)
