"""Tree attention at the ends of its ranges on the GPU."""

import math

import paged_oracle as O
import pytest
import torch
from test_tree_gpu import W_STEP, batch, check, i32, starts, status

from infera_b200.ops import tree

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


@pytest.mark.parametrize("plan", [None, (3, True), (40, True), (5, False)])
@pytest.mark.parametrize("over", [3, 6, 7, 70, 5000])
@pytest.mark.parametrize("pages", [1, 2, 3, 4, 5, 13, 14, 15, 16])
def test_a_context_beyond_the_table_is_cut(pages, over, plan):
    """The keys of the table's places count, the nodes' places stay where the length puts them."""
    room, hq, hkv = 16 * pages, 8, 2
    n, ctx = [5, 6], [16, room + over]
    q, k, v, table, mask, masks = batch(n, [16, room], hq, hkv, 1, pages + over)
    out = tree.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(starts(n)), i32(n), i32(ctx), mask.cuda(), hq, hkv,
                         SCALE, host_meta=(n, [16, room]), plan=plan).cpu()
    assert status()["code"] == 7
    check(out[:5], q, k, v, table, masks[:1], n[:1], ctx[:1], hq, hkv)
    kk, vv = (O.rows_of(x, table[1], room, hkv) for x in (k, v))
    seen = O.seen_of(masks[1], 6, ctx[1])[:, :room]
    want, bound, _, _ = O.attend(q[5:11, : hq * 128], kk, vv, seen, hq, hkv, SCALE, W_STEP)
    O.close(out[5:11], want, bound)
