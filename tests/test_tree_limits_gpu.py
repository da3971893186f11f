"""Tree attention at the ends of its ranges on the GPU: contexts that the table cuts, more nodes than fit, long contexts,
values that are huge or not finite."""

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


@pytest.mark.parametrize("n,ctx", [(20, 260), (200, 700)])
def test_values_near_the_largest(n, ctx):
    """Sums of weighted values stay in range, however far the maximum lags and in however many pieces an item is cut."""
    hq = 4
    q, k, v, table, mask, masks = batch([n], [ctx], hq, 1, 8, 3)
    slot = lambda p: int(table[0, p // 16]) * 16 + p % 16  # noqa: E731
    for p in range(ctx):  # scores that grow by some 6 in log2 from tile to tile, under the lag
        k[slot(p), 0] = p / 64
        v[slot(p), 20] = 3.3e38
        v[slot(p), 21] = -3.3e38 if p % 3 else 3.3e38
        v[slot(p), 22] = 3.3e38 if p % 50 == 7 else 1.0
    for h in range(hq):
        q[:, 128 * h] = 48
    args = [x.cuda() for x in (q, k, v, table)] + [i32([0]), i32([n]), i32([ctx]), mask.cuda()]
    for plan in ((1, True), (2, False), (9, True), (40, True), (290, True)):
        out = tree.attn_tree(*args, hq, 1, SCALE, plan=plan)
        check(out.cpu(), q, k, v, table, masks, [n], [ctx], hq, 1)
    assert status()["code"] == 0


@pytest.mark.parametrize("hq", [1, 4])
def test_infinities_in_items_of_several_pieces(hq):
    """A value that is not finite stays so however far above its piece's scores those of the pieces behind it are (the
    weight of the whole piece is then 0 in 32 bits), and finite ones there count nothing."""
    n, ctx = 256, 1000
    q, k, v, table, mask, _ = batch([n], [ctx], hq, 1, 8, 2)
    rows = O.mask_of(list(range(-1, n - 1)), 8)  # a chain: node i sees all nodes before it
    mask[:n] = rows
    slot = lambda p: int(table[0, p // 16]) * 16 + p % 16  # noqa: E731
    base = ctx - n
    for j, d, x in ((5, 11, float("inf")), (70, 12, float("-inf")), (100, 13, float("nan")), (130, 14, float("inf")), (6, 15, 3e38)):
        v[slot(base + j), d] = x
    for h in range(hq):
        q[:, 128 * h] = 8
    for p in range(ctx - 60, ctx):  # 300 above the others in log2
        k[slot(p), 0] = 300
    kk, vv = (O.rows_of(x, table[0], ctx, 1) for x in (k, v))
    want, bound, _, _ = O.attend(q[:n, : hq * 128], kk, vv, O.seen_of(rows, n, ctx), hq, 1, SCALE, W_STEP)
    args = [x.cuda() for x in (q, k, v, table)] + [i32([0]), i32([n]), i32([ctx]), mask.cuda()]
    for ctas in range(1, 70):
        out = tree.attn_tree(*args, hq, 1, SCALE, plan=(ctas, True))
        O.close(out[:n].cpu(), want, bound, f"{ctas} CTAs")
    assert status()["code"] == 0


def test_more_nodes_than_fit():
    """The first nodes, as far as the plan's rows and the queries' go, see what they would in the whole tree."""
    n, ctx, hq = [6, 6, 6], [100, 200, 60], 4
    q, k, v, table, mask, masks = batch(n, ctx, hq, 1, 1, 6)
    args = [x.cuda() for x in (q, k, v, table)]
    out = tree.attn_tree(*args, i32(starts(n)), i32([6, 6, 50]), i32(ctx), mask.cuda(), hq, 1, SCALE, host_meta=(n, ctx)).cpu()
    assert status()["code"] == 7
    check(out[:12], q, k, v, table, masks[:2], n[:2], ctx[:2], hq, 1)
    kk, vv = (O.rows_of(x, table[2], 60, 1) for x in (k, v))
    seen = O.seen_of(torch.cat([mask[12:], torch.zeros(42, 1, dtype=torch.int32)]), 50, 60)[:8]
    want, bound, _, _ = O.attend(q[12:, : hq * 128], kk, vv, seen, hq, 1, SCALE, W_STEP)
    O.close(out[12:], want, bound)


@pytest.mark.parametrize("plan", [None, (296, True), (3, False)])
def test_long_contexts(plan):
    n, ctx, hq, hkv = [5, 40], [30011, 9001], 4, 1
    q, k, v, table, mask, masks = batch(n, ctx, hq, hkv, 2, 12)
    out = tree.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(starts(n)), i32(n), i32(ctx), mask.cuda(), hq, hkv,
                         SCALE, plan=plan)
    assert status()["code"] == 0
    check(out.cpu(), q, k, v, table, masks, n, ctx, hq, hkv)
