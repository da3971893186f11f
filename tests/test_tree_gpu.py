"""A speculative step's tree on the GPU: masks, attention over the paged cache, the accepted path and the moved rows,
against 64-bit forms."""

import math

import paged_oracle as O
import pytest
import torch

from infera_b200.ops import kernels as K
from infera_b200.ops import tree

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)
W_STEP = 2.0 ** -8  # weights are rounded to bf16


def i32(x, dev="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def starts(n):
    return [sum(n[:i]) for i in range(len(n))]


def status():
    torch.cuda.synchronize()
    s = K.scratch().read_status_detail()
    K.scratch().clear_status()
    return s


# ---------------------------------------------------------------- masks and paths


@pytest.mark.parametrize("n,words", [([1], 1), ([8, 0, 32], 1), ([61, 64, 1, 33], 2), ([256, 200], 8), ([100] * 40, 4)])
def test_masks_and_paths_match_cpu(n, words):
    g = torch.Generator().manual_seed(sum(n))
    flat = i32([p for x in n for p in (O.random_tree(x, g) if x else [])], "cpu")
    T = sum(n)
    tokens, target = torch.randint(0, 2, (2, T), generator=g, dtype=torch.int32)
    s, q = i32(starts(n), "cpu"), i32(n, "cpu")
    cu = [x.cuda() for x in (flat, s, q)]
    assert torch.equal(tree.tree_mask(*cu, words).cpu(), tree.tree_mask(flat, s, q, words))
    for most in (1, 2, 50):
        got = tree.tree_accept(tokens.cuda(), target.cuda(), *cu, most)
        for a, b in zip(got, tree.tree_accept(tokens, target, flat, s, q, most)):
            assert torch.equal(a.cpu(), b)
    assert status()["code"] == 0


def test_masks_of_bad_trees():
    m = tree.tree_mask(i32([-1, 0, 2, 9, -5, 1]), i32([0]), i32([6]), 1)
    assert m[:, 0].tolist() == [1, 3, 4, 8, 16, 32 | 3]
    assert status()["code"] == 7
    # more nodes than fit, rows that are not there: only what fits is written
    m = tree.tree_mask(i32([-1] * 50), i32([0, 45, -3, 99]), i32([40, 10, 5, 5]), 1)
    assert m[:32, 0].tolist() == [1 << i if i < 31 else -(1 << 31) for i in range(32)]
    assert m[45:, 0].tolist() == [1, 2, 4, 8, 16]
    assert status()["code"] == 7
    path, count, after = tree.tree_accept(i32([5] * 50), i32([5] * 50), i32([-1] + list(range(49))), i32([0, 99]), i32([50, 3]), 60)
    assert count.tolist() == [50, 0] and after.tolist() == [5, -1] and path[1].tolist() == [-1] * 60
    assert status()["code"] == 7


# ---------------------------------------------------------------- attention


def batch(n, ctx, hq, hkv, words, seed=0, runs=False, pad=0, dense=False):
    g = torch.Generator().manual_seed(seed)
    table, pool = O.page_table(ctx, seed, runs)
    k, v = O.caches(pool, hkv, seed)
    q = torch.randn(sum(n) + 2, (hq + 2 * hkv) * 128 + pad, generator=g).to(torch.bfloat16)
    masks = []
    for x in n:
        if dense:  # any mask, some rows without a node
            m = torch.randint(-2 ** 31, 2 ** 31 - 1, (x, words), generator=g).to(torch.int32)
            m[torch.rand(x, generator=g) < 0.2] = 0
            masks.append(m)
        else:
            masks.append(O.mask_of(O.random_tree(x, g), words) if x else torch.zeros(0, words, dtype=torch.int32))
    mask = torch.cat(masks + [torch.zeros(2, words, dtype=torch.int32)])
    # places that no sequence has are NaN, as a recycled page may leave them
    own = torch.zeros(k.shape[0], dtype=torch.bool)
    for row, c in zip(table, ctx):
        p = torch.arange(c)
        own[row[p // 16].long() * 16 + p % 16] = True
    k[~own], v[~own] = float("nan"), float("nan")
    return q, k, v, table, mask, masks


def check(out, q, k, v, table, masks, n, ctx, hq, hkv, scale=SCALE):
    at = 0
    for s in range(len(n)):
        kk, vv = (O.rows_of(x, table[s], ctx[s], hkv) for x in (k, v))
        want, bound, _, _ = O.attend(q[at:at + n[s], : hq * 128], kk, vv, O.seen_of(masks[s], n[s], ctx[s]), hq, hkv,
                                     scale, W_STEP)
        O.close(out[at:at + n[s]], want, bound, f"sequence {s}")
        at += n[s]


CASES = {
    "one node alone": ([1], [1], 4, 1, 1),
    "one node": ([1], [100], 8, 2, 1),
    "small": ([8], [500], 32, 8, 1),
    "a tile exactly": ([8], [128], 4, 1, 1),
    "nodes over a tile's end": ([20], [263], 4, 1, 1),
    "nodes without keys": ([9, 5], [3, 0], 4, 1, 1),
    "only nodes": ([61], [61], 4, 1, 2),
    "128 rows": ([32], [700], 4, 1, 1),
    "129 rows": ([43], [700], 3, 1, 2),
    "ragged": ([3, 0, 26, 11, 1], [40, 16, 300, 11, 1029], 8, 2, 1),
    "two tiles of rows": ([64], [1000], 8, 2, 2),
    "ragged, two tiles of rows": ([64, 2, 33, 40], [1000, 2, 33, 129], 8, 2, 2),
    "several items": ([150, 70], [400, 200], 4, 1, 5),
    "one head": ([200, 256], [333, 256], 1, 1, 8),
    "five heads to one": ([30, 61], [333, 100], 5, 1, 2),
    "sixteen heads to one": ([8, 3], [333, 100], 16, 1, 1),
    "sixteen heads to one, two tiles of rows": ([20], [333], 16, 1, 1),
}


@pytest.mark.parametrize("plan", [None, (300, False), (7, False), (1, True), (2, True), (31, True), (300, True)])
@pytest.mark.parametrize("name", CASES)
def test_attention(name, plan):
    n, ctx, hq, hkv, words = CASES[name]
    q, k, v, table, mask, masks = batch(n, ctx, hq, hkv, words, seed=len(name))
    out = torch.full((q.shape[0], hq * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    tree.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(starts(n)), i32(n), i32(ctx), mask.cuda(), hq, hkv,
                   SCALE, out=out, plan=plan)
    assert status()["code"] == 0
    assert torch.all(out[sum(n):] == 7.0)
    check(out.cpu(), q, k, v, table, masks, n, ctx, hq, hkv)


@pytest.mark.parametrize("runs", [False, True])
@pytest.mark.parametrize("scale", [SCALE, -0.3, 0.0, 2.0])
def test_any_mask_scale_and_stride(runs, scale):
    n, ctx, hq, hkv, words = [40, 100], [300, 555], 4, 2, 4
    q, k, v, table, mask, masks = batch(n, ctx, hq, hkv, words, 3, runs, pad=24, dense=True)
    buf = torch.zeros(q.shape[0], hq * 128 + 8, dtype=torch.bfloat16, device="cuda")
    out = tree.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(starts(n)), i32(n), i32(ctx), mask.cuda(), hq,
                         hkv, scale, out=buf)
    assert torch.all(buf[:, hq * 128:] == 0)
    check(out.cpu()[:, : hq * 128], q, k, v, table, masks, n, ctx, hq, hkv, scale)
    assert status()["code"] == 0


@pytest.mark.parametrize("n,hq", [(20, 4), (40, 4)])
@pytest.mark.parametrize("plan", [(7, False), (3, True), (40, True)])
def test_what_is_masked_may_be_anything(n, hq, plan):
    ctx = 250
    q, k, v, table, mask, masks = batch([n], [ctx], hq, 1, 2, 4)
    slot = lambda p: int(table[0, p // 16]) * 16 + p % 16  # noqa: E731
    base = ctx - n
    for j, x in ((3, float("nan")), (5, float("inf")), (7, float("-inf")), (n - 1, float("inf"))):
        v[slot(base + j), 10 + j] = x
    v[slot(base + 5), 17] = float("inf")  # with node 7's -inf there: NaN for rows that see both
    # a key of NaN that one row sees alone
    k[slot(base + n - 2)] = float("nan")
    masks[0][:, (n - 2) // 32] &= ~(1 << (n - 2) % 32)
    masks[0][2, (n - 2) // 32] |= 1 << (n - 2) % 32
    mask[:n] = masks[0]
    out = tree.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32([0]), i32([n]), i32([ctx]), mask.cuda(), hq, 1,
                         SCALE, plan=plan).cpu()
    assert bool(out[2].isnan().all())
    rest = [i for i in range(n) if i != 2]
    kk, vv = (O.rows_of(x, table[0], ctx, 1) for x in (k, v))
    seen = O.seen_of(masks[0], n, ctx)[rest]
    kk[base + n - 2] = 0
    want, bound, _, _ = O.attend(q[rest, : hq * 128], kk, vv, seen, hq, 1, SCALE, W_STEP)
    O.close(out[rest], want, bound)


def test_scores_of_very_different_size():
    # maxima that grow from tile to tile, and fall: the running maximum lags and catches up
    n, ctx, hq = [50], [900], 4
    q, k, v, table, mask, masks = batch(n, ctx, hq, 1, 2, 5)
    size = torch.linspace(0.1, 40, ctx[0])
    for p in range(ctx[0]):
        k[int(table[0, p // 16]) * 16 + p % 16] *= size[p if p % 2 else ctx[0] - 1 - p]
    for plan in ((2, False), (9, True), (100, True)):
        out = tree.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32([0]), i32(n), i32(ctx), mask.cuda(), hq, 1,
                             SCALE, plan=plan)
        check(out.cpu(), q, k, v, table, masks, n, ctx, hq, 1)


def test_bad_pages_rows_and_lengths():
    n, ctx, hq = [6, 6, 6], [100, 200, 60], 4
    q, k, v, table, mask, masks = batch(n, ctx, hq, 1, 1, 6)
    table[0, 2], table[1, 5] = -4, 2 ** 30 + 1
    args = [q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(starts(n)), i32(n), i32(ctx), mask.cuda(), hq, 1, SCALE]
    out = tree.attn_tree(*args).cpu()
    check(out, q, k, v, table, masks, n, ctx, hq, 1)
    assert status()["code"] == 0
    out = tree.attn_tree(*args, bt_rows=i32([0, 3, -1])).cpu()
    assert torch.all(out[6:18] == 0) and status()["code"] == 7
    check(out[:6], q, k, v, table, masks[:1], n[:1], ctx[:1], hq, 1)
    # lengths on the device other than the host's: cut where the table ends
    args[6] = i32([100, 200, 5000])
    out = tree.attn_tree(*args, host_meta=(n, ctx)).cpu()
    check(out[:12], q, k, v, table, masks[:2], n[:2], ctx[:2], hq, 1)
    assert status()["code"] == 7
    args[5], args[6] = i32([6, 6, 50]), i32(ctx)
    tree.attn_tree(*args, host_meta=(n, ctx))
    assert status()["code"] == 7


def test_into_the_queries_and_on_another_stream():
    n, ctx, hq, hkv = [30, 40], [600, 90], 8, 2
    q, k, v, table, mask, masks = batch(n, ctx, hq, hkv, 2, 7)
    dev = [x.cuda() for x in (q, k, v, table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = tree.attn_tree(*dev, i32(starts(n)), i32(n), i32(ctx), mask.cuda(), hq, hkv, SCALE, out=dev[0])
    side.synchronize()
    assert out.data_ptr() == dev[0].data_ptr()
    check(out.cpu()[:, : hq * 128], q, k, v, table, masks, n, ctx, hq, hkv)


@pytest.mark.parametrize("planned", [[700, 300], [100, 30]])
def test_captured_calls_follow_lengths_and_share_nothing(planned):
    hq, hkv, n = 8, 2, [20, 12]
    q, k, v, table, mask, masks = batch(n, [1300, 300], hq, hkv, 1, 8)
    dev = [x.cuda() for x in (q, k, v, table)]
    lens, rows, first, m = i32(planned), i32(n), i32(starts(n)), mask.cuda()
    call = lambda: tree.attn_tree(*dev, first, rows, lens, m, hq, hkv, SCALE, host_meta=(n, planned))  # noqa: E731
    call()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for c, r in ((planned, n), ([40, 20], n), ([1300, 300], n), ([520, 7], [17, 7])):
        lens.copy_(i32(c)), rows.copy_(i32(r))
        sub = [masks[s][: r[s]] for s in range(2)]
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for st, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for s in range(2):
                check(out.cpu()[20 * s:], q[20 * s:], k, v, table[s:], sub[s:s + 1], r[s:s + 1], c[s:s + 1], hq, hkv)
    assert status()["code"] == 0


def test_many_sequences_of_every_length():
    # more than a warp's, some without nodes, some without keys of their own
    g = torch.Generator().manual_seed(3)
    n = torch.randint(0, 20, (75,), generator=g).tolist()
    ctx = [m + int(torch.randint(0, 2, (1,), generator=g)) * int(torch.randint(0, 500, (1,), generator=g)) for m in n]
    q, k, v, table, mask, masks = batch(n, ctx, 16, 1, 1, 9)
    for plan in (None, (296, True), (5, False)):
        out = tree.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(starts(n)), i32(n), i32(ctx), mask.cuda(), 16, 1,
                             SCALE, plan=plan)
        check(out.cpu(), q, k, v, table, masks, n, ctx, 16, 1)
    assert status()["code"] == 0


# ---------------------------------------------------------------- moved rows


@pytest.mark.parametrize("hkv,layers,n", [(8, 32, 1), (1, 1, 3), (2, 5, 40), (8, 80, 48)])
def test_path_rows_move(hkv, layers, n):
    g = torch.Generator().manual_seed(n)
    ctx = torch.randint(0, 40, (n,), generator=g).tolist()
    table, pool = O.page_table([c + 64 for c in ctx], n)
    k, v = (torch.randn(layers, pool * 16, hkv * 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    path = torch.full((n, 9), -1, dtype=torch.int32)
    count = torch.randint(0, 9, (n,), generator=g).to(torch.int32)
    for s in range(n):
        path[s, : count[s]] = torch.randperm(60, generator=g)[: count[s]].sort().values.to(torch.int32)
    src, dst = [], []
    for s in range(n):
        for i in range(int(count[s])):
            a, b = ctx[s] + int(path[s, i]), ctx[s] + i
            src.append(int(table[s, a // 16]) * 16 + a % 16)
            dst.append(int(table[s, b // 16]) * 16 + b % 16)
    want = []
    for x in (k, v):
        y = x.clone()
        y[:, dst] = x[:, src]
        want.append(y)
    K.kv_compact(k, v, table.cuda(), path.cuda(), count.cuda(), start=i32(ctx))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and status()["code"] == 0


def test_latent_rows_and_entries_that_do_not_move():
    table, pool = O.page_table([200], 4)
    k = torch.randn(2, pool * 16, 576).to(torch.bfloat16)
    v = torch.zeros(2, 1, 1, dtype=torch.bfloat16)
    want = O.moved(k, table[0], [3, 4, 30, 170], 5, 576, 0)
    kc = k.cuda()
    K.kv_compact(kc, v.cuda(), table.cuda(), i32([[3, 4, 30, 170]]), i32([4]), start=i32([5]))
    assert torch.equal(kc.cpu(), want) and status()["code"] == 0
    for bad, rows, first in (([-1, 0, 1, 999, 999], None, None), ([-1, -1, -1, 40, 41], None, None),
                             ([1, 2, 3, 4, 5], [3], None), ([1, 2, 3, 4, 5], [-1], None), ([1, 2, 3, 4, 5], None, [-2])):
        t = table.clone()
        t[0, 2] = pool + 7
        kc = k.cuda()
        K.kv_compact(kc, v.cuda(), t.cuda(), i32([bad]), i32([5]), start=None if first is None else i32(first),
                     bt_rows=None if rows is None else i32(rows))
        assert torch.equal(kc.cpu(), k) and status()["code"] == 7


@pytest.mark.parametrize("width,layers", [(256, 1), (1024, 3), (576, 2), (4608, 1)])
def test_long_lists_of_whole_rows(width, layers):
    g = torch.Generator().manual_seed(width)
    lens = [1500, 700, 40]
    table, pool = O.page_table(lens, 5)
    k = torch.randn(layers, pool * 16, width, generator=g).to(torch.bfloat16)
    v = torch.randn(layers, pool * 16, width, generator=g).to(torch.bfloat16) if width % 128 == 0 else torch.zeros(1, 1, 1).to(torch.bfloat16).expand(layers, 1, 1).contiguous()
    src, start = torch.full((3, 600), -1, dtype=torch.int32), [3, 0, 17]
    count = [600, 333, 23]
    for s in range(3):
        src[s, : count[s]] = torch.randperm(lens[s] - start[s], generator=g)[: count[s]].sort().values.to(torch.int32)
    want_k, want_v = k, v
    for s in range(3):
        want_k = O.moved(want_k, table[s], src[s, : count[s]].tolist(), start[s], width, 0)
        if v.shape == k.shape:
            want_v = O.moved(want_v, table[s], src[s, : count[s]].tolist(), start[s], width, 0)
    kc, vc = k.cuda(), v.cuda()
    K.kv_compact(kc, vc, table.cuda(), src.cuda(), i32(count), start=i32(start))
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v) and status()["code"] == 0


def test_a_whole_step():
    """Masks, attention in every layer, the walk and the moves: the next step's keys are the accepted nodes'."""
    hq, hkv, layers = 8, 2, 2
    n, past = [12, 1, 30], [100, 15, 260]
    ctx = [a + b for a, b in zip(n, past)]
    g = torch.Generator().manual_seed(9)
    trees = [O.random_tree(x, g) for x in n]
    table, pool = O.page_table(ctx, 9)
    k, v = (torch.stack([O.caches(pool, hkv, 10 + i)[j] for i in range(layers)]) for j in range(2))
    q = torch.randn(sum(n), hq * 128, generator=g).to(torch.bfloat16)
    target = torch.randint(0, 2, (sum(n),), generator=g, dtype=torch.int32)
    tokens = torch.randint(0, 2, (sum(n),), generator=g, dtype=torch.int32)
    up, s, c = i32([p for t in trees for p in t]), i32(starts(n)), i32(n)
    mask = tree.tree_mask(up, s, c, 1)
    kc, vc, tc = k.cuda(), v.cuda(), table.cuda()
    for i in range(layers):
        out = tree.attn_tree(q.cuda(), kc[i], vc[i], tc, s, c, i32(ctx), mask, hq, hkv, SCALE, host_meta=(n, ctx))
        check(out.cpu(), q, k[i], v[i], table, [O.mask_of(t, 1) for t in trees], n, ctx, hq, hkv)
    path, count, after = tree.tree_accept(tokens.cuda(), target.cuda(), up, s, c, 16)
    K.kv_compact(kc, vc, tc, path, count, start=i32(past))
    new = [p + int(m) for p, m in zip(past, count)]
    for i in range(layers):
        out = K.attn_decode(q.cuda()[:3], kc[i], vc[i], tc, i32(new), hq, hkv, SCALE, splits=3).cpu()
        at = 0
        for b in range(3):
            walk = O.walk(tokens[at:at + n[b]].tolist(), target[at:at + n[b]].tolist(), trees[b], 16)
            assert path[b].tolist()[: len(walk)] == walk and int(after[b]) == int(target[at + walk[-1]])
            keep = list(range(past[b])) + [past[b] + j for j in walk]
            kk, vv = (O.rows_of(x[i], table[b], ctx[b], hkv)[keep] for x in (k, v))
            want, bound, _, _ = O.attend(q[b:b + 1], kk, vv, torch.ones(1, len(keep), dtype=torch.bool), hq, hkv, SCALE, W_STEP)
            O.close(out[b:b + 1], want, bound)
            at += n[b]
    assert status()["code"] == 0
