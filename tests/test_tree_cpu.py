"""A speculative step's tree on the CPU: masks, attention, the accepted path, the moved rows; and what is refused."""

import math

import paged_oracle as O
import pytest
import torch

from infera_b200.ops import kernels as K
from infera_b200.ops import kv8, tree

SCALE = 1 / math.sqrt(128)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def starts(n):
    return i32([sum(n[:i]) for i in range(len(n))])


def test_mask_accept_and_masks_of_bad_parents():
    g = torch.Generator().manual_seed(1)
    n = [1, 33, 0, 64, 7]
    trees = [O.random_tree(x, g) if x else [] for x in n]
    flat = i32([p for t in trees for p in t])
    mask = tree.tree_mask(flat, starts(n), i32(n), 2)
    at = 0
    for t in trees:
        assert torch.equal(mask[at:at + len(t)], O.mask_of(t, 2))
        at += len(t)
    bad = tree.tree_mask(i32([-1, 0, 2, 9, -5, 1]), i32([0]), i32([6]), 1)
    assert bad[:, 0].tolist() == [1, 3, 4, 8, 16, 32 | 3]
    tokens, target = torch.randint(0, 3, (2, sum(n)), generator=g, dtype=torch.int32)
    for most in (1, 3, 40):
        path, count, after = tree.tree_accept(tokens, target, flat, starts(n), i32(n), most)
        at = 0
        for s, t in enumerate(trees):
            tok, tgt = tokens[at:at + len(t)].tolist(), target[at:at + len(t)].tolist()
            want = O.walk(tok, tgt, t, most)
            assert path[s].tolist() == want + [-1] * (most - len(want)) and int(count[s]) == len(want)
            assert int(after[s]) == (tgt[want[-1]] if want else -1)
            at += len(t)


def batch(n, ctx, hq, hkv, words, seed=0, runs=False):
    g = torch.Generator().manual_seed(seed)
    table, pool = O.page_table(ctx, seed, runs)
    k, v = O.caches(pool, hkv, seed)
    q = torch.randn(sum(n) + 2, (hq + 2 * hkv) * 128, generator=g).to(torch.bfloat16)
    masks = [O.mask_of(O.random_tree(x, g), words) if x else torch.zeros(0, words, dtype=torch.int32) for x in n]
    mask = torch.cat(masks + [torch.zeros(2, words, dtype=torch.int32)])
    return q, k, v, table, mask, masks


@pytest.mark.parametrize("n,ctx,hq,hkv", [([1], [1], 1, 1), ([5, 0, 17], [40, 16, 17], 6, 2), ([9], [3], 4, 1),
                                          ([33, 2], [70, 200], 8, 8)])
def test_attention(n, ctx, hq, hkv):
    words = 2
    q, k, v, table, mask, masks = batch(n, ctx, hq, hkv, words)
    out = torch.full((q.shape[0], hq * 128), 7.0, dtype=torch.bfloat16)
    tree.attn_tree(q, k, v, table, starts(n), i32(n), i32(ctx), mask, hq, hkv, SCALE, out=out)
    at = 0
    for s in range(len(n)):
        kk, vv = (O.rows_of(x, table[s], ctx[s], hkv) for x in (k, v))
        want, bound, _, _ = O.attend(q[at:at + n[s], : hq * 128], kk, vv, O.seen_of(masks[s], n[s], ctx[s]), hq, hkv,
                                     SCALE, 0.0)
        O.close(out[at:at + n[s]], want, bound, f"sequence {s}")
        at += n[s]
    assert torch.all(out[sum(n):] == 7.0)


def test_rows_that_see_nothing_and_values_that_are_not_finite():
    q, k, v, table, mask, _ = batch([4], [4], 2, 1, 1)
    mask[:4, 0] = i32([0, 1, 2, 15])
    v[table[0, 0] * 16 + 1, 5] = float("nan")
    v[table[0, 0] * 16 + 3, 6] = float("inf")
    k[table[0, 0] * 16 + 2] = float("nan")
    out = tree.attn_tree(q, k, v, table, i32([0]), i32([4]), i32([4]), mask, 2, 1, SCALE)
    assert torch.all(out[0] == 0) and bool(out[1].isfinite().all())
    assert out[2, [5, 133]].isnan().all() and int(out[2].isnan().sum()) == 2
    assert torch.equal(out[1, :128], v[table[0, 0] * 16])


def test_refusals():
    q, k, v, table, mask, _ = batch([4, 3], [40, 20], 4, 2, 1)
    args = dict(q=q, k_cache=k, v_cache=v, block_table=table, q_start=i32([0, 4]), q_len=i32([4, 3]),
                ctx_len=i32([40, 20]), mask=mask, hq=4, hkv=2, scale=SCALE)
    tree.attn_tree(**args)
    k8 = kv8.alloc(k.shape[0], 2, device="cpu")
    for change, error in [(dict(k_cache=k8, v_cache=k8), TypeError), (dict(hq=34), ValueError), (dict(hq=3), ValueError),
                          (dict(k_cache=k.float()), ValueError), (dict(k_cache=k[:-1]), ValueError),
                          (dict(v_cache=v[:16]), ValueError), (dict(q=q.float()), ValueError),
                          (dict(q=q[:, :100]), ValueError), (dict(mask=mask[:, :0]), ValueError),
                          (dict(mask=mask.long()), ValueError), (dict(mask=mask[:-1]), ValueError),
                          (dict(mask=mask.repeat(1, 9)), ValueError), (dict(q_len=i32([4])), ValueError),
                          (dict(ctx_len=i32([40, 2000])), ValueError), (dict(q_len=i32([4, 33])), ValueError),
                          (dict(q_len=i32([4, 30])), ValueError), (dict(q_len=i32([4, -1])), ValueError),
                          (dict(host_meta=([4], [40])), ValueError), (dict(block_table=table[:1]), ValueError),
                          (dict(block_table=table.long()), ValueError),
                          (dict(out=torch.empty(9, 100, dtype=torch.bfloat16)), ValueError)]:
        with pytest.raises(error):
            tree.attn_tree(**{**args, **change})
    with pytest.raises(ValueError):
        tree.tree_mask(i32([-1]), i32([0]), i32([1]), 9)
    with pytest.raises(ValueError):
        tree.tree_mask(torch.tensor([-1]), i32([0]), i32([1]), 1)
    with pytest.raises(ValueError):
        tree.tree_accept(i32([1]), i32([1]), i32([-1]), i32([0]), i32([1]), 0)
    with pytest.raises(ValueError):
        tree.tree_accept(i32([1]), i32([1, 2]), i32([-1]), i32([0]), i32([1]), 2)


@pytest.mark.parametrize("layers", [None, 3])
def test_path_rows_move(layers):
    ctx, path = [37, 16], [[0, 2, 5, 9, -1], [0, -1, -1, -1, -1]]
    table, pool = O.page_table([c + 12 for c in ctx], 2)
    k, v = O.caches(pool, 2, 3)
    if layers:
        k, v = (torch.stack([x * (i + 1) for i in range(layers)]) for x in (k, v))
    want = [x.clone() for x in (k, v)]
    for s in range(2):
        want = [O.moved(x, table[s], path[s], ctx[s], x.shape[-1], 0) for x in want]
    K.kv_compact(k, v, table, i32(path), i32([4, 1]), start=i32(ctx))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_moves_of_a_latent_cache_and_refusals():
    table, pool = O.page_table([40], 4)
    k = torch.randn(2, pool * 16, 576).to(torch.bfloat16)
    v = torch.zeros(2, 1, 1, dtype=torch.bfloat16)
    want = O.moved(k, table[0], [3, 4, 30], 5, 576, 0)
    K.kv_compact(k, v, table, i32([[3, 4, 30]]), i32([3]), start=i32([5]))
    assert torch.equal(k, want)
    # entries below their index, beyond the table, on pages outside the cache, a table row twice: not moved
    kc, vc = O.caches(pool, 1, 5)
    was = kc.clone()
    t2 = table.clone()
    t2[0, 1] = pool + 7
    K.kv_compact(kc, vc, t2, i32([[-1, 0, 1, 999, 20]]), i32([5]))
    assert torch.equal(kc, was)
    K.kv_compact(kc, vc, table, i32([[-1, 5], [-1, 9]]), i32([2, 2]), bt_rows=i32([0, 0]))
    assert torch.equal(kc, O.moved(was, table[0], [-1, 5], 0, 128, 0))
    k8 = kv8.alloc(16 * pool, 1, device="cpu")
    good = dict(k_cache=kc, v_cache=vc, block_table=table, src=i32([[1]]), count=i32([1]))
    for change, error in [(dict(k_cache=k8, v_cache=k8), TypeError), (dict(v_cache=kc), ValueError),
                          (dict(k_cache=kc.float(), v_cache=vc.float()), ValueError), (dict(src=i32([1])), ValueError),
                          (dict(src=torch.tensor([[1]])), ValueError), (dict(count=i32([1, 1])), ValueError),
                          (dict(start=i32([1, 2])), ValueError), (dict(src=i32([[[1]] * 3])), ValueError),
                          (dict(k_cache=kc[:-1], v_cache=vc[:-1]), ValueError), (dict(block_table=table[:0]), ValueError),
                          (dict(v_cache=vc[:-16]), ValueError), (dict(v_cache=vc[:, :64]), ValueError)]:
        with pytest.raises(error):
            K.kv_compact(**{**good, **change})
