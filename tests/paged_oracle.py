"""Plain 64-bit forms of the calls on the bf16 paged KV cache, and batches for their tests (CPU and GPU).

``attend`` also gives the bound of an output: rounding the result to bf16 costs half a step of it (2^-8 of its size);
rounding a weight costs ``w_step`` of it, and so at most w_step * sum w |v|; a score that is off by d changes a weight
by e^d - 1, and a dot product of 128 exact products added in fp32 is off by at most 128 * 2^-24 * sum |q k| (and the
scale, the maximum's and the sum's roundings and exp2's own error of some 2^-22 are as small: counted as 2^-18).
"""

import torch

D, PAGE = 128, 16


def page_table(lens, seed=0, runs=False, spare=3, extra=0):
    """(table [sequences, most pages + extra], pages of the pool)"""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // PAGE) for n in lens]
    pool = sum(need) + spare
    order = torch.arange(pool) if runs else torch.randperm(pool, generator=g)
    table = torch.zeros(len(lens), max(need, default=0) + extra, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table, pool


def caches(pool, hkv, seed=0):
    g = torch.Generator().manual_seed(seed + 100)
    k = torch.randn(pool * PAGE, hkv * D, generator=g)
    v = torch.randn(pool * PAGE, hkv * D, generator=g) * torch.exp2(torch.randint(-3, 3, (pool * PAGE, 1), generator=g))
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def rows_of(x, table_row, n, hkv):
    """fp64 [n, hkv, 128] of a sequence's first n places; pages outside the cache are zeros."""
    pages = x.shape[0] // PAGE
    t = table_row[: -(-n // PAGE)].long()
    ok = (t >= 0) & (t < pages)
    y = x.double().view(pages, PAGE, hkv, D)[t.clamp(0, pages - 1)] * 1.0
    y[~ok] = 0
    return y.reshape(-1, hkv, D)[:n]


def attend(q, k, v, seen, hq, hkv, scale, w_step):
    """q [rows, hq*128], k / v fp64 [keys, hkv, 128], seen bool [rows, keys] -> (out [rows, hq*128], bound of it, weights
    [rows, hq, keys], bound of them). A value that a row does not see counts as zero; rows that see nothing are zero."""
    r, n = seen.shape
    if n == 0:
        return torch.zeros(2, r, hq * D, dtype=torch.float64).unbind() + torch.zeros(2, r, hq, 0, dtype=torch.float64).unbind()
    qd = q.double().view(r, hq, D)
    G = hq // hkv
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("rhd,khd->rhk", qd, kk) * scale
    mag = torch.einsum("rhd,khd->rhk", qd.abs(), kk.abs()) * abs(scale)
    s = s.masked_fill(~seen[:, None], float("-inf"))
    some = seen.any(1)[:, None, None]
    w = torch.where(some, torch.softmax(s, -1), torch.zeros((), dtype=torch.float64))
    mag = torch.where(seen[:, None], mag, 0.0).nan_to_num(0.0)
    d = 2 * 128 * 2.0 ** -24 * mag.amax(-1, keepdim=True) + 2.0 ** -18
    out, size = torch.zeros(r, hq, D, dtype=torch.float64), torch.zeros(r, hq, D, dtype=torch.float64)
    for h in range(hq):
        x = vv[:, h]
        wild = ~x.isfinite()
        y = x.masked_fill(wild, 0.0)
        out[:, h] = w[:, h] @ y
        size[:, h] = w[:, h] @ y.abs()
        if wild.any():
            extra = torch.where(seen[:, :, None] & wild, x, 0.0).sum(1)
            out[:, h] = torch.where(extra != 0, extra, out[:, h])
    bound = 2.0 ** -8 * out.abs() + (w_step + 2 * d) * size + 1e-37
    return out.view(r, hq * D), bound.view(r, hq * D), w, 2 * d * w


def close(got, want, bound, what=""):
    got, want, bound = got.double().cpu(), want.double(), bound.double()
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]), what
    off = (got - want).abs()[fine] - bound[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {float(off.max())} over the bound, at {int(off.argmax())}"


def mask_of(parents, words):
    """Masks of one tree as lists of ints (bit j: node j)."""
    bits = []
    for i, up in enumerate(parents):
        bits.append(1 << i | (bits[up] if 0 <= up < i else 0))
    rows = [[b >> 32 * w & 0xFFFFFFFF for w in range(words)] for b in bits]
    t = torch.tensor(rows, dtype=torch.int64).view(-1, words)
    return torch.where(t >= 1 << 31, t - (1 << 32), t).to(torch.int32)


def random_tree(n, g):
    return [-1] + [int(torch.randint(max(0, i - 5), i, (1,), generator=g)) for i in range(1, n)]


def seen_of(mask, n, ctx):
    """bool [n, ctx]: what the rows of a tree see of its sequence's ctx keys."""
    words = mask.shape[1]
    base = ctx - n
    seen = torch.ones(n, ctx, dtype=torch.bool)
    for i in range(n):
        for k in range(max(base, 0), ctx):
            j = k - base
            seen[i, k] = j < 32 * words and bool(int(mask[i, j // 32]) >> (j % 32) & 1)
    return seen


def walk(tokens, target, parents, most):
    path = [0] if parents else []
    while path and len(path) < most:
        on = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == target[path[-1]]]
        if not on:
            break
        path.append(on[0])
    return path


def select(x, keep, recent, sink):
    """Places that a list of weights keeps."""
    n = len(x)
    if n <= keep:
        return list(range(n))
    rank = lambda j: (0 if x[j] != x[j] else 1, -x[j] if x[j] == x[j] else 0)  # noqa: E731
    mid = sorted(range(sink, n - recent), key=lambda j: (-rank(j)[0], rank(j)[1], j))[: keep - sink - recent]
    return sorted(list(range(sink)) + mid + list(range(n - recent, n)))


def moved(cache, table_row, src, start, width, at):
    """The cache after the rows src[i] -> i of one list moved, as if all were read first."""
    out = cache.clone()
    slot = lambda p: int(table_row[p // PAGE]) * PAGE + p % PAGE  # noqa: E731
    for i, s in enumerate(src):
        if s > i:
            out[..., slot(start + i), at:at + width] = cache[..., slot(start + s), at:at + width]
    return out
