"""Drafted tokens that form a tree: the masks, the attention and the accepted path of a speculative step.

A step puts each sequence's nodes behind its cached keys: node 0 is the token that the step before chose, every other
node a drafted token that continues its parent. A parent comes before its children; ``parents`` holds the parent's
number in the sequence, -1 for none. The step writes the nodes' keys and values to the next places of the sequence
(each rotated to its depth's position), attends with :func:`attn_tree`, and walks with :func:`tree_accept` along the
nodes that the model would have chosen itself. :func:`infera_b200.ops.kernels.kv_compact` then moves the accepted
nodes' rows together, in every layer, with the path as ``src`` and the sequence's length before the step as ``start``.

Sequences' nodes are rows of flat tensors, as prompt chunks are: sequence s has rows ``q_start[s] .. + q_len[s]``. On
CPU every function computes the same with PyTorch in fp32.

The reference has speculative decoding in the engines that it drives only; there is no source in its tree.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from infera_b200.ops import _native
from infera_b200.ops import kernels as K
from infera_b200.ops import paged
from infera_b200.ops.kv8 import HEAD_DIM, PAGE, _check_heads, _check_i32, _check_rows, _check_table, _name, _on

_BF16, _I32 = torch.bfloat16, torch.int32
MAX_NODES = 256
# Contexts of up to so many tiles of 64 keys are not cut. Captured, uncut against cut: 8 nodes of 32 heads (over 8) in 6
# tiles 11.9 against 13.8 us, in 8 13.8 against 13.4, in 10 15.7 against 13.6, in 14 19.4 against 13.6; 40 trees of 16 nodes
# in 8 tiles 29.3 against 31.3, in 10 33.6 against 33.9, in 14 42.9 against 38.3. (Trees of several items gain from cuts
# later, 4 of 64 nodes and 64 heads not before 20 tiles, 33.1 against 36.1.) Uncut is also one launch instead of two.
UNCUT = 10


def _rows_of(q_start: list[int], q_len: list[int], T: int, most: int) -> list[tuple[int, int]]:
    """(first row, rows) of each sequence, as the kernels take them."""
    return [(s, 0 if not 0 <= s <= T else min(max(n, 0), most, T - s)) for s, n in zip(q_start, q_len)]


def tree_mask(parents: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor, words: int = 2) -> torch.Tensor:
    """int32 [T, words]: bit j of a row's word w is set where node 32*w + j of its sequence is the row's own node or an
    ancestor. Up to 32*words nodes a sequence (words 1 to 8). Rows of no sequence are not written. To the status word:
    a parent that does not come before its node (the node counts as one without), more nodes than fit."""
    T, n, dev = parents.shape[0], q_len.shape[0], parents.get_device()
    _check_i32("parents", parents, T, dev)
    _check_i32("q_start", q_start, n, dev)
    _check_i32("q_len", q_len, n, dev)
    if not 1 <= words <= MAX_NODES // 32:
        raise ValueError(f"{words} words: 1 to {MAX_NODES // 32}")
    mask = torch.empty(T, words, dtype=_I32, device=parents.device)
    if n == 0 or T == 0:
        return mask
    if dev < 0:
        for start, count in _rows_of(q_start.tolist(), q_len.tolist(), T, 32 * words):
            bits = []
            for i, up in enumerate(parents[start:start + count].tolist()):
                bits.append(1 << i | (bits[up] if 0 <= up < i else 0))
                for w in range(words):
                    x = bits[i] >> 32 * w & 0xFFFFFFFF
                    mask[start + i, w] = x - (1 << 32) if x >> 31 else x
        return mask
    status, stream = _on(dev)
    rc = _native.kernels().ib_tree_mask(parents.data_ptr(), q_start.data_ptr(), q_len.data_ptr(), n, T, words,
                                        mask.data_ptr(), status, stream)
    _native.check(rc, "ib_tree_mask")
    K._count()
    return mask


def tree_accept(tokens: torch.Tensor, target: torch.Tensor, parents: torch.Tensor, q_start: torch.Tensor,
                q_len: torch.Tensor, most: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The accepted path of each sequence's tree: from node 0 on to the first child whose token (``tokens`` int32 [T])
    is what the model chose at its parent (``target`` int32 [T], :func:`infera_b200.ops.kernels.sample` of the nodes'
    logits), at most ``most`` nodes.

    Returns (nodes int32 [n, most], ascending, -1 behind the last; how many, int32 [n]; what the model chose at the
    last, int32 [n], the token that the next step starts from). A sequence without nodes has 0 and -1; up to 256 nodes
    (more: left out, to the status word)."""
    T, n, dev = tokens.shape[0], q_len.shape[0], tokens.get_device()
    for name, t in (("tokens", tokens), ("target", target), ("parents", parents)):
        _check_i32(name, t, T, dev)
    _check_i32("q_start", q_start, n, dev)
    _check_i32("q_len", q_len, n, dev)
    if most < 1:
        raise ValueError(f"a path of at most {most} nodes")
    path = torch.empty(n, most, dtype=_I32, device=tokens.device)
    count, after = torch.empty(2, n, dtype=_I32, device=tokens.device).unbind()
    if n == 0:
        return path, count, after
    if dev < 0:
        path.fill_(-1)
        for s, (start, c) in enumerate(_rows_of(q_start.tolist(), q_len.tolist(), T, MAX_NODES)):
            up, tok, tgt = (t[start:start + c].tolist() for t in (parents, tokens, target))
            walk = [0] if c else []
            while walk and len(walk) < most:
                on = [i for i in range(walk[-1] + 1, c) if up[i] == walk[-1] and tok[i] == tgt[walk[-1]]]
                if not on:
                    break
                walk.append(on[0])
            path[s, : len(walk)] = torch.tensor(walk, dtype=_I32)
            count[s], after[s] = len(walk), tgt[walk[-1]] if walk else -1
        return path, count, after
    status, stream = _on(dev)
    rc = _native.kernels().ib_tree_accept(tokens.data_ptr(), target.data_ptr(), parents.data_ptr(), q_start.data_ptr(),
                                          q_len.data_ptr(), n, T, most, path.data_ptr(), count.data_ptr(),
                                          after.data_ptr(), status, stream)
    _native.check(rc, "ib_tree_accept")
    K._count()
    return path, count, after


# ---------------------------------------------------------------- attention


@lru_cache(maxsize=256)
def _plan(q_lens: tuple[int, ...], ctx_lens: tuple[int, ...], group: int, hkv: int, num_sms: int) -> tuple[int, bool]:
    per_item = 128 // group
    units = [3 + (-(-c // 64) or 1) for c in ctx_lens]  # an item's start and end cost some three tiles
    items = [-(-n // per_item) for n in q_lens]
    total = hkv * sum(i * u for i, u in zip(items, units))
    top, levels = max((u for i, u in zip(items, units) if i), default=4), max(1, max(items, default=1))
    ctas = max(1, min(2 * num_sms // levels * levels or levels, -(-total // 5)))
    return ctas, top > UNCUT + 3


def tree_plan(q_lens: list[int], ctx_lens: list[int], hq: int, hkv: int, num_sms: int = 148) -> tuple[int, bool]:
    """(CTAs, whether several may share an item) of :func:`attn_tree`: one wave of two CTAs to an SM, as many for each
    128 rows of the longest tree, at least two tiles of 64 keys each; contexts of up to :data:`UNCUT` tiles are not
    cut."""
    return _plan(tuple(q_lens), tuple(ctx_lens), hq // hkv, hkv, num_sms)


def attn_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
              q_start: torch.Tensor, q_len: torch.Tensor, ctx_len: torch.Tensor, mask: torch.Tensor, hq: int, hkv: int,
              scale: float, out: torch.Tensor | None = None, host_meta: tuple[list[int], list[int]] | None = None,
              bt_rows: torch.Tensor | None = None, plan: tuple[int, bool] | None = None) -> torch.Tensor:
    """Attention of the nodes of trees whose K/V already sit in the bf16 cache. q: [T, >=hq*128] bf16; q_start / q_len
    / ctx_len: int32 [sequences], as of :func:`infera_b200.ops.kernels.attn_prefill`: a sequence's last ``q_len`` of
    ``ctx_len`` keys are its nodes, in order. A node sees all keys before them and the nodes whose bits ``mask`` int32
    [T, words] names (:func:`tree_mask`, or any other mask: its own node need not be among them). Up to 32*words nodes
    (words 1 to 8), up to 16 query heads per KV head. ``out`` may be ``q`` itself.

    ``host_meta`` (q_len, ctx_len on the host; read back from the device without it) sizes the grid and the workspace
    (``plan``: :func:`tree_plan`). In a captured graph the lengths on the device may change from replay to replay: up
    to the most nodes of ``host_meta``, and any context that the page table holds. What ``host_meta``'s contexts do not
    cut (up to :data:`UNCUT` tiles) stays so, and an item of a far longer context is then one CTA's: plan a capture with
    the longest contexts that it will see.

    A row that sees no key is zero; rows of no sequence are left as they are. What a masked key or value holds does not
    reach the row, an infinity or a NaN neither; where a node's value is not finite, rows that see it get it in that
    dim. (An infinity before the nodes makes the rows that dim's infinity, or a NaN where its weight is 0 in bf16.)
    Weights are rounded to bf16 for the product with V, as in the prompt attention. To the status word: more nodes
    than fit (the first are computed), a context beyond the page table's places (cut there: the keys that it has are
    seen as in the whole context), a ``bt_rows`` entry that is no row of the table (its rows are zero). A page id
    outside the cache reads as zeros."""
    _check_heads(hq, hkv, 16)
    n, T, dev = q_len.shape[0], q.shape[0], q.get_device()
    ldq = _check_rows("q", q, T, hq * HEAD_DIM, dev, 16)
    _check_i32("q_start", q_start, n, dev)
    _check_i32("q_len", q_len, n, dev)
    _check_i32("ctx_len", ctx_len, n, dev)
    paged.check_caches(k_cache, v_cache, hkv, dev)
    _check_table(block_table, bt_rows, n, dev)
    words = mask.shape[1] if mask.dim() == 2 else 0
    if mask.dtype is not _I32 or mask.shape[0] != T or not 1 <= words <= MAX_NODES // 32 or not mask.is_contiguous():
        raise ValueError(f"mask: a contiguous int32 [{T}, 1 to {MAX_NODES // 32}], not {tuple(mask.shape)} {mask.dtype}")
    if mask.get_device() != dev:
        raise ValueError(f"mask is on {mask.device}, the queries on {_name(dev)}")
    if host_meta is None:
        if dev >= 0 and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("attn_tree needs host_meta during capture")
        host_meta = (q_len.tolist(), ctx_len.tolist())
    q_lens, ctx_lens = host_meta
    if len(q_lens) != n or len(ctx_lens) != n:
        raise ValueError(f"host_meta is of {len(q_lens)} / {len(ctx_lens)} sequences, q_len of {n}")
    if n and min(q_lens) < 0:
        raise ValueError(f"a tree of {min(q_lens)} nodes")
    most = max(q_lens, default=0)
    if most > 32 * words:
        raise ValueError(f"{most} nodes, the mask has room for {32 * words}")
    if out is None:
        out = torch.empty(T, hq * HEAD_DIM, dtype=_BF16, device=q.device)
        ldo = hq * HEAD_DIM
    else:
        ldo = _check_rows("out", out, T, hq * HEAD_DIM, dev, 16, True)
    if n > 65535:
        raise ValueError(f"{n} sequences")
    places = block_table.shape[1]
    if n and max(ctx_lens) > places * PAGE:
        raise ValueError(f"a context of {max(ctx_lens)} keys needs {-(-max(ctx_lens) // PAGE)} pages, block_table has "
                         f"room for {places}")
    if sum(q_lens) > T:
        raise ValueError(f"{sum(q_lens)} nodes, q has {T} rows")
    if most == 0:
        return out
    if dev < 0:
        _attn_tree_cpu(q, k_cache, v_cache, block_table, q_start.tolist(), q_lens, ctx_lens, mask, hq, hkv, scale, out,
                       bt_rows)
        return out
    ctas, cut = plan or tree_plan(q_lens, ctx_lens, hq, hkv, K._num_sms())
    if not 1 <= ctas <= 65535:
        raise ValueError(f"a plan of {ctas} CTAs")
    part = lse = pieces = None
    if cut:
        # partials of this call: its own memory, so that calls on several streams and captured graphs share none
        m = 2 * ctas * 128
        ws = torch.empty(m * (HEAD_DIM + 1) + 2 * n * hkv * -(-most // (128 // (hq // hkv))), dtype=torch.float32,
                         device=q.device)
        part = ws.data_ptr()
        lse = part + 4 * m * HEAD_DIM
        pieces = lse + 4 * m
    status, stream = _on(dev)
    rc = _native.kernels().ib_attn_tree(q.data_ptr(), T, ldq, k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0],
                                        q_start.data_ptr(), q_len.data_ptr(), ctx_len.data_ptr(), mask.data_ptr(),
                                        words, n, most, block_table.data_ptr(), K._ptr(bt_rows), block_table.shape[0],
                                        places, block_table.stride(0), hq, hkv, scale, ctas, part, lse, pieces,
                                        out.data_ptr(), ldo, status, stream)
    _native.check(rc, "ib_attn_tree")
    K._count(2 if cut else 1)
    return out


def _attn_tree_cpu(q, k_cache, v_cache, block_table, q_start, q_lens, ctx_lens, mask, hq, hkv, scale, out,
                   bt_rows) -> None:
    k, v, bt, lens, _ = paged.cpu_view(k_cache, v_cache, block_table, bt_rows, ctx_lens)
    T, words = mask.shape
    bit = torch.arange(32 * words)
    for i, (start, n) in enumerate(_rows_of(q_start, q_lens, T, 32 * words)):
        if n == 0:
            continue
        rows, ctx, base = slice(start, start + n), lens[i], ctx_lens[i] - q_lens[i]
        if ctx == 0:
            out[rows, : hq * HEAD_DIM] = 0
            continue
        place = torch.arange(ctx) - base
        bits = (mask[rows][:, bit // 32] >> bit % 32) & 1 > 0
        seen = (place < 0) | (bits[:, place.clamp(0, 32 * words - 1)] & (place < 32 * words))
        kb, vb = (paged.cpu_keys(x, bt[i], ctx, hkv) for x in (k, v))
        qi = q[rows, : hq * HEAD_DIM].float().view(n, hkv, -1, HEAD_DIM).permute(1, 2, 0, 3)
        s = (qi @ kb[:, None].transpose(2, 3) * scale).masked_fill(~seen, float("-inf"))
        w = torch.softmax(s, -1).masked_fill(~seen.any(1)[:, None], 0.0)
        # a node's value that is not finite reaches the rows that see it, and not by a weight of zero
        wild = ~vb.isfinite() & (place >= 0)[:, None]
        o = w @ vb.masked_fill(wild, 0.0)[:, None]
        if bool(wild.any()):
            extra = torch.where(seen[None, :, :, None] & wild[:, None], vb[:, None], 0.0).sum(2)  # [hkv, n, 128]
            o = torch.where(extra[:, None] != 0, extra[:, None], o)
        out[rows, : hq * HEAD_DIM] = o.permute(2, 0, 1, 3).reshape(n, -1).to(q.dtype)
