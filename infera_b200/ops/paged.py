"""What the calls on the bf16 paged KV cache that came after the 8-bit one share: their checks, the view of a batch
that their CPU forms take, and :func:`kv_compact`, which moves rows within sequences' pages.

A layer's cache is a pair of bf16 [slots, hkv*128], slot = page*16 + offset.
"""

from __future__ import annotations

import torch

from infera_b200.ops import _native
from infera_b200.ops import kernels as K
from infera_b200.ops.kv8 import HEAD_DIM, PAGE, KV8Cache, _check_i32, _check_table, _name, _on

_BF16, _I32 = torch.bfloat16, torch.int32


def check_caches(k: torch.Tensor, v: torch.Tensor, hkv: int, dev: int) -> None:
    if type(k) is KV8Cache or type(v) is KV8Cache:
        raise TypeError("this call reads bf16 caches, not a KV8Cache")
    if k.dtype is not _BF16 or v.dtype is not _BF16:
        raise ValueError(f"caches of {k.dtype} and {v.dtype}, not bf16")
    shape = k.shape
    if len(shape) != 2 or shape != v.shape or shape[1] != hkv * HEAD_DIM or shape[0] < PAGE or shape[0] % PAGE:
        raise ValueError(f"caches {tuple(shape)} and {tuple(v.shape)}: both [slots, {hkv} * {HEAD_DIM}] of one layer, "
                         f"whole pages of {PAGE} slots")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("the caches have to be contiguous")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError(f"caches on {k.device} and {v.device}, queries on {_name(dev)}")
    if dev >= 0 and (k.data_ptr() | v.data_ptr()) & 15:
        raise ValueError("the caches have to start on multiples of 16 bytes")


def cpu_view(k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, bt_rows: torch.Tensor | None,
             lens: list[int]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, list[int], list[int]]:
    """(K, V, page table, lengths, table rows) of a batch as the kernels take them: fp32 caches that end with a page of
    zeros, which page ids outside the cache name; lengths end where the table does, and are 0 (row -1) where
    ``bt_rows`` names no row of it."""
    pages, (table_rows, places) = k.shape[0] // PAGE, block_table.shape
    k, v = (torch.cat([c.float(), torch.zeros(PAGE, c.shape[1])]) for c in (k, v))
    rows = list(range(len(lens))) if bt_rows is None else bt_rows.tolist()
    rows = [r if 0 <= r < table_rows else -1 for r in rows]
    if not table_rows:
        return k, v, block_table.new_zeros(len(lens), places), [0] * len(lens), rows
    bt = block_table[torch.tensor(rows, dtype=torch.long).clamp(min=0)].long()
    return (k, v, torch.where((bt >= 0) & (bt < pages), bt, pages),
            [min(max(n, 0), places * PAGE) if r >= 0 else 0 for n, r in zip(lens, rows)], rows)


def cpu_keys(x: torch.Tensor, table_row: torch.Tensor, n: int, hkv: int) -> torch.Tensor:
    """[hkv, n, 128] of the first n keys of one sequence."""
    slots = (table_row[: -(-n // PAGE), None] * PAGE + torch.arange(PAGE)).flatten()[:n]
    return x[slots].view(n, hkv, HEAD_DIM).transpose(0, 1)


# ---------------------------------------------------------------- moving rows


def kv_compact(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, src: torch.Tensor,
               count: torch.Tensor, start: torch.Tensor | None = None, bt_rows: torch.Tensor | None = None) -> None:
    """See :func:`infera_b200.ops.kernels.kv_compact`."""
    if type(k_cache) is KV8Cache or type(v_cache) is KV8Cache:
        raise TypeError("rows of a KV8Cache do not move alone: 16 of them share a scale")
    shape, dev = k_cache.shape, k_cache.get_device()
    if k_cache.dtype is not _BF16 or v_cache.dtype is not _BF16:
        raise ValueError(f"caches of {k_cache.dtype} and {v_cache.dtype}, not bf16")
    two = v_cache.shape == shape
    if len(shape) not in (2, 3) or v_cache.dim() != len(shape) or shape[-2] < PAGE or shape[-2] % PAGE:
        raise ValueError(f"caches {tuple(shape)} and {tuple(v_cache.shape)}: [(layers,) slots, width], whole pages of "
                         f"{PAGE} slots")
    if not two and v_cache.shape[-2:] != (1, 1):  # (a latent cache's V is a placeholder)
        raise ValueError(f"caches {tuple(shape)} and {tuple(v_cache.shape)}: K and V differ")
    if not k_cache.is_contiguous() or (two and not v_cache.is_contiguous()):
        raise ValueError("the caches have to be contiguous")
    if v_cache.get_device() != dev:
        raise ValueError(f"caches on {k_cache.device} and {v_cache.device}")
    dims = src.dim()
    if src.dtype is not _I32 or dims not in (2, 3) or not src.is_contiguous():
        raise ValueError(f"src: a contiguous int32 [sequences, (KV heads,) rows], not {tuple(src.shape)} {src.dtype}")
    if src.get_device() != dev:
        raise ValueError(f"src is on {src.device}, the caches on {_name(dev)}")
    n, m = src.shape[0], src.shape[-1]
    heads = src.shape[1] if dims == 3 else 1
    _check_i32("count", count, n, dev)
    if start is not None:
        _check_i32("start", start, n, dev)
    _check_table(block_table, bt_rows, n, dev)
    width = shape[-1]
    if heads < 1 or width % heads or (width // heads) % 8:
        raise ValueError(f"rows of {width} elements for {heads} heads: a multiple of 8 elements each")
    kp, vp = k_cache.data_ptr(), v_cache.data_ptr() if two else 0
    if two and abs(kp - vp) < k_cache.numel() * 2:
        raise ValueError("K and V are the same memory")
    if n == 0 or m == 0 or k_cache.numel() == 0:
        return
    if dev < 0:
        _kv_compact_cpu(k_cache, v_cache if two else None, block_table, src, count, start, bt_rows)
        return
    if (kp | vp) & 15:
        raise ValueError("the caches have to start on multiples of 16 bytes")
    status, stream = _on(dev)
    rc = _native.kernels().ib_kv_compact(kp, vp or None, shape[0] if len(shape) == 3 else 1, shape[-2], 2 * width,
                                         block_table.data_ptr(), K._ptr(bt_rows), block_table.shape[0],
                                         block_table.shape[1], block_table.stride(0), src.data_ptr(), n, heads, m,
                                         count.data_ptr(), K._ptr(start), K._num_sms(), status, stream)
    _native.check(rc, "ib_kv_compact")
    K._count()


def _kv_compact_cpu(k, v, block_table, src, count, start, bt_rows) -> None:
    (table_rows, places), pages = block_table.shape, k.shape[-2] // PAGE
    heads = src.shape[1] if src.dim() == 3 else 1
    src = src.view(src.shape[0], heads, -1).long()
    rows = list(range(src.shape[0])) if bt_rows is None else bt_rows.tolist()
    for s, row in enumerate(rows):
        first = 0 if start is None else int(start[s])
        if not 0 <= row < table_rows or row in rows[:s] or first < 0:
            continue
        m = min(max(int(count[s]), 0), src.shape[2])
        for h in range(heads):
            to = torch.arange(m)
            frm = src[s, h, :m]
            ok = (frm > to) & (first + frm < places * PAGE)
            frm, to = first + frm[ok], first + to[ok]
            pf, pt = block_table[row, frm // PAGE].long(), block_table[row, to // PAGE].long()
            ok = (pf >= 0) & (pf < pages) & (pt >= 0) & (pt < pages)
            a, b = (pf * PAGE + frm % PAGE)[ok], (pt * PAGE + to % PAGE)[ok]
            w = k.shape[-1] // heads
            for c in (k,) if v is None else (k, v):
                c[..., b, h * w:(h + 1) * w] = c[..., a, h * w:(h + 1) * w].clone()
