"""Eviction from the bf16 paged KV cache by accumulated attention weight.

``mass`` (fp32 [rows, hkv, places], a row for each row of the page table) holds what each cached key of a sequence has
received: the softmax weights of a KV head's query heads, summed over the decode steps so far. It starts at zero, and
the prompt calls add nothing to it: until some steps have, all keys of a prompt have the same 0, and of those the lowest
places stay.

* :func:`attn_decode` attends with one query token per sequence and adds the step's weights to ``mass``
  (:func:`infera_b200.ops.kernels.attn_decode` comes here when it is given ``mass``);
* :func:`select_keys` picks the keys that each KV head of a sequence keeps;
* :func:`infera_b200.ops.kernels.kv_compact` moves their rows to the front of the sequence's pages.

After the three the sequence has fewer keys (``select_keys`` returns how many) and needs fewer pages. Each KV head then
holds keys of its own choice, in the order of their positions; keys carry their rotation with them, so later queries
attend as before. On CPU every function computes the same with PyTorch in fp32.

The reference serves with its engines' full caches; it has no counterpart.
"""

from __future__ import annotations

import torch

from infera_b200.ops import _native
from infera_b200.ops import kernels as K
from infera_b200.ops import paged
from infera_b200.ops.kv8 import HEAD_DIM, PAGE, _check_heads, _check_i32, _check_rows, _check_table, _name, _on

_BF16, _F32 = torch.bfloat16, torch.float32
# Scores of a KV head that the CTA of an uncut sequence turns into weights itself; more are spread over the GPU by a
# second kernel. (1 x 100 keys of 32 heads: 8.3 us in one kernel, 8.75 in two; a CTA takes some 1.2 us for 3000 scores,
# and 61 ragged sequences up to 12000 keys took 287 us that way, 256 in two kernels.)
FUSED_SCORES = 8192


def alloc_mass(rows: int, hkv: int, places: int, layers: int | None = None,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """Zeroed weights of ``rows`` sequences with up to ``places`` keys; with ``layers``, ``mass[layer]`` is one layer's."""
    return torch.zeros(*(() if layers is None else (layers,)), rows, hkv, places, dtype=_F32, device=device)


def _check_mass(mass: torch.Tensor, hkv: int, dev: int) -> None:
    if mass.dtype is not _F32 or mass.dim() != 3 or mass.shape[1] != hkv or not mass.is_contiguous():
        raise ValueError(f"mass: a contiguous fp32 [rows, {hkv}, places], not {tuple(mass.shape)} {mass.dtype}")
    if mass.get_device() != dev:
        raise ValueError(f"mass is on {mass.device}, the other tensors on {_name(dev)}")


def decode_plan(batch: int, hkv: int, max_len: int, num_sms: int = 148) -> tuple[int, int]:
    """(splits, 128-key tiles per split) of :func:`attn_decode` for ``batch`` sequences whose longest has ``max_len``
    keys: one wave of the CTAs that fit (two on each SM) if all were that long, and at most 32 tiles."""
    tiles = max(1, -(-max_len // 128))
    shares = max(1, 2 * num_sms // max(1, batch * hkv))
    tps = min(32, -(-tiles // shares))
    return -(-tiles // tps), tps


def attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, hq: int, hkv: int, scale: float, mass: torch.Tensor, splits: int = 1,
                out: torch.Tensor | None = None, bt_rows: torch.Tensor | None = None,
                tiles_per_split: int = 0) -> torch.Tensor:
    """Single-token attention per sequence over the bf16 cache, and ``mass[row, h, j] +=`` the weights that key j got
    from the query heads of KV head h. q: [B, >=hq*128] bf16 (row stride free), seq_lens: int32 [B] (keys including
    the current token; 0 gives a row of zeros). Up to 8 query heads per KV head. A sequence's row of ``mass`` is its
    row of the page table (``bt_rows[b]``, or b). ``out`` may be ``q`` itself.

    ``splits`` and ``tiles_per_split`` come from :func:`decode_plan`: split s covers the 128-key tiles [s*T, (s+1)*T)
    of every sequence, so ``splits * tiles_per_split * 128`` must cover the longest one (``tiles_per_split=0``: enough
    tiles for every key that the page table has room for). The call keeps the raw scores in a workspace of 4 bytes a
    key that the splits cover and query head (1, 2, 4 or 8 to a KV head), for every sequence as for the longest: 1.6 GB for
    128 sequences and 32 heads over 8 where one has 100000 keys.

    What the device finds wrong goes to the status word: keys that no split covers (they are left out), a length beyond
    the page table's places (cut there) or beyond ``mass``'s (no weights are added there), a ``bt_rows`` entry that is
    no row of the table (the sequence gets zeros) or of ``mass``, or that an earlier sequence has (both: no weights are
    added). Sequences of length 0 may share a row with others before them: so a batch is padded. A page id outside the
    cache reads as zeros. An infinity among a sequence's values is the output's in its dim."""
    _check_heads(hq, hkv, 8)
    B, dev = seq_lens.shape[0], q.get_device()
    ldq = _check_rows("q", q, B, hq * HEAD_DIM, dev, 4)
    _check_i32("seq_lens", seq_lens, B, dev)
    paged.check_caches(k_cache, v_cache, hkv, dev)
    _check_table(block_table, bt_rows, B, dev)
    _check_mass(mass, hkv, dev)
    if not 1 <= splits <= 65535 or tiles_per_split < 0 or B > 65535:
        raise ValueError(f"splits {splits}, tiles_per_split {tiles_per_split}, {B} sequences")
    if out is None:
        out = torch.empty(B, hq * HEAD_DIM, dtype=_BF16, device=q.device)
        ldo = hq * HEAD_DIM
    else:
        ldo = _check_rows("out", out, B, hq * HEAD_DIM, dev, 4, True)
    if B == 0:
        return out
    if dev < 0:
        _attn_decode_cpu(q, k_cache, v_cache, block_table, seq_lens, hq, hkv, scale, mass, out, bt_rows)
        return out
    places = block_table.shape[1]
    room = max(1, -(-places * PAGE // 128))  # tiles of the longest sequence that the table can hold
    tiles_per_split = min(tiles_per_split, room) if tiles_per_split else -(-room // splits)
    keys = max(1, min(splits * tiles_per_split * 128, places * PAGE))
    group = hq // hkv
    gp = 1 if group == 1 else 2 if group == 2 else 4 if group <= 4 else 8
    # scores and partials of this call: its own memory, so that calls on several streams and captured graphs share none
    n_s, n = B * hkv * keys * gp + 3 & ~3, B * hq * splits
    ws = torch.empty(n_s + n * (2 + HEAD_DIM if splits > 1 else 2), dtype=_F32, device=q.device)
    scores = ws.data_ptr()
    part = scores + 4 * n_s
    ml = part + 4 * n * HEAD_DIM if splits > 1 else part
    fused = splits == 1 and keys * gp <= FUSED_SCORES
    status, stream = _on(dev)
    rc = _native.kernels().ib_attn_decode_mass(q.data_ptr(), ldq, k_cache.data_ptr(), v_cache.data_ptr(),
                                               k_cache.shape[0], block_table.data_ptr(), K._ptr(bt_rows),
                                               seq_lens.data_ptr(), block_table.shape[0], places,
                                               block_table.stride(0), B, hq, hkv, splits, tiles_per_split, scale,
                                               scores, keys, ml, part if splits > 1 else None, mass.data_ptr(),
                                               mass.shape[0], mass.shape[2], fused, out.data_ptr(), ldo, status, stream)
    _native.check(rc, "ib_attn_decode_mass")
    K._count(1 if fused else 2)
    return out


def _attn_decode_cpu(q, k_cache, v_cache, block_table, seq_lens, hq, hkv, scale, mass, out, bt_rows) -> None:
    k, v, bt, lens, rows = paged.cpu_view(k_cache, v_cache, block_table, bt_rows, seq_lens.tolist())
    y = torch.zeros(len(lens), hq * HEAD_DIM)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        kb, vb = (paged.cpu_keys(x, bt[b], n, hkv) for x in (k, v))
        s = q[b, : hq * HEAD_DIM].float().view(hkv, -1, HEAD_DIM) @ kb.transpose(1, 2) * scale
        w = torch.softmax(s, -1)
        wild = ~vb.isfinite()  # (reaches the row, and not by a weight of zero)
        y[b] = (w @ vb.masked_fill(wild, 0.0) + torch.where(wild, vb, 0.0).sum(1, keepdim=True)).flatten()
        if rows[b] < mass.shape[0] and rows[b] not in rows[:b]:
            cut = min(n, mass.shape[2])
            mass[rows[b], :, :cut] += w.sum(1)[:, :cut]
    out[: len(lens), : hq * HEAD_DIM] = y.to(_BF16)


# ---------------------------------------------------------------- selection


def _select_ctas(lists: int, places: int, num_sms: int = 148) -> int:
    """CTAs that share a list of :func:`select_keys`."""
    ctas = 1
    while ctas < 8 and 2 * lists * ctas <= num_sms and places > 4096 * ctas:
        ctas *= 2
    return ctas


def select_keys(mass: torch.Tensor, seq_lens: torch.Tensor, keep: int, recent: int = 0, sink: int = 0,
                bt_rows: torch.Tensor | None = None, update: bool = False
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The keys that each KV head of each sequence keeps: its first ``sink``, its last ``recent`` and, of the others,
    those with the largest ``mass`` (equal ones: the lowest place first; a NaN is below every number), ``keep`` in all.
    A sequence of up to ``keep`` keys keeps them all. seq_lens: int32 [n]; sequence s has row ``bt_rows[s]`` (or s) of
    ``mass`` [rows, hkv, places].

    Returns (places int32 [n, hkv, keep], ascending, -1 behind the last; their mass fp32 [n, hkv, keep], 0 behind the
    last; keys that each sequence keeps, int32 [n]). ``update=True`` also brings ``mass`` in line with a cache whose
    rows were moved together (:func:`infera_b200.ops.kernels.kv_compact` with the places and counts): the kept mass at
    the front, zero behind it.

    To the status word: a length beyond ``mass``'s places (cut there), a ``bt_rows`` entry that is no row of ``mass``
    or, with ``update``, that an earlier sequence has (it keeps nothing). Sequences of length 0 may share a row with others
    before them."""
    if mass.dim() != 3:
        raise ValueError(f"mass: [rows, hkv, places], not {tuple(mass.shape)}")
    hkv, n, dev = mass.shape[1], seq_lens.shape[0], mass.get_device()
    _check_mass(mass, hkv, dev)
    _check_i32("seq_lens", seq_lens, n, dev)
    if bt_rows is not None:
        _check_i32("bt_rows", bt_rows, n, dev)
    if hkv < 1 or keep < 1 or recent < 0 or sink < 0 or sink + recent > keep:
        raise ValueError(f"keep {keep} of {hkv} heads' keys: at least one, the first {sink} and the last {recent} among them")
    kept = torch.empty(n, hkv, keep, dtype=torch.int32, device=mass.device)
    kept_mass = torch.empty(n, hkv, keep, dtype=_F32, device=mass.device)
    count = torch.empty(n, dtype=torch.int32, device=mass.device)
    if n == 0:
        return kept, kept_mass, count
    if dev < 0:
        _select_cpu(mass, seq_lens, keep, recent, sink, bt_rows, update, kept, kept_mass, count)
        return kept, kept_mass, count
    status, stream = _on(dev)
    rc = _native.kernels().ib_kv_select(mass.data_ptr(), mass.shape[0], hkv, mass.shape[2], seq_lens.data_ptr(),
                                        K._ptr(bt_rows), n, keep, sink, recent, int(update),
                                        _select_ctas(n * hkv, mass.shape[2], K._num_sms()), kept.data_ptr(),
                                        kept_mass.data_ptr(), count.data_ptr(), status, stream)
    _native.check(rc, "ib_kv_select")
    K._count()
    return kept, kept_mass, count


def _select_cpu(mass, seq_lens, keep, recent, sink, bt_rows, update, kept, kept_mass, count) -> None:
    kept.fill_(-1)
    kept_mass.zero_()
    rows = list(range(len(seq_lens))) if bt_rows is None else bt_rows.tolist()
    for s, (row, n) in enumerate(zip(rows, seq_lens.tolist())):
        bad = not 0 <= row < mass.shape[0] or (update and row in rows[:s])
        n = 0 if bad else min(max(n, 0), mass.shape[2])
        count[s] = min(n, keep)
        for h in range(mass.shape[1]):
            x = mass[row, h, :n] if n else mass.new_empty(0)
            on = torch.arange(n)
            if n > keep:
                mid = x[sink:n - recent]
                value = torch.where(mid == float("-inf"), -1e300, mid.double())  # a NaN is below them all
                value = torch.where(mid.isnan(), float("-inf"), value)
                best = torch.sort(value, descending=True, stable=True).indices[: keep - sink - recent]
                on = torch.cat([on[:sink], sink + best.sort().values, on[n - recent:]])
            kept[s, h, : len(on)] = on.to(torch.int32)
            kept_mass[s, h, : len(on)] = x[on]
            if update and n > keep:
                mass[row, h, :n] = 0
                mass[row, h, :keep] = kept_mass[s, h]
