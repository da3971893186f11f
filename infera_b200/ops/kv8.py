"""An 8-bit paged KV cache and the attention that reads it.

One channel (K or V) of a layer holds

* ``q``  [slots, hkv*128] float8_e4m3fn, slot = page*16 + offset, and
* ``sf`` [slots/16, hkv] uint8: one scale 2^(sf-127) for each page of 16
  tokens and KV head (0 counts as 1, so a zeroed cache holds zeros; 254 and
  255 as 253, whose inverse is a normal number too: no append needs more than
  247).

A key or value element is ``q * 2^(sf-127)``: half the bytes of the bf16 cache
plus 1/2048 for the scales. A power of two keeps both conversions exact: a
page whose scale grows keeps its codes' values (only codes that become
subnormal round again), and code times scale is exact in bf16.

* :func:`rope_kvwrite` rotates q, and writes k (rotated) and v of an engine
  step's rows. A page's scale is the smallest that holds every finite value
  of the rows written to it (largest code 448). Writing a page's first slot
  starts the page anew: its scale comes from this call's rows alone, and its
  other slots hold nothing until they are written. Any other write keeps at
  least the page's scale and brings the page's other rows to a grown one.
  An infinity or a NaN is stored as NaN. Two rows with the same slot: the
  later one stays.
* :func:`attn_decode` attends with one query token per sequence.
* :func:`attn_prefill` attends causally with chunks of new tokens.

Both give the result in bf16 as if from exact arithmetic over the codes, as
long as neither a query's elements nor a head's page scales of V are worlds
apart: a query element is exact down to 2^-13 of the head's largest element and
off by at most 2^-21 of that one below it; a weight is rounded to 2^-12 of
itself, or to 2^-26 (prompts: 2^-31) of the row's largest weight counted at the
largest scale that the row sees.

:mod:`infera_b200.ops.kernels`'s ``rope_kvwrite``, ``attn_decode`` and
``attn_prefill`` come here for :class:`KV8Cache` caches. On CPU every
function computes the same values with PyTorch in fp32.

Reference counterpart: the reference's engines serve with fp8 KV caches
(their stock workers' default); the kernels are not in its tree.
"""

from __future__ import annotations

import torch

from infera_b200.ops import _native
from infera_b200.ops import kernels as K

E4M3_MAX = 448.0
PAGE = 16
HEAD_DIM = 128
MAX_EXP = 253
_BF16, _I32, _U8, _E4M3 = torch.bfloat16, torch.int32, torch.uint8, torch.float8_e4m3fn


class KV8Cache:
    """One channel (K or V) of one layer, or of all layers with a leading
    dimension; ``cache[layer]`` is one layer's. The tensors are checked here,
    once, and stay what they are."""

    __slots__ = ("q", "sf", "slots", "hkv", "dev", "_layers")

    def __init__(self, q: torch.Tensor, sf: torch.Tensor):
        self.q = q    # [(layers,) slots, hkv*128] float8_e4m3fn
        self.sf = sf  # [(layers,) slots/16, hkv] uint8
        qs, ss = q.shape, sf.shape
        if q.dtype is not _E4M3 or sf.dtype is not _U8:
            raise ValueError(f"a KV8Cache holds float8_e4m3fn codes and uint8 scales, not {q.dtype} and {sf.dtype}")
        if len(ss) == 2:
            pages, heads = ss
            whole = qs == (pages * PAGE, heads * HEAD_DIM)
            self._layers = None
        else:
            layers, pages, heads = ss if len(ss) == 3 else (0, 0, 0)
            whole = layers > 0 and qs == (layers, pages * PAGE, heads * HEAD_DIM)
            self._layers = [KV8Cache(q[i], sf[i]) for i in range(layers)] if whole else None
        if not whole or pages < 1 or heads < 1:
            raise ValueError(f"codes {tuple(qs)} and scales {tuple(ss)} do not hold whole pages of {PAGE} slots with "
                             f"heads of {HEAD_DIM}")
        if not (q.is_contiguous() and sf.is_contiguous()):
            raise ValueError("a KV8Cache's tensors have to be contiguous")
        self.slots, self.hkv, self.dev = pages * PAGE, heads, q.get_device()
        if sf.get_device() != self.dev:
            raise ValueError(f"codes on {q.device}, scales on {sf.device}")
        if self.dev >= 0 and q.data_ptr() & 15:
            raise ValueError("a KV8Cache's codes have to start on a multiple of 16 bytes")

    @property
    def shape(self) -> torch.Size:
        return self.q.shape

    @property
    def device(self) -> torch.device:
        return self.q.device

    @property
    def is_cuda(self) -> bool:
        return self.q.is_cuda

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.sf.numel()

    def __getitem__(self, layer: int) -> "KV8Cache":
        if self._layers is None:
            raise TypeError("this KV8Cache is one layer's")
        return self._layers[layer]

    def to(self, device) -> "KV8Cache":
        return KV8Cache(self.q.to(device), self.sf.to(device))

    def dequant(self) -> torch.Tensor:
        """fp32 [.., slots, hkv*128]."""
        s = _pow2(_exponents(self.sf) - 127)
        x = self.q.float().unflatten(-1, (self.hkv, -1)).unflatten(-3, (-1, PAGE))
        return (x * s[..., :, None, :, None]).flatten(-4, -3).flatten(-2)


def alloc(slots: int, hkv: int, layers: int | None = None, device: torch.device | str = "cuda") -> KV8Cache:
    """One zeroed channel of ``slots`` slots (a multiple of 16) and ``hkv`` heads of 128."""
    if slots < PAGE or slots % PAGE or hkv < 1:
        raise ValueError(f"{slots} slots x {hkv} heads: whole pages of {PAGE} slots and at least one head")
    lead = () if layers is None else (layers,)
    return KV8Cache(torch.zeros(*lead, slots, hkv * HEAD_DIM, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                    torch.zeros(*lead, slots // PAGE, hkv, dtype=torch.uint8, device=device))


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, e a whole number in [-126, 127], from its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponents(sf: torch.Tensor) -> torch.Tensor:
    return sf.to(torch.int32).clamp(1, MAX_EXP)


def _scale_exp(amax: torch.Tensor) -> torch.Tensor:
    """Smallest biased exponent e in [1, 253] with amax <= 448 * 2^(e-127)."""
    m, e = torch.frexp(amax.double() / E4M3_MAX)
    e = torch.where(m == 0.5, e - 1, e) + 127
    return torch.where(amax > 0, e, torch.ones_like(e)).clamp(1, MAX_EXP).to(torch.int32)


# ---------------------------------------------------------------- checks
# The calls take some 10 us of host time, a small batch's kernel less: each
# check is one comparison of plain attributes, and words its error only after
# it failed.


def _check_caches(k: KV8Cache, v: KV8Cache, hkv: int, dev: int) -> None:
    if type(k) is not KV8Cache or type(v) is not KV8Cache:
        raise TypeError(f"caches of {type(k).__name__} and {type(v).__name__}: K and V are both KV8Cache, or neither")
    if k._layers is not None or v._layers is not None:
        raise ValueError("the caches hold all layers: pass one layer's, cache[layer]")
    if k.hkv != hkv or v.hkv != hkv:
        raise ValueError(f"the caches hold {k.hkv} and {v.hkv} heads, not {hkv}")
    if k.slots != v.slots:
        raise ValueError(f"the caches hold {k.slots} and {v.slots} slots")
    if k.dev != dev or v.dev != dev:
        raise ValueError(f"caches on {k.device} and {v.device}, queries on {_name(dev)}")


def _name(dev: int) -> str:
    return "cpu" if dev < 0 else f"cuda:{dev}"


def _check_i32(name: str, t: torch.Tensor, n: int, dev: int) -> None:
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 vector of {n}, not {tuple(t.shape)} {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the queries on {_name(dev)}")


def _check_heads(hq: int, hkv: int, most: int) -> None:
    if hkv < 1 or hq < 1 or hq % hkv or hq // hkv > most:
        raise ValueError(f"{hq} query heads over {hkv} KV heads: a whole number of at most {most} to one")


def _check_rows(name: str, t: torch.Tensor, rows: int, width: int, dev: int, align: int, written: bool = False) -> int:
    """Rows of ``width`` adjacent bf16 elements; returns their pitch. Rows that are written share no memory."""
    shape = t.shape
    if t.dtype is not _BF16 or len(shape) != 2 or shape[0] < rows or shape[1] < width:
        raise ValueError(f"{name}: bf16 [{rows} or more, {width} or more], not {tuple(shape)} {t.dtype}")
    pitch, one = t.stride()
    if one != 1:
        raise ValueError(f"{name}: a row's elements have to be adjacent, not {one} apart")
    if written and pitch < width and shape[0] > 1:
        raise ValueError(f"{name}: rows of {width} elements that start {pitch} apart share memory")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the queries on {_name(dev)}")
    if dev >= 0 and (t.data_ptr() | (2 * pitch if shape[0] > 1 else 0)) & (align - 1):
        raise ValueError(f"{name}: rows have to start on multiples of {align} bytes")
    return pitch if shape[0] > 1 else width  # (of a single row the pitch means nothing)


def _check_table(table: torch.Tensor, bt_rows: torch.Tensor | None, n: int, dev: int) -> None:
    if table.dtype is not _I32 or table.dim() != 2 or (table.stride(1) != 1 and table.shape[1] > 1):
        raise ValueError("block_table: int32 [rows, pages] with adjacent pages")
    if table.get_device() != dev:
        raise ValueError(f"block_table is on {table.device}, the queries on {_name(dev)}")
    if bt_rows is not None:
        _check_i32("bt_rows", bt_rows, n, dev)
    elif table.shape[0] < n:
        raise ValueError(f"block_table has {table.shape[0]} rows for {n} sequences")


def _on(dev: int) -> tuple[int, int]:
    """(status word, stream) of a launch on the current device, which ``dev`` has to be."""
    sc = K._scratch.get(dev)
    if sc is None or torch._C._cuda_getDevice() != dev:
        sc = K.scratch(dev)  # made now, or refused
    return sc.status.data_ptr(), torch._C._cuda_getCurrentRawStream(dev)


# ---------------------------------------------------------------- append


def rope_kvwrite(qkv: torch.Tensor, pos: torch.Tensor, slots: torch.Tensor, cos_sin: torch.Tensor, hq: int,
                 hkv: int, head_dim: int, k_cache: KV8Cache, v_cache: KV8Cache,
                 q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate the q heads of ``qkv`` [T, >=(hq+2*hkv)*128] (bf16; q, k, v side
    by side) into ``q_out`` [T, >=hq*128] (None: in place) and append the rotated
    k and the v to the caches at ``slots`` (int32; -1: not stored). ``qkv``'s
    k and v are left as they are. Returns ``q_out``."""
    if head_dim != HEAD_DIM:
        raise ValueError(f"head_dim {head_dim}: the 8-bit cache holds heads of {HEAD_DIM}")
    _check_heads(hq, hkv, hq)
    T, dev = qkv.shape[0], qkv.get_device()
    ld = _check_rows("qkv", qkv, T, (hq + 2 * hkv) * HEAD_DIM, dev, 16, q_out is None)
    if q_out is None:
        q_out, ldq = qkv, ld
    else:
        ldq = _check_rows("q_out", q_out, T, hq * HEAD_DIM, dev, 16, True)
    _check_i32("pos", pos, T, dev)
    _check_i32("slots", slots, T, dev)
    _check_caches(k_cache, v_cache, hkv, dev)
    kq, vq = k_cache.q.data_ptr(), v_cache.q.data_ptr()
    if abs(kq - vq) < k_cache.slots * hkv * HEAD_DIM or k_cache.sf.data_ptr() == v_cache.sf.data_ptr():
        raise ValueError("K and V are appended to the same memory")
    max_pos = cos_sin.shape[0]
    if cos_sin.dtype is not torch.float32 or cos_sin.shape != (max_pos, HEAD_DIM // 2, 2) \
            or not cos_sin.is_contiguous():
        raise ValueError(f"cos_sin: contiguous fp32 [positions, {HEAD_DIM // 2}, 2], not {tuple(cos_sin.shape)} "
                         f"{cos_sin.dtype}")
    if cos_sin.get_device() != dev or (dev >= 0 and cos_sin.data_ptr() & 15):
        raise ValueError(f"cos_sin on {cos_sin.device} at {cos_sin.data_ptr():#x}: on the queries' device, at a "
                         "multiple of 16 bytes")
    if T == 0:
        return q_out
    if dev < 0:
        _rope_kvwrite_cpu(qkv, pos, slots, cos_sin, hq, hkv, k_cache, v_cache, q_out)
        return q_out
    status, stream = _on(dev)
    rc = _native.kernels().ib_kv8_append(qkv.data_ptr(), T, ld, q_out.data_ptr(), ldq, pos.data_ptr(),
                                         slots.data_ptr(), cos_sin.data_ptr(), hq, hkv, kq, k_cache.sf.data_ptr(),
                                         vq, v_cache.sf.data_ptr(), k_cache.slots, max_pos, status, stream)
    _native.check(rc, "ib_kv8_append")
    K._count()
    return q_out


def _rope_kvwrite_cpu(qkv, pos, slots, cos_sin, hq, hkv, k_cache, v_cache, q_out) -> None:
    T, half = qkv.shape[0], HEAD_DIM // 2
    ok = (pos >= 0) & (pos < cos_sin.shape[0])
    cs = cos_sin[pos.long().clamp(0, cos_sin.shape[0] - 1)][:, None]
    c, s = cs[..., 0], cs[..., 1]
    x = qkv[:, : (hq + 2 * hkv) * HEAD_DIM].float().view(T, hq + 2 * hkv, HEAD_DIM)
    a, b = x[:, : hq + hkv, :half], x[:, : hq + hkv, half:]
    rot = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    q_out[:T, : hq * HEAD_DIM][ok] = rot[:, :hq].to(qkv.dtype).reshape(T, -1)[ok]
    live = ok & (slots >= 0) & (slots < k_cache.q.shape[0])
    for cache, rows in ((k_cache, rot[:, hq:]), (v_cache, x[:, hq + hkv:])):
        codes = cache.q.view(-1, PAGE, hkv, HEAD_DIM)
        on: dict[int, dict[int, int]] = {}
        for t in torch.nonzero(live).flatten().tolist():
            on.setdefault(int(slots[t]) // PAGE, {})[int(slots[t]) % PAGE] = t
        for page, at in on.items():
            offs = list(at)
            new = rows[list(at.values())]
            new = torch.where(new.isfinite(), new, float("nan"))
            e = _scale_exp(torch.nan_to_num(new, nan=0.0).abs().amax(dim=(0, 2)))
            if 0 not in at:
                old = _exponents(cache.sf[page])
                e = torch.maximum(e, old)
                shift = _pow2((old - e).clamp_min(-60))
                codes[page] = (codes[page].float() * shift[None, :, None]).to(torch.float8_e4m3fn)
            codes[page, offs] = (new * _pow2(127 - e)[None, :, None]).to(torch.float8_e4m3fn)
            cache.sf[page] = e.to(torch.uint8)


# ---------------------------------------------------------------- decode attention


def decode_plan(batch: int, hkv: int, max_len: int, num_sms: int = 148, group: int = 4) -> tuple[int, int]:
    """(splits, 128-key tiles per split) of :func:`attn_decode` for ``batch``
    sequences whose longest has ``max_len`` keys, ``group`` query heads to a
    KV head: one wave of the CTAs that fit (three on each SM, two for more
    than 4 heads) if all were that long, and at most 32 tiles. A CTA alone
    takes 0.75 to 1 us a tile and some 3 us to start, so few sequences want
    short shares (1 x 8000 keys over 8 heads: 9.7 us in shares of 2 tiles, 47
    us in one of 64), and shares beyond 32 tiles gain no more (32 x 8192 with
    8 heads: 333 us at 1, 96 at 16, 89 at 32, 86 at 64) while ragged batches
    lose their balance."""
    tiles = max(1, -(-max_len // 128))
    ctas = max(1, batch * hkv)
    shares = max(1, num_sms * (3 if group <= 4 else 2) // ctas)
    tps = min(32, -(-tiles // shares))
    return -(-tiles // tps), tps


def attn_decode(q: torch.Tensor, k_cache: KV8Cache, v_cache: KV8Cache, block_table: torch.Tensor,
                seq_lens: torch.Tensor, hq: int, hkv: int, scale: float, splits: int = 1,
                out: torch.Tensor | None = None, bt_rows: torch.Tensor | None = None,
                tiles_per_split: int = 0) -> torch.Tensor:
    """Single-token attention per sequence over the 8-bit cache. q: [B,
    >=hq*128] bf16 (row stride free), seq_lens: int32 [B] (keys including the
    current token; 0 gives a row of zeros). Up to 8 query heads per KV head.
    ``out`` may be ``q`` itself.

    ``splits`` and ``tiles_per_split`` come from :func:`decode_plan`: split s
    covers the 128-key tiles [s*T, (s+1)*T) of every sequence, so ``splits *
    tiles_per_split * 128`` must cover the longest one (``tiles_per_split=0``:
    enough tiles for every key that the page table has room for).

    What the device finds wrong goes to the status word: keys that no split
    covers (they are left out), a length beyond the page table's places (cut
    there), a ``bt_rows`` entry that is no row of the table (the sequence gets
    zeros). A page id outside the cache reads as zeros."""
    _check_heads(hq, hkv, 8)
    B, dev = seq_lens.shape[0], q.get_device()
    ldq = _check_rows("q", q, B, hq * HEAD_DIM, dev, 4)
    _check_i32("seq_lens", seq_lens, B, dev)
    _check_caches(k_cache, v_cache, hkv, dev)
    _check_table(block_table, bt_rows, B, dev)
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
        _attn_decode_cpu(q, k_cache, v_cache, block_table, seq_lens, hq, hkv, scale, out, bt_rows)
        return out
    places = block_table.shape[1]
    room = max(1, -(-places * PAGE // 128))  # tiles of the longest sequence that the table can hold
    tiles_per_split = min(tiles_per_split, room) if tiles_per_split else -(-room // splits)
    part = lse = None
    if splits > 1:
        # partials of this call: its own memory, so that calls on several
        # streams and captured graphs share none
        n = B * hq * splits
        ws = torch.empty(n * (HEAD_DIM + 1), dtype=torch.float32, device=q.device)
        part = ws.data_ptr()
        lse = part + 4 * n * HEAD_DIM
    status, stream = _on(dev)
    rc = _native.kernels().ib_attn_decode_kv8(q.data_ptr(), ldq, k_cache.q.data_ptr(), k_cache.sf.data_ptr(),
                                              v_cache.q.data_ptr(), v_cache.sf.data_ptr(), k_cache.slots,
                                              block_table.data_ptr(), K._ptr(bt_rows), seq_lens.data_ptr(),
                                              block_table.shape[0], places, block_table.stride(0), B, hq, hkv,
                                              splits, tiles_per_split, scale, part, lse, out.data_ptr(), ldo, status,
                                              stream)
    _native.check(rc, "ib_attn_decode_kv8")
    K._count(2 if splits > 1 else 1)
    return out


def _cpu_view(k_cache, v_cache, block_table, bt_rows, lens) -> tuple:
    """(K, V, page table, lengths) for the CPU forms, what the kernels find wrong treated alike: the values end with a
    page of zeros, which page ids outside the cache name; lengths end where the table does, and are 0 where ``bt_rows``
    names no row of it."""
    pages, (table_rows, places) = k_cache.sf.shape[0], block_table.shape
    k, v = (torch.cat([c.dequant(), torch.zeros(PAGE, c.hkv * HEAD_DIM)]) for c in (k_cache, v_cache))
    rows = torch.arange(len(lens)) if bt_rows is None else bt_rows.long()
    known = ((rows >= 0) & (rows < table_rows)).tolist()
    if not table_rows:
        return k, v, block_table.new_zeros(len(lens), places), [0] * len(lens)
    bt = block_table[rows.clamp(0, table_rows - 1)].long()
    return (k, v, torch.where((bt >= 0) & (bt < pages), bt, pages),
            [min(max(n, 0), places * PAGE) if ok else 0 for n, ok in zip(lens, known)])


def _attn_decode_cpu(q, k_cache, v_cache, block_table, seq_lens, hq, hkv, scale, out, bt_rows) -> None:
    k, v, bt, lens = _cpu_view(k_cache, v_cache, block_table, bt_rows, seq_lens.tolist())
    y = out[: len(lens), : hq * HEAD_DIM]
    some = [b for b, n in enumerate(lens) if n > 0]
    kept = [lens[b] for b in some]
    rows = K._ref_attention(q[some, : hq * HEAD_DIM], k, v, bt[some], [[n - 1] for n in kept], kept, hq, hkv, scale)
    y.zero_()  # (may be q)
    if some:
        y[some] = torch.cat(rows, 0).to(q.dtype)


# ---------------------------------------------------------------- prompt attention


def prefill_plan(q_lens: list[int], ctx_lens: list[int], hq: int, hkv: int, num_sms: int = 148
                 ) -> tuple[int, int, int]:
    """(items, rows, key shares) of :func:`attn_prefill`: an item is 256 rows
    of (token, query head of one KV head). The share count minimises waves x
    (key tiles per share + 2 to start), in units of a tile of 128 keys (2.1
    us), plus the merge's launch and its bytes (each share's fp32 row written
    and read; 1024 rows x 64 heads over 32768 keys at the power cap: 1152 us
    in one share, 1172 in four). With few rows the shares are short (17 rows x
    32 heads over 4113 keys: 70 us in one share, 18.4 in 11 of 3 tiles, 16.7
    in 17; 5 rows over 1005 keys: 14.2 us in 4 shares, 12.1 in 8). Of the counts
    with as many waves only the largest is tried, and of those with as many
    tiles a share the smallest."""
    per = 256 // (hq // hkv)
    rows = items = 0
    for n in q_lens:
        rows += n
        items += -(-n // per)
    ctas = max(1, items * hkv)
    tiles = -(-max(ctx_lens, default=0) // 128)
    best, best_cost = 1, -(-ctas // num_sms) * (tiles + 2)
    most = min(64, tiles)
    for waves in range(1, 5):
        sp = min(most, num_sms * waves // ctas)
        if sp < 2:
            continue
        share = -(-tiles // sp)
        sp = -(-tiles // share)
        cost = waves * (share + 2) + 2 + rows * hq * sp / 10000
        if cost < best_cost:
            best, best_cost = sp, cost
        if sp >= most:
            break
    return items, rows, best


def attn_prefill(q: torch.Tensor, k_cache: KV8Cache, v_cache: KV8Cache, block_table: torch.Tensor,
                 q_start: torch.Tensor, q_len: torch.Tensor, ctx_len: torch.Tensor, tiles: torch.Tensor | None,
                 hq: int, hkv: int, scale: float, out: torch.Tensor | None = None,
                 host_meta: tuple[list[int], list[int]] | None = None, bt_rows: torch.Tensor | None = None,
                 kv_splits: int | None = None, tile_rows: int | None = None) -> torch.Tensor:
    """Causal attention for chunks of new tokens whose K/V already sit in the
    8-bit cache; arguments as of :func:`infera_b200.ops.kernels.attn_prefill`.
    ``host_meta`` (q lengths, context lengths on the host; read back from the
    device without it) sizes the grid. The kernel makes its own work items of
    256 / group tokens, so ``tiles`` and ``tile_rows`` are not used. Up to 8
    query heads per KV head. ``out`` may be ``q`` itself. A row that sees no key (a context shorter than
    its chunk) is zero; rows of no sequence are left as they are. Bad lengths
    and table rows are treated as in :func:`attn_decode`. Nothing of a key
    that a row does not see reaches the row, a NaN neither."""
    _check_heads(hq, hkv, 8)
    n, T, dev = q_len.shape[0], q.shape[0], q.get_device()
    ldq = _check_rows("q", q, T, hq * HEAD_DIM, dev, 16)
    _check_i32("q_start", q_start, n, dev)
    _check_i32("q_len", q_len, n, dev)
    _check_i32("ctx_len", ctx_len, n, dev)
    _check_caches(k_cache, v_cache, hkv, dev)
    _check_table(block_table, bt_rows, n, dev)
    if host_meta is None:
        if dev >= 0 and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("attn_prefill over an 8-bit cache needs host_meta during capture")
        host_meta = (q_len.tolist(), ctx_len.tolist())
    q_lens, ctx_lens = host_meta
    if len(q_lens) != n or len(ctx_lens) != n:
        raise ValueError(f"host_meta is of {len(q_lens)} / {len(ctx_lens)} sequences, q_len of {n}")
    if n and min(q_lens) < 0:
        raise ValueError(f"a chunk of {min(q_lens)} tokens")
    if out is None:
        out = torch.empty(T, hq * HEAD_DIM, dtype=_BF16, device=q.device)
        ldo = hq * HEAD_DIM
    else:
        ldo = _check_rows("out", out, T, hq * HEAD_DIM, dev, 16, True)
    places = block_table.shape[1]
    if n and max(ctx_lens) > places * PAGE:
        raise ValueError(f"a context of {max(ctx_lens)} keys needs {-(-max(ctx_lens) // PAGE)} pages, block_table has "
                         f"room for {places}")
    items, rows, splits = prefill_plan(q_lens, ctx_lens, hq, hkv)
    if kv_splits is not None:
        splits = kv_splits
        if not 1 <= splits <= 65535:
            raise ValueError(f"kv_splits {splits}")
    if rows > T:
        raise ValueError(f"{rows} rows in the chunks, q has {T}")
    if rows == 0:
        return out
    if dev < 0:
        _attn_prefill_cpu(q, k_cache, v_cache, block_table, q_start, q_lens, ctx_lens, hq, hkv, scale, out, bt_rows)
        return out
    part = lse = None
    if splits > 1:
        # partials of this call, as in attn_decode
        m = T * hq * splits
        ws = torch.empty(m * (HEAD_DIM + 1), dtype=torch.float32, device=q.device)
        part = ws.data_ptr()
        lse = part + 4 * m * HEAD_DIM
    status, stream = _on(dev)
    rc = _native.kernels().ib_attn_prefill_kv8(q.data_ptr(), T, ldq, k_cache.q.data_ptr(), k_cache.sf.data_ptr(),
                                               v_cache.q.data_ptr(), v_cache.sf.data_ptr(), k_cache.slots,
                                               q_start.data_ptr(), q_len.data_ptr(), ctx_len.data_ptr(), n, items,
                                               rows, block_table.data_ptr(), K._ptr(bt_rows), block_table.shape[0],
                                               places, block_table.stride(0), hq, hkv, scale, splits, part, lse,
                                               out.data_ptr(), ldo, status, stream)
    _native.check(rc, "ib_attn_prefill_kv8")
    K._count(2 if splits > 1 else 1)
    return out


def _attn_prefill_cpu(q, k_cache, v_cache, block_table, q_start, q_lens, ctx_lens, hq, hkv, scale, out,
                      bt_rows) -> None:
    k, v, bt, ctx_lens = _cpu_view(k_cache, v_cache, block_table, bt_rows, ctx_lens)
    # a value that is NaN reaches the rows that see it, and not by a weight of zero
    nan = v.isnan()
    v = v.masked_fill(nan, 0.0)
    for i, (n, ctx, at) in enumerate(zip(q_lens, ctx_lens, q_start.tolist())):
        row = bt[i:i + 1]
        blind = min(n, max(0, n - ctx))  # the first rows of a chunk longer than its context
        out[at:at + blind, : hq * HEAD_DIM] = 0
        if n > blind:
            o, = K._ref_attention(q[at + blind:at + n, : hq * HEAD_DIM], k, v, row, [list(range(ctx - n + blind, ctx))],
                                  [ctx], hq, hkv, scale)
            slots = (row[0, : -(-ctx // PAGE), None] * PAGE + torch.arange(PAGE)).flatten()[:ctx]
            seen = nan[slots].cumsum(0)[ctx - n + blind:] > 0
            seen = seen.unflatten(-1, (hkv, 1, HEAD_DIM)).expand(-1, -1, hq // hkv, -1).flatten(1)
            out[at + blind:at + n, : hq * HEAD_DIM] = o.masked_fill(seen, float("nan")).to(q.dtype)
