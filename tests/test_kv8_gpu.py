"""The 8-bit paged KV cache on a GPU: appended codes against the CPU form bit
for bit, attention against plain attention in 64 bits, and the calls that
engines make of them (graphs, streams, padded rows, long caches)."""

import math

import pytest
import torch

from infera_b200.ops import kernels as K
from infera_b200.ops import kv8

pytestmark = pytest.mark.gpu

D = 128
DEV = "cuda"


def check_status(want=0):
    torch.cuda.synchronize()
    s = K.scratch()
    got = s.read_status()
    s.clear_status()
    assert got == want, f"kernel status {got}"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def same(a, b):
    return torch.equal(a.q.cpu().view(torch.uint8), b.q.cpu().view(torch.uint8)) and torch.equal(a.sf.cpu(), b.sf.cpu())


def random_cache(slots, hkv, seed=0, spread=3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(slots, hkv * D, generator=g, device=DEV) * 60
    sf = torch.randint(127 - spread, 128 + spread, (slots // 16, hkv), generator=g, device=DEV).to(torch.uint8)
    return kv8.KV8Cache(x.clamp(-448, 448).to(torch.float8_e4m3fn), sf)


def step(rows, hq, hkv, seed=0, max_pos=5000, pad=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(rows, (hq + 2 * hkv) * D + pad, generator=g) \
        * torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g))
    pos = torch.randint(0, max_pos, (rows,), generator=g).to(torch.int32)
    return qkv.to(torch.bfloat16), pos, K.rope_cos_sin(max_pos, D, 10000.0)


# ---------------------------------------------------------------- append


def chunk(start, n, pages, seed=0):
    """Slots of positions start .. start + n of a sequence on random pages of ``pages``."""
    g = torch.Generator().manual_seed(seed)
    own = torch.randperm(pages, generator=g)
    p = torch.arange(start, start + n)
    return (own[p // 16] * 16 + p % 16).tolist()


APPENDS = {
    "one row": ([37], 12),
    "one row, first of its page": ([48], 12),
    "a page and more": (list(range(5, 40)), 12),
    "out of order": ([70, 33, 66, 35, 64, 34, 7, 65], 12),
    "not stored": ([-1, 20, -1, 21, -1], 12),
    "same slot twice": ([20, 21, 20, 99, 20], 12),
    "one slot only": ([20] * 33, 12),
    "all skipped": ([-1, -1], 12),
    "64 decoding rows": ([16 * i + (7 * i) % 16 for i in range(64)], 64),
    "mixed": ([16 * i + 3 for i in range(48)] + [s + 16 * 48 for s in chunk(13, 223, 15)], 64),
    "prompt": (chunk(0, 1040, 65, 1), 65),
    "long step": (chunk(9, 2500, 157, 2), 157),
    "long step, mixed order": (torch.randperm(1500, generator=torch.Generator().manual_seed(4)).tolist(), 94),
}


@pytest.mark.parametrize("name", APPENDS)
@pytest.mark.parametrize("hq,hkv", [(4, 2), (1, 1), (7, 7), (32, 8)])
def test_append_matches_cpu(name, hq, hkv):
    """Every product and sum of the rotation is rounded on its own on both sides: the same bits."""
    slots, pages = APPENDS[name]
    slots = torch.tensor(slots, dtype=torch.int32)
    qkv, pos, cs = step(len(slots), hq, hkv, seed=len(name), pad=24)
    kc, vc = random_cache(pages * 16, hkv, 1), random_cache(pages * 16, hkv, 2)
    k_cpu, v_cpu = kc.to("cpu"), vc.to("cpu")
    q_cpu = kv8.rope_kvwrite(qkv, pos, slots, cs, hq, hkv, D, k_cpu, v_cpu, q_out=torch.zeros(len(slots), hq * D + 8,
                                                                                            dtype=torch.bfloat16))
    dev = [t.to(DEV) for t in (qkv, pos, slots, cs)]
    out = torch.zeros(len(slots), hq * D + 8, dtype=torch.bfloat16, device=DEV)
    for _ in range(2):  # the second call changes nothing
        kv8.rope_kvwrite(*dev, hq, hkv, D, kc, vc, q_out=out)
        check_status()
        assert torch.equal(out.cpu(), q_cpu)
        assert same(kc, k_cpu) and same(vc, v_cpu)
    assert torch.equal(dev[0].cpu(), qkv)
    K.rope_kvwrite(*dev, hq, hkv, D, kc, vc)  # in place
    check_status()
    assert torch.equal(dev[0][:, :hq * D].cpu(), q_cpu[:, :hq * D])
    assert torch.equal(dev[0][:, hq * D:].cpu(), qkv[:, hq * D:]) and same(kc, k_cpu)


def test_append_special_values():
    kc, vc = kv8.alloc(32, 1, device=DEV), kv8.alloc(32, 1, device=DEV)
    kc.q.view(torch.uint8).fill_(0x7F)  # a recycled page may hold anything
    qkv = torch.zeros(3, 3 * D, dtype=torch.bfloat16)
    qkv[1, 2 * D], qkv[1, 2 * D + 1] = float("inf"), 2.0
    qkv[2, 2 * D + 5], qkv[2, D + 70] = float("nan"), float("-inf")
    slots, pos = torch.tensor([0, 1, 16], dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    cs = K.rope_cos_sin(4, D, 1e4)
    k_cpu, v_cpu = kc.to("cpu"), vc.to("cpu")
    kv8.rope_kvwrite(qkv, pos, slots, cs, 1, 1, D, k_cpu, v_cpu)
    kv8.rope_kvwrite(qkv.to(DEV), pos.to(DEV), slots.to(DEV), cs.to(DEV), 1, 1, D, kc, vc)
    check_status()
    for a, b in ((kc, k_cpu), (vc, v_cpu)):
        assert torch.equal(a.sf.cpu(), b.sf)
        x, y = a.dequant().cpu(), b.dequant()
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
    # a later row of ordinary size in the page of zeros: its scale grows from the smallest
    qkv[:, D:] = 1.0
    kv8.rope_kvwrite(qkv[:1].to(DEV), pos[:1].to(DEV), i32([5]), cs.to(DEV), 1, 1, D, kc, vc)
    check_status()
    assert float(kc.dequant()[5, 0]) == 1.0 and float(vc.dequant()[5, 0]) == 1.0


@pytest.mark.parametrize("hq,hkv", [(8, 4), (8, 8), (7, 7)])
def test_append_long_step_with_everything(hq, hkv):
    """Whole pages of a prompt with infinities, NaN, rows without a slot, slots named twice and bad positions among them."""
    n, pages = 700, 50
    qkv, pos, cs = step(n, hq, hkv, seed=5, max_pos=900)
    g = torch.Generator().manual_seed(6)
    slots = torch.tensor(chunk(0, n, pages, 3), dtype=torch.int32)
    pick = torch.randperm(n, generator=g)
    slots[pick[:20]], slots[pick[20:40]] = -1, slots[pick[40:60]]
    pos[pick[60:70]], pos[pick[70:80]] = 900, -5
    kv = qkv[:, hq * D:]
    for i, x in enumerate((float("inf"), float("-inf"), float("nan"))):
        rows = pick[100 + 30 * i:130 + 30 * i]
        kv[rows, torch.randint(0, 2 * hkv * D, (30,), generator=g)] = x
    kc, vc = random_cache(pages * 16, hkv, 1), random_cache(pages * 16, hkv, 2)
    k_cpu, v_cpu = kc.to("cpu"), vc.to("cpu")
    q_cpu = kv8.rope_kvwrite(qkv, pos, slots, cs, hq, hkv, D, k_cpu, v_cpu, q_out=torch.zeros(n, hq * D).bfloat16())
    q = torch.zeros(n, hq * D, dtype=torch.bfloat16, device=DEV)
    kv8.rope_kvwrite(*[t.to(DEV) for t in (qkv, pos, slots, cs)], hq, hkv, D, kc, vc, q_out=q)
    torch.cuda.synchronize()
    assert K.scratch().read_status_detail()["what"] == 1  # a position, whichever came first
    K.scratch().clear_status()
    assert torch.equal(q.cpu(), q_cpu)
    for a, b in ((kc, k_cpu), (vc, v_cpu)):
        x, y = a.q.cpu().float(), b.q.float()
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
        assert torch.equal(a.sf.cpu(), b.sf)


@pytest.mark.parametrize("what,pos,slot,detail", [("position", 50, 3, 1), ("position", -1, 3, 1), ("slot", 5, 64, 2)])
def test_append_bad_index_is_skipped(what, pos, slot, detail):
    qkv, _, cs = step(3, 4, 2, max_pos=50)
    kc, vc = random_cache(64, 2, 1), random_cache(64, 2, 2)
    k_cpu, v_cpu = kc.to("cpu"), vc.to("cpu")
    p, s = torch.tensor([1, pos, 2], dtype=torch.int32), torch.tensor([1, slot, 40], dtype=torch.int32)
    kv8.rope_kvwrite(qkv.to(DEV), p.to(DEV), s.to(DEV), cs.to(DEV), 4, 2, D, kc, vc)
    torch.cuda.synchronize()
    assert K.scratch().read_status_detail() == {"code": 7, "what": detail, "where": 1,
                                                "value": pos if what == "position" else slot}
    K.scratch().clear_status()
    kv8.rope_kvwrite(qkv.clone(), p, s, cs, 4, 2, D, k_cpu, v_cpu)  # the CPU form skips the row too
    assert same(kc, k_cpu) and same(vc, v_cpu)


# ---------------------------------------------------------------- attention


def plain(q, kc, vc, pages, first, hq, hkv, scale):
    """64-bit attention of rows q [n, hq*128]; row i sees the first ``first + i`` keys of ``pages``. Also what the
    errors of an output element are measured against: ``size`` = sum of p|v|, and ``unit`` = the largest p times the sum
    of |code| at the largest V scale of the head."""
    n, total = q.shape[0], first + q.shape[0] - 1
    pages = pages[: -(-total // 16)].long()

    def rows(c):
        codes = c.q.view(torch.uint8).view(-1, 16, hkv, D)[pages].view(torch.float8_e4m3fn).double()
        s = torch.pow(2.0, c.sf[pages].double().clamp_min(1) - 127)[:, None, :, None]
        return (codes * s).view(-1, hkv, D)[:total], codes.view(-1, hkv, D)[:total].abs().sum(0) * s.amax(0)[0]

    (k, _), (v, most) = rows(kc), rows(vc)
    G = hq // hkv
    qg = q[:, : hq * D].double().view(n, hkv, G, D)
    s = torch.einsum("nkgd,skd->kgns", qg, k) * scale
    hidden = torch.arange(total, device=q.device)[None] >= torch.arange(first, first + n, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
    out = torch.einsum("kgns,skd->nkgd", p, v)
    size = torch.einsum("kgns,skd->nkgd", p, v.abs())
    unit = torch.einsum("kgn,kd->nkgd", p.amax(-1), most)
    return [t.reshape(n, -1) for t in (out, size, unit)]


# Single tokens. A weight is rounded to f16 and that split into three e4m3 digits: off by at most 2^-12 of itself or
# 2^-20 where a weight at the running maximum is 2^6, so 2^-26 of it, times the code at the largest V scale. That
# maximum may lag behind the row's largest weight, never be above it, so p_max >= 2^6 / (sum of weights): the second
# part is at most 2^-26 of ``unit``. Scores are 32-bit sums of exact products: 2^-20 of sum |q k| (at most 2^7 here) is
# 2^-13 of a weight, its exponential and the sums some 2^-20 more: 2^-12 + 2^-13 + 2^-20 < 2^-11 of ``size``.
TOKEN = (2 ** -11, 2 ** -26)
# Prompts. Weights are rounded to f16, where one at the running maximum is 2^6: off by at most 2^-12 of itself or 2^-25,
# 2^-31 of it; the query's digits are off by 2^-18 of its row's largest element, so the score of one key by at most that
# times sum |k| max|q|: with random elements some 4 times sum |q k| (2^7), 2^-9; the rest as above. Scores here are
# below 2^5, and sums of |q k| below 2^6: 2^-12 + 2^-10 + 2^-13 < 2^-9 of ``size``.
PROMPT = (2 ** -9, 2 ** -31)


def assert_close(got, want, tol):
    """Half a step of bf16 on the output, and ``tol`` of the terms."""
    out, size, unit = want
    assert got.shape == out.shape
    err = (got.double() - out).abs()
    bad = ~(err <= out.abs() * 2 ** -8 + size * tol[0] + unit * tol[1])
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}, worst {float((err / (size + 1e-30)).max()):.2e} of the terms"


def decode_case(lens, hq, hkv, seed, runs=False, spread=3, qsize=1 / 60):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // 16) for n in lens]
    pool = sum(need) + 5
    order = torch.arange(pool) if runs else torch.randperm(pool, generator=g)
    bt = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32)
    at = 2
    for i, n in enumerate(need):
        bt[i, :n] = order[at:at + n]
        at += n
    kc, vc = random_cache(pool * 16, hkv, seed, spread), random_cache(pool * 16, hkv, seed + 1, spread)
    q = (torch.randn(len(lens), hq * D, generator=g) * qsize).to(torch.bfloat16).to(DEV)
    return q, kc, vc, bt.to(DEV), i32(lens)


def poison(kc, vc, bt, lens):
    """NaN codes in every slot that no sequence has: behind its last key, and in the pool's other pages."""
    live = torch.zeros(kc.q.shape[0], dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        live[(bt[b].long()[:, None] * 16 + torch.arange(16, device=DEV)).flatten()[:n]] = True
    for c in (kc, vc):
        c.q.view(torch.uint8)[~live] = 0x7F


def check_decode(lens, hq, hkv, y, q, kc, vc, bt, scale):
    for b, n in enumerate(lens):
        if n <= 0:
            assert not y[b].any()
            continue
        assert_close(y[b:b + 1, : hq * D], plain(q[b:b + 1], kc, vc, bt[b], n, hq, hkv, scale), TOKEN)


LENS = {
    "one key": [1], "short": [15, 16, 17, 31], "tile borders": [127, 128, 129, 255, 256, 257], "empty rows": [0, 5, 0, 300, 0],
    "ragged": [1, 700, 33, 2049, 128, 1100], "long": [9000], "two long": [4097, 5000],
}


@pytest.mark.parametrize("name", LENS)
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("runs", [False, True])
def test_decode(name, G, runs):
    lens, hkv = LENS[name], 2
    hq = hkv * G
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=G, runs=runs)
    scale = 1 / math.sqrt(D)
    for splits, tps in {kv8.decode_plan(len(lens), hkv, max(lens)), (1, -(-max(lens) // 128)), (3, -(-max(lens) // 384)),
                        (1, 0), (2, 0)}:
        y = K.attn_decode(q, kc, vc, bt, sl, hq, hkv, scale, splits=splits, tiles_per_split=tps)
        check_status()
        check_decode(lens, hq, hkv, y, q, kc, vc, bt, scale)


@pytest.mark.parametrize("hq,hkv", [(8, 8), (8, 1), (64, 8), (7, 7)])
def test_decode_heads(hq, hkv):
    lens = [100, 1030]
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=hq)
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 0.09, *kv8.decode_plan(2, hkv, 1030)[:1], tiles_per_split=0)
    check_status()
    check_decode(lens, hq, hkv, y, q, kc, vc, bt, 0.09)


@pytest.mark.parametrize("qsize", [1e-4, 1 / 10, 1.0])
@pytest.mark.parametrize("spread", [1, 30])
def test_decode_flat_and_peaked(qsize, spread):
    """All weights alike, and one key that has all the weight; scales that differ by 2^60 (the accumulators are
    rescaled for both the maximum and the V exponent). Scores of peaked rows reach 2^9 (2^39 with the scales): only
    their largest keys count, and these are told apart by far more than their rounding; where K's scales differ that
    much the row's largest score decides alone."""
    lens, hq, hkv = [1500, 40], 8, 2
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=3, spread=spread, qsize=qsize)
    if spread == 30:
        kc = random_cache(kc.q.shape[0], hkv, 9, 1)  # K's scales alike: the scores stay distinct
    if qsize == 1.0:
        q = q / 8  # scores of about 2^5
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 1 / math.sqrt(D), splits=2, tiles_per_split=6)
    check_status()
    check_decode(lens, hq, hkv, y, q, kc, vc, bt, 1 / math.sqrt(D))


def test_decode_small_weights_add_up():
    """One key with half of the weight and no value, 8000 others that share the rest: each is 2^-14 of it."""
    n, hq, hkv = 8001, 4, 1
    q, kc, vc, bt, sl = decode_case([n], hq, hkv, seed=5, runs=True)
    page = int(bt[0, 0])
    k = kc.q.view(torch.uint8).view(-1, 16, D)
    k.zero_()
    kc.sf.fill_(127)
    q.zero_()
    q.view(1, hq, D)[:, :, 0] = 1.0
    k[page, 0, 0] = torch.tensor([9.0]).to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)  # e^9 = 8103
    vc.q.view(torch.uint8).view(-1, 16, D)[page, 0] = 0
    vc.sf.fill_(127)
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 1.0, splits=1, tiles_per_split=63)
    check_status()
    check_decode([n], hq, hkv, y, q, kc, vc, bt, 1.0)


def test_decode_stale_nan_behind_the_sequence():
    """NaN codes in the slots behind a sequence's last key, and in the pool's other pages, do not reach it."""
    lens, hq, hkv = [1, 100, 129, 1000], 8, 2
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=8)
    poison(kc, vc, bt, lens)
    bt = torch.cat([bt, torch.full((4, 8), 12345678, dtype=torch.int32, device=DEV)], 1)  # entries nothing reads
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 0.1, splits=2, tiles_per_split=4)
    check_status()
    check_decode(lens, hq, hkv, y, q, kc, vc, bt, 0.1)
    # one in a key that counts reaches that sequence's heads of its KV head, and no other
    first = int(bt[2, 0]) * 16
    kc.q.view(torch.uint8)[first, 5] = 0x7F
    y2 = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 0.1, splits=2, tiles_per_split=4)
    check_status()
    assert y2[2, : 4 * D].isnan().all() and not y2[2, 4 * D:].isnan().any()
    assert torch.equal(y2[[0, 1, 3]], y[[0, 1, 3]])


def test_decode_strides_rows_and_tables():
    """Rows inside wider buffers, more rows than sequences, table rows by index, rows behind the last left alone."""
    lens, hq, hkv = [77, 300, 1000], 8, 2
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=9)
    wide = torch.full((5, (hq + 4) * D + 2), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[:3, : hq * D] = q
    big = torch.zeros(9, bt.shape[1] + 3, dtype=torch.int32, device=DEV)
    rows = i32([8, 0, 4])
    big[rows.long(), : bt.shape[1]] = bt
    out = torch.full((5, hq * D + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    got = kv8.attn_decode(wide, kc, vc, big[:, : bt.shape[1] + 1], sl, hq, hkv, 0.1, splits=2, tiles_per_split=4,
                          out=out, bt_rows=rows)
    check_status()
    assert got is out and bool((out[3:] == 3).all()) and bool((out[:, hq * D:] == 3).all())
    check_decode(lens, hq, hkv, out, q, kc, vc, bt, 0.1)
    # the result does not depend on what stands beside a sequence
    alone = kv8.attn_decode(q[1:2], kc, vc, bt[1:2], sl[1:2], hq, hkv, 0.1, splits=2, tiles_per_split=4)
    assert torch.equal(alone[0], out[1, : hq * D])


def test_decode_bad_table():
    """A page id outside the cache reads as zeros; a length beyond the table's places is cut there and reported."""
    q, kc, vc, bt, sl = decode_case([40], 4, 2, seed=10)
    y0 = kv8.attn_decode(q, kc, vc, bt, i32([16 * bt.shape[1]]), 4, 2, 0.1)
    check_status()
    y = kv8.attn_decode(q, kc, vc, bt, i32([100000]), 4, 2, 0.1, splits=1, tiles_per_split=1000)
    torch.cuda.synchronize()
    assert K.scratch().read_status_detail() == {"code": 7, "what": 1, "where": 0, "value": 100000}
    K.scratch().clear_status()
    assert torch.equal(y, y0)
    bt[0, 1] = kc.sf.shape[0] + 3
    y = kv8.attn_decode(q, kc, vc, bt, sl, 4, 2, 0.1)
    torch.cuda.synchronize()
    K.scratch().clear_status()
    assert bool(y.isfinite().all())


def detail():
    torch.cuda.synchronize()
    d = K.scratch().read_status_detail()
    K.scratch().clear_status()
    return d


def test_bad_table_rows_and_keys_that_no_split_takes():
    """A row index outside the table gives zeros, keys behind the last split are left out; both are reported."""
    lens = [300, 200]
    q, kc, vc, bt, sl = decode_case(lens, 8, 2, seed=12)
    good = kv8.attn_decode(q, kc, vc, bt, sl, 8, 2, 0.1, bt_rows=i32([0, 1]))
    check_status()
    for bad in (2, -1):
        y = kv8.attn_decode(q, kc, vc, bt, sl, 8, 2, 0.1, splits=2, bt_rows=i32([0, bad]))
        assert detail() == {"code": 7, "what": 4, "where": 1, "value": bad}
        check_decode([300, 0], 8, 2, y, q, kc, vc, bt, 0.1)
        y = kv8.attn_prefill(q, kc, vc, bt, i32([0, 1]), i32([1, 1]), sl, None, 8, 2, 0.1, bt_rows=i32([0, bad]),
                             host_meta=([1, 1], lens), kv_splits=1)
        assert detail() == {"code": 7, "what": 4, "where": 1, "value": bad}
        assert not y[1].any() and bool(((y[0].float() - good[0].float()).abs() <= 2 ** -7 * good[0].abs() + 1e-2).all())
    y = kv8.attn_decode(q, kc, vc, bt, sl, 8, 2, 0.1, splits=1, tiles_per_split=2)
    assert detail() == {"code": 6, "what": 5, "where": 0, "value": 300}
    check_decode([256, 200], 8, 2, y, q, kc, vc, bt, 0.1)


def test_one_row_in_a_buffer_of_any_pitch():
    q, kc, vc, bt, sl = decode_case([70], 8, 2, seed=13)
    want = kv8.attn_decode(q, kc, vc, bt, sl, 8, 2, 0.1)
    wide = torch.zeros(1, 8 * D + 5, dtype=torch.bfloat16, device=DEV)
    wide[:, : 8 * D] = q
    out = torch.zeros(1, 8 * D + 3, dtype=torch.bfloat16, device=DEV)
    kv8.attn_decode(wide, kc, vc, bt, sl, 8, 2, 0.1, out=out)
    check_status()
    assert torch.equal(out[:, : 8 * D], want)
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    a = kv8.attn_prefill(q, kc, vc, bt, one - 1, one, sl, None, 8, 2, 0.1, host_meta=([1], [70]))
    b = kv8.attn_prefill(wide, kc, vc, bt, one - 1, one, sl, None, 8, 2, 0.1, host_meta=([1], [70]), out=out)
    check_status()
    assert torch.equal(a, b[:, : 8 * D])


def test_scale_zero_counts_as_one():
    """Codes under a scale exponent of 0 and of 1 are the same values, in attention and when the page's scale grows."""
    q, kc, vc, bt, sl = decode_case([20], 4, 2, seed=14)
    q = q * 2.0 ** 60
    caches = []
    for e in (0, 1):
        k, v = kv8.KV8Cache(kc.q.clone(), torch.full_like(kc.sf, e)), kv8.KV8Cache(vc.q.clone(), torch.full_like(vc.sf, e))
        caches.append((k, v))
    a, b = [kv8.attn_decode(q, k, v, bt, sl, 4, 2, 2.0 ** 60) for k, v in caches]
    assert torch.equal(a, b)
    qkv = torch.full((1, 8 * D), 2.0 ** -115, dtype=torch.bfloat16, device=DEV)
    slot = (bt[0, 1:2] * 16 + 9).contiguous()
    for k, v in caches:
        kv8.rope_kvwrite(qkv, i32([0]), slot, K.rope_cos_sin(2, D, 1e4, device=DEV), 4, 2, D, k, v)
    check_status()
    page = int(bt[0, 1])
    for x, y in zip(*caches):
        here = slice(page * 16, page * 16 + 16)
        assert torch.equal(x.q[here].view(torch.uint8), y.q[here].view(torch.uint8))
        assert torch.equal(x.sf[page], y.sf[page]) and int(x.sf[page, 0]) > 1


@pytest.mark.parametrize("splits", [1, 3])
def test_prefill_rows_that_see_nothing(splits):
    """A context shorter than its chunk: the chunk's first rows see no key and are zero; a chunk over no context is."""
    hq, hkv = 8, 2
    q, kc, vc, bt, _ = decode_case([300, 300, 300], hq, hkv, seed=15)
    ql, ctx = [40, 200, 5], [10, 129, 0]
    g = torch.Generator().manual_seed(1)
    q = (torch.randn(sum(ql) + 3, hq * D, generator=g) / 60).to(torch.bfloat16).to(DEV)
    out = torch.full((sum(ql) + 3, hq * D), 3.0, dtype=torch.bfloat16, device=DEV)
    kv8.attn_prefill(q, kc, vc, bt, i32([0, 40, 240]), i32(ql), i32(ctx), None, hq, hkv, 0.1, host_meta=(ql, ctx),
                     out=out, kv_splits=splits)
    check_status()
    assert not out[:30].any() and not out[40:111].any() and not out[240:245].any() and bool((out[245:] == 3).all())
    assert_close(out[30:40], plain(q[30:40], kc, vc, bt[0], 1, hq, hkv, 0.1), PROMPT)
    assert_close(out[111:240], plain(q[111:240], kc, vc, bt[1], 1, hq, hkv, 0.1), PROMPT)


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("hq,hkv", [(2, 1), (9, 3), (10, 2), (12, 2), (7, 1), (16, 2)])
def test_prefill_heads(hq, hkv, splits):
    """Items whose 256 rows end inside a token's heads, and query tiles that part them."""
    ql, ctx = [100, 1, 37], [500, 129, 37]
    g = torch.Generator().manual_seed(hq)
    _, kc, vc, bt, sl = decode_case(ctx, hq, hkv, seed=hq)
    poison(kc, vc, bt, ctx)
    q = (torch.randn(sum(ql), hq * D, generator=g) / 60).to(torch.bfloat16).to(DEV)
    y = kv8.attn_prefill(q, kc, vc, bt, i32([0, 100, 101]), i32(ql), sl, None, hq, hkv, 0.1, host_meta=(ql, ctx),
                         kv_splits=splits)
    check_status()
    at = 0
    for b, n in enumerate(ql):
        assert_close(y[at:at + n], plain(q[at:at + n], kc, vc, bt[b], ctx[b] - n + 1, hq, hkv, 0.1), PROMPT)
        at += n


@pytest.mark.parametrize("splits", [1, 2])
def test_prefill_many_sequences(splits):
    """More sequences than a warp has lanes, some without a token in this step."""
    n, hq, hkv = 70, 8, 2
    ql, ctx = [(7 * i) % 11 for i in range(n)], [(7 * i) % 11 + (53 * i) % 300 for i in range(n)]
    g = torch.Generator().manual_seed(4)
    _, kc, vc, bt, sl = decode_case(ctx, hq, hkv, seed=17)
    start = [sum(ql[:i]) + 3 for i in range(n)]
    q = (torch.randn(sum(ql) + 5, hq * D, generator=g) / 60).to(torch.bfloat16).to(DEV)
    out = torch.full_like(q, 3.0)
    kv8.attn_prefill(q, kc, vc, bt, i32(start), i32(ql), sl, None, hq, hkv, 0.1, host_meta=(ql, ctx), out=out,
                     kv_splits=splits)
    check_status()
    assert bool((out[:3] == 3).all()) and bool((out[-2:] == 3).all())
    for b in range(n):
        if ql[b]:
            rows = slice(start[b], start[b] + ql[b])
            assert_close(out[rows], plain(q[rows], kc, vc, bt[b], ctx[b] - ql[b] + 1, hq, hkv, 0.1), PROMPT)


def test_append_and_prefill_in_a_graph():
    """A step of an append and a prompt's attention, captured once and replayed with other rows, on another stream."""
    n, ctx, hq, hkv = 60, 700, 8, 2
    _, kc, vc, bt, sl = decode_case([ctx], hq, hkv, seed=18)
    slots = i32([int(bt[0, p // 16]) * 16 + p % 16 for p in range(ctx - n, ctx)])
    steps = [step(n, hq, hkv, seed=s, max_pos=900) for s in (1, 2)]
    pos, cs = torch.arange(ctx - n, ctx, dtype=torch.int32, device=DEV), steps[0][2].to(DEV)
    qkv = torch.empty_like(steps[0][0], device=DEV)
    args = (i32([0]), i32([n]), sl, None, hq, hkv, 0.05)

    def run(k, v):
        q = torch.empty(n, hq * D, dtype=torch.bfloat16, device=DEV)
        kv8.rope_kvwrite(qkv, pos, slots, cs, hq, hkv, D, k, v, q_out=q)
        return kv8.attn_prefill(q, k, v, bt, *args, host_meta=([n], [ctx]), kv_splits=3)

    caches = [kv8.KV8Cache(c.q.clone(), c.sf.clone()) for c in (kc, vc)]
    want = []
    for x in steps:
        qkv.copy_(x[0])
        want.append(run(*caches))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(kc, vc)
    side = torch.cuda.Stream()
    for x, w in zip(steps, want):
        with torch.cuda.stream(side):
            qkv.copy_(x[0].to(DEV))
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w)
    check_status()
    assert same(kc, caches[0].to("cpu")) and same(vc, caches[1].to("cpu"))


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("G", [1, 4, 8])
def test_prefill_nothing_unseen_reaches_a_row(G, splits):
    """NaN values and keys, and values of 2^90, behind a row's last key: the row is what it is without them, and the rows
    that do see them have them, dim by dim."""
    hkv, n, ctx, scale = 2, 300, 811, 0.1  # rows see 512 .. 811 keys
    hq = hkv * G
    q, kc, vc, bt, _ = decode_case([ctx], hq, hkv, seed=16)
    g = torch.Generator().manual_seed(2)
    q = (torch.randn(n, hq * D, generator=g) / 60).to(torch.bfloat16).to(DEV)

    def run():
        return kv8.attn_prefill(q, kc, vc, bt, i32([0]), i32([n]), i32([ctx]), None, hq, hkv, scale,
                                host_meta=([n], [ctx]), kv_splits=splits)

    clean = run()
    check_status()
    assert_close(clean, plain(q, kc, vc, bt[0], ctx - n + 1, hq, hkv, scale), PROMPT)
    slot = lambda k: int(bt[0, k // 16]) * 16 + k % 16  # noqa: E731
    # (key, column of the values): seen by all, by the chunk's middle and last rows, the last key; both heads
    holes = [(5, 7), (530, 3), (531, D + 64), (639, 127), (640, D + 127), (700, 0), (ctx - 1, D + 1)]
    held = vc.q.clone()
    for k, col in holes:
        vc.q.view(torch.uint8)[slot(k), col] = 0x7F if col % 2 else 0xFF
    y = run()
    check_status()
    want = torch.zeros(n, hkv, G, D, dtype=torch.bool, device=DEV)
    for k, col in holes:
        want[max(0, k - (ctx - n)):, col // D, :, col % D] = True
    want = want.view(n, -1)
    assert torch.equal(y.isnan(), want) and bool((y == clean)[~want].view(-1).all())
    vc.q.copy_(held)
    # a key that is NaN: whole rows, from the first that sees it
    kc.q.view(torch.uint8)[slot(650), D + 9] = 0x7F
    y = run()
    check_status()
    at = 650 - (ctx - n)
    assert torch.equal(y[:at], clean[:at]) and bool(y[at:, G * D:].isnan().all())
    assert torch.equal(y[at:, : G * D], clean[at:, : G * D])
    kc.q.view(torch.uint8)[slot(650), D + 9] = 0
    # pages of far larger values
    kc.q.view(torch.uint8)[slot(650)] = 0
    vc.sf[bt[0, 704 // 16:].long(), 0] += 90
    y = run()
    check_status()
    for i in (0, 1, 100, 127, 128, 190, 191, 192, 200, 255, 256, n - 1):
        assert_close(y[i:i + 1], plain(q[i:i + 1], kc, vc, bt[0], ctx - n + 1 + i, hq, hkv, scale), PROMPT)


def test_decode_and_append_in_a_far_page():
    """Codes more than 2^31 bytes into the cache."""
    hkv, hq, pages = 8, 16, (1 << 31) // (16 * 8 * D) + 40
    kc, vc = kv8.alloc(pages * 16, hkv, device=DEV), kv8.alloc(pages * 16, hkv, device=DEV)
    assert kc.q.numel() > 1 << 31
    n = 200
    own = torch.arange(pages - 13, pages, dtype=torch.int32)
    slots = (own.long()[:, None] * 16 + torch.arange(16)).flatten()[:n].to(torch.int32)
    qkv, pos, cs = step(n, hq, hkv, seed=3)
    qkv = qkv / 4
    kv8.rope_kvwrite(qkv.to(DEV), pos.to(DEV), slots.to(DEV), cs.to(DEV), hq, hkv, D, kc, vc)
    check_status()
    ks, vs = kv8.alloc(13 * 16, hkv, device="cpu"), kv8.alloc(13 * 16, hkv, device="cpu")
    kv8.rope_kvwrite(qkv, pos, torch.arange(n, dtype=torch.int32), cs, hq, hkv, D, ks, vs)
    assert torch.equal(kc.q[-13 * 16:].view(torch.uint8).cpu(), ks.q.view(torch.uint8))
    assert torch.equal(vc.sf[-13:].cpu(), vs.sf) and not kc.sf[:-13].any()
    q = qkv[:1].to(DEV)
    y = kv8.attn_decode(q, kc, vc, own.view(1, -1).to(DEV), i32([n]), hq, hkv, 0.05)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    yp = kv8.attn_prefill(q, kc, vc, own.view(1, -1).to(DEV), one, one + 1, i32([n]), i32([[0, 0]]), hq, hkv, 0.05,
                          host_meta=([1], [n]))
    check_status()
    near = [c.to(DEV) for c in (ks, vs)]
    want = plain(q, *near, torch.arange(13, device=DEV), n, hq, hkv, 0.05)
    assert_close(y, want, TOKEN)
    assert_close(yp, want, PROMPT)


def test_decode_in_graphs_and_on_two_streams():
    """Two captured graphs replayed at once on two streams, beside eager calls, share no workspace."""
    hq, hkv = 32, 8
    cases = [decode_case([3000, 50, 2000], hq, hkv, seed=s) for s in (1, 2)]
    calls = [lambda c=c: kv8.attn_decode(*c, hq, hkv, 0.1, splits=6, tiles_per_split=4) for c in cases]
    want = [f().clone() for f in calls]
    graphs, outs = [], []
    for f in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = calls[0]()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
    check_status()
    del graphs


# ---------------------------------------------------------------- prompts

CHUNKS = {
    "one row": ([1], [1]), "whole prompt": ([300], [300]), "chunk": ([130], [1000]), "one row of many": ([1], [2000]),
    "ragged": ([17, 256, 1, 300, 5], [17, 700, 90, 301, 1500]), "an empty one": ([20, 0, 40], [50, 0, 40]),
    "shares of a tile": ([3], [8100]),
}


@pytest.mark.parametrize("name", CHUNKS)
@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 8), (32, 8)])
@pytest.mark.parametrize("rows", [128, 256])
def test_prefill(name, hq, hkv, rows):
    ql, ctx = CHUNKS[name]
    g = torch.Generator().manual_seed(len(name))
    _, kc, vc, bt, sl = decode_case(ctx, hq, hkv, seed=hq)
    poison(kc, vc, bt, ctx)
    T = sum(ql)
    q = (torch.randn(T, (hq + 2) * D, generator=g) / 60).to(torch.bfloat16).to(DEV)
    start = [sum(ql[:i]) for i in range(len(ql))]
    tiles = i32(K.prefill_tiles(ql, rows))
    args = (q, kc, vc, bt, i32(start), i32(ql), sl, tiles, hq, hkv, 0.1)
    y = K.attn_prefill(*args, host_meta=(ql, ctx), tile_rows=rows)
    check_status()
    for b in range(len(ql)):
        if ql[b]:
            want = plain(q[start[b]:start[b] + ql[b]], kc, vc, bt[b], ctx[b] - ql[b] + 1, hq, hkv, 0.1)
            assert_close(y[start[b]:start[b] + ql[b]], want, PROMPT)
    again = kv8.attn_prefill(*args, tile_rows=rows, out=torch.empty_like(y))  # lengths read from the device
    check_status()
    if len(ql) == 1:
        return  # (without host lengths the key shares of a tile may differ)
    out = torch.full((T + 2, hq * D + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    kv8.attn_prefill(*args, host_meta=(ql, ctx), tile_rows=rows, out=out)
    check_status()
    assert torch.equal(out[:T, : hq * D], y) and bool((out[T:] == 3).all()) and bool((out[:, hq * D:] == 3).all())
    assert again.shape == y.shape


# ---------------------------------------------------------------- together


def test_prompt_then_tokens():
    """As an engine runs them: a prompt in two chunks, then single tokens, each step appended and attended to. Every
    row's output is attention over what the cache holds after its step."""
    hq, hkv, scale = 16, 2, 1 / math.sqrt(D)
    pages = torch.randperm(30, generator=torch.Generator().manual_seed(1))[:20].to(torch.int32)
    bt = pages.view(1, -1).to(DEV)
    kc, vc = random_cache(30 * 16, hkv, 5), random_cache(30 * 16, hkv, 6)  # recycled pages
    cs = K.rope_cos_sin(400, D, 10000.0, device=DEV)
    done = 0
    for n in (200, 75, 1, 1, 1, 1, 1):
        qkv, _, _ = step(n, hq, hkv, seed=done)
        qkv = (qkv / 4).to(DEV)
        pos = torch.arange(done, done + n, dtype=torch.int32)
        slots = (pages.long()[pos.long() // 16] * 16 + pos % 16).to(torch.int32).to(DEV)
        K.rope_kvwrite(qkv, pos.to(DEV), slots, cs, hq, hkv, D, kc, vc)
        done += n
        if n > 1:
            y = K.attn_prefill(qkv, kc, vc, bt, i32([0]), i32([n]), i32([done]), i32(K.prefill_tiles([n])), hq, hkv,
                               scale, host_meta=([n], [done]))
        else:
            splits, tps = kv8.decode_plan(1, hkv, done)
            y = K.attn_decode(qkv, kc, vc, bt, i32([done]), hq, hkv, scale, splits=splits, tiles_per_split=tps)
        check_status()
        assert_close(y, plain(qkv, kc, vc, bt[0], done - n + 1, hq, hkv, scale), PROMPT if n > 1 else TOKEN)


def test_refusals_on_the_gpu():
    q, kc, vc, bt, sl = decode_case([40], 4, 2, seed=10)
    odd = torch.zeros(4 * D + 2, dtype=torch.bfloat16, device=DEV)[1:4 * D + 1].view(1, -1)
    with pytest.raises(ValueError, match="multiples of 4 bytes"):
        kv8.attn_decode(odd, kc, vc, bt, sl, 4, 2, 0.1)
    with pytest.raises(ValueError, match="is on cpu"):
        kv8.attn_decode(q, kc, vc, bt.cpu(), sl, 4, 2, 0.1)
    qkv = torch.zeros(2, 8 * D + 4, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="multiples of 16 bytes"):
        kv8.rope_kvwrite(qkv, i32([0, 1]), i32([0, 1]), K.rope_cos_sin(4, D, 1e4, device=DEV), 4, 2, D, kc, vc)
    with pytest.raises(ValueError, match="needs .* pages"):
        kv8.attn_prefill(q, kc, vc, bt, i32([0]), i32([1]), i32([900]), i32([[0, 0]]), 4, 2, 0.1,
                         host_meta=([1], [900]))
