"""The 8-bit paged KV cache on CPU: what an append stores, against the definition
in 64 bits, attention over it, and every refusal."""

import math

import pytest
import torch

from infera_b200.ops import kernels as K
from infera_b200.ops import kv8

D = 128


def random_cache(slots, hkv, seed=0, spread=3):
    """A channel with random codes (no NaN) and scales around 2^0."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(slots, hkv * D, generator=g) * 60
    sf = torch.randint(127 - spread, 128 + spread, (slots // 16, hkv), generator=g).to(torch.uint8)
    return kv8.KV8Cache(x.clamp(-448, 448).to(torch.float8_e4m3fn), sf)


def step(rows, hq, hkv, seed=0, max_pos=5000):
    """qkv, positions, cos / sin of a step with ``rows`` tokens."""
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(rows, (hq + 2 * hkv) * D, generator=g) * torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g))
    pos = torch.randint(0, max_pos, (rows,), generator=g).to(torch.int32)
    return qkv.to(torch.bfloat16), pos, K.rope_cos_sin(max_pos, D, 10000.0)


def turned(qkv, pos, cos_sin, hq, hkv):
    """(q, k, v) [T, heads, 128] in 64 bits: complex multiplication by each position's angle."""
    x = qkv[:, : (hq + 2 * hkv) * D].double().view(-1, hq + 2 * hkv, D)
    z = torch.complex(x[..., : D // 2], x[..., D // 2:])
    cs = cos_sin.double()[pos.long()]
    z = z * torch.complex(cs[..., 0], cs[..., 1])[:, None]
    r = torch.cat([z.real, z.imag], -1)
    return r[:, :hq], r[:, hq:hq + hkv], x[:, hq + hkv:]


def check_channel(before, after, rows, slots, hkv):
    """``after`` holds ``before`` with the 64-bit ``rows`` [T, heads, 128] appended at ``slots``.

    A code is off by half a step of its own (2^-4 of the value, 2^-10 below the
    normals) and the 32-bit rotation by 3 roundings of values that are at most
    sqrt(2) times the pair's, 2^-22 of the largest value of the page. A held
    row that was brought to a grown scale is off by half a step more."""
    last = {}
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            last[s] = t
    pages = {s // 16 for s in last}
    old, new = before.dequant().double().view(-1, hkv, D), after.dequant().double().view(-1, hkv, D)
    for page in range(after.sf.shape[0]):
        here = slice(page * 16, page * 16 + 16)
        if page not in pages:
            assert torch.equal(after.sf[page], before.sf[page])
            assert torch.equal(after.q[here].view(torch.uint8), before.q[here].view(torch.uint8))
            continue
        offs = [s % 16 for s in last if s // 16 == page]
        vals = rows[[last[page * 16 + o] for o in offs]]
        top = vals.abs().amax(dim=(0, 2))
        anew = 0 in offs
        for h in range(hkv):
            e = int(after.sf[page, h])
            grown = e > int(before.sf[page, h])
            t = float(top[h])
            unit = 2.0 ** (e - 127)
            # large enough, and the smallest that is (but for a value next to the border)
            assert t <= 448 * unit * (1 + 2 ** -22)
            if anew or grown:
                assert e == 1 or t > 224 * unit * (1 - 2 ** -22)
            else:
                assert e == int(before.sf[page, h])
            slack = t * 2 ** -22
            for o, x in zip(offs, vals[:, h]):
                err = (new[page * 16 + o, h] - x).abs()
                assert bool((err <= torch.maximum(x.abs() * 2 ** -4, torch.tensor(unit * 2 ** -10)) + slack).all())
            for o in set(range(16)) - set(offs):
                if anew or not grown:  # as they were (of a page that starts anew: the codes)
                    assert torch.equal(after.q[page * 16 + o].view(torch.uint8).view(hkv, D)[h],
                                       before.q[page * 16 + o].view(torch.uint8).view(hkv, D)[h])
                else:
                    err = (new[page * 16 + o, h] - old[page * 16 + o, h]).abs()
                    assert bool((err <= unit * 2 ** -10).all())  # codes that became subnormal


APPENDS = {
    "one row": [37],
    "one row, first of its page": [48],
    "last slot": [16 * 12 - 1],
    "a page and more": list(range(5, 40)),
    "whole pages": list(range(32, 64)),
    "out of order": [70, 33, 66, 35, 64, 34, 7, 65],
    "not stored": [-1, 20, -1, 21, -1],
    "same slot twice": [20, 21, 20, 99, 20],
    "all skipped": [-1, -1],
}


@pytest.mark.parametrize("name", APPENDS)
@pytest.mark.parametrize("hq,hkv", [(4, 2), (1, 1), (8, 1)])
def test_append(name, hq, hkv):
    slots = torch.tensor(APPENDS[name], dtype=torch.int32)
    qkv, pos, cs = step(len(slots), hq, hkv, seed=len(name))
    kc, vc = random_cache(192, hkv, 1), random_cache(192, hkv, 2)
    k0, v0 = kv8.KV8Cache(kc.q.clone(), kc.sf.clone()), kv8.KV8Cache(vc.q.clone(), vc.sf.clone())
    before = qkv.clone()
    out = torch.empty(len(slots), hq * D, dtype=torch.bfloat16)
    got = kv8.rope_kvwrite(qkv, pos, slots, cs, hq, hkv, D, kc, vc, q_out=out)
    assert got is out and torch.equal(qkv, before)
    q, k, v = turned(qkv, pos, cs, hq, hkv)
    check_channel(k0, kc, k, slots, hkv)
    check_channel(v0, vc, v, slots, hkv)
    # bf16: half a step, and the roundings of the rotation (against the pair's size)
    size = q.abs().amax()
    assert bool(((out.double().view_as(q) - q).abs() <= q.abs() * 2 ** -8 + size * 2 ** -22).all())
    # the same call again changes nothing
    k1, v1 = kc.q.clone(), vc.sf.clone()
    kv8.rope_kvwrite(qkv, pos, slots, cs, hq, hkv, D, kc, vc, q_out=out)
    assert torch.equal(kc.q.view(torch.uint8), k1.view(torch.uint8)) and torch.equal(vc.sf, v1)


def test_append_in_place_and_through_the_kernel_entry():
    qkv, pos, cs = step(9, 4, 2)
    slots = torch.arange(9, dtype=torch.int32) + 16
    a, b = [kv8.alloc(64, 2, device="cpu") for _ in range(2)], [kv8.alloc(64, 2, device="cpu") for _ in range(2)]
    mine = qkv.clone()
    out = kv8.rope_kvwrite(qkv, pos, slots, cs, 4, 2, D, *a, q_out=torch.empty(9, 4 * D, dtype=torch.bfloat16))
    K.rope_kvwrite(mine, pos, slots, cs, 4, 2, D, *b)
    assert torch.equal(mine[:, :4 * D], out) and torch.equal(mine[:, 4 * D:], qkv[:, 4 * D:])
    for x, y in zip(a, b):
        assert torch.equal(x.q.view(torch.uint8), y.q.view(torch.uint8)) and torch.equal(x.sf, y.sf)


def test_append_zeros_infinities_and_nan():
    kc, vc = kv8.alloc(32, 1, device="cpu"), kv8.alloc(32, 1, device="cpu")
    qkv = torch.zeros(3, 3 * D, dtype=torch.bfloat16)
    qkv[1, 2 * D] = float("inf")
    qkv[1, 2 * D + 1] = 2.0
    qkv[2, 2 * D + 5] = float("nan")
    pos = torch.zeros(3, dtype=torch.int32)
    kv8.rope_kvwrite(qkv, pos, torch.tensor([0, 1, 16], dtype=torch.int32), K.rope_cos_sin(4, D, 1e4), 1, 1, D, kc, vc)
    assert int(kc.sf[0, 0]) == 1 and not kc.dequant().any()  # zeros: the smallest scale, which any later row raises
    v = vc.dequant()
    assert v[1, 0].isnan() and v[1, 1] == 2.0 and int(vc.sf[0, 0]) == 127 - 7  # 2 = 256 * 2^-7: the finite values set it
    assert v[16, 5].isnan() and int(v[16:17].isnan().sum()) == 1 and int(vc.sf[1, 0]) == 1


@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_attention(G):
    hkv, hq = 2, 2 * G
    kc, vc = random_cache(16 * 40, hkv, 3), random_cache(16 * 40, hkv, 4)
    lens = [1, 0, 100, 33]
    g = torch.Generator().manual_seed(5)
    bt = torch.randperm(40, generator=g).to(torch.int32).view(4, 10)
    q = (torch.randn(4, hq * D, generator=g) / 60).to(torch.bfloat16)
    y = K.attn_decode(q, kc, vc, bt, torch.tensor(lens, dtype=torch.int32), hq, hkv, 0.1)
    k, v = kc.dequant().double().view(-1, hkv, D), vc.dequant().double().view(-1, hkv, D)
    for b, n in enumerate(lens):
        slots = (bt[b].long()[:, None] * 16 + torch.arange(16)).flatten()[:n]
        for h in range(hq):
            s = k[slots, h // G] @ q[b, h * D:(h + 1) * D].double() * 0.1
            p = torch.softmax(s, 0)
            o = p @ v[slots, h // G] if n else torch.zeros(D, dtype=torch.float64)
            a = p @ v[slots, h // G].abs() if n else o
            # half a step of bf16, and 32-bit sums (2^-20 of the terms' sizes)
            assert bool(((y[b, h * D:(h + 1) * D].double() - o).abs() <= o.abs() * 2 ** -8 + a * 2 ** -20).all())
    # a prompt chunk's rows see what single tokens at their places see
    n = 21
    qp = (torch.randn(n, hq * D, generator=g) / 60).to(torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    tiles = torch.tensor(K.prefill_tiles([n]), dtype=torch.int32)
    yp = K.attn_prefill(qp, kc, vc, bt, i32(0), i32(n), i32(90), tiles, hq, hkv, 0.1, bt_rows=i32(2))
    ones = kv8.attn_decode(qp, kc, vc, bt, torch.arange(90 - n + 1, 91).to(torch.int32), hq, hkv, 0.1,
                           bt_rows=torch.full((n,), 2, dtype=torch.int32))
    assert bool(((yp.float() - ones.float()).abs() <= 2 ** -7 * ones.float().abs() + 1e-5).all())


def test_alloc_layers_and_dequant():
    c = kv8.alloc(64, 3, layers=2, device="cpu")
    assert tuple(c.shape) == (2, 64, 3 * D) and tuple(c.sf.shape) == (2, 4, 3) and not c.dequant().any()
    assert c.nbytes == 2 * (64 * 3 * D + 12)
    one = c[1]
    one.q.view(torch.uint8)[17, D + 4] = torch.tensor([1.5]).to(torch.float8_e4m3fn).view(torch.uint8)
    one.sf[1, 1] = 130
    assert c.dequant()[1, 17, D + 4] == 12.0 and int((c.dequant() != 0).sum()) == 1
    for bad in ((40, 1), (0, 1), (16, 0)):
        with pytest.raises(ValueError):
            kv8.alloc(*bad, device="cpu")


@pytest.mark.parametrize("batch", [1, 3, 64, 500])
@pytest.mark.parametrize("hkv", [1, 8])
@pytest.mark.parametrize("group", [1, 8])
@pytest.mark.parametrize("longest", [0, 1, 128, 129, 5000, 131072])
def test_decode_plan_covers(batch, hkv, longest, group):
    splits, tps = kv8.decode_plan(batch, hkv, longest, group=group)
    assert splits >= 1 and tps >= 1 and splits * tps * 128 >= longest
    assert (splits - 1) * tps * 128 < max(longest, 1)


def append_args(**over):
    qkv, pos, cs = step(3, 4, 2)
    a = dict(qkv=qkv, pos=pos, slots=torch.arange(3, dtype=torch.int32), cos_sin=cs, hq=4, hkv=2, head_dim=D,
             k_cache=kv8.alloc(32, 2, device="cpu"), v_cache=kv8.alloc(32, 2, device="cpu"))
    a.update(over)
    return a


APPEND_REFUSALS = {
    "head_dim": dict(head_dim=64),
    "heads": dict(hq=3),
    "no heads": dict(hkv=0),
    "narrow qkv": dict(hq=6),
    "qkv type": dict(qkv=torch.zeros(3, 8 * D)),
    "qkv layout": dict(qkv=torch.zeros(8 * D, 3, dtype=torch.bfloat16).t()),
    "pos type": dict(pos=torch.zeros(3, dtype=torch.int64)),
    "pos length": dict(pos=torch.zeros(2, dtype=torch.int32)),
    "slots stride": dict(slots=torch.zeros(6, dtype=torch.int32)[::2]),
    "angles type": dict(cos_sin=torch.zeros(10, 64, 2, dtype=torch.bfloat16)),
    "angles shape": dict(cos_sin=torch.zeros(10, 32, 2)),
    "mixed caches": dict(v_cache=torch.zeros(32, 2 * D, dtype=torch.bfloat16)),
    "slots of K and V": dict(v_cache=kv8.alloc(48, 2, device="cpu")),
    "cache heads": dict(k_cache=kv8.alloc(32, 4, device="cpu"), v_cache=kv8.alloc(32, 4, device="cpu")),
    "all layers": dict(k_cache=kv8.alloc(32, 2, layers=2, device="cpu")),
    "q_out rows": dict(q_out=torch.zeros(2, 4 * D, dtype=torch.bfloat16)),
    "q_out width": dict(q_out=torch.zeros(3, 3 * D, dtype=torch.bfloat16)),
    "q_out type": dict(q_out=torch.zeros(3, 4 * D)),
}


@pytest.mark.parametrize("name", APPEND_REFUSALS)
def test_append_refuses(name):
    with pytest.raises((ValueError, TypeError)):
        kv8.rope_kvwrite(**append_args(**APPEND_REFUSALS[name]))


def test_cache_refuses():
    e4m3, u8 = torch.float8_e4m3fn, torch.uint8
    q, sf = torch.zeros(32, 2 * D, dtype=u8).view(e4m3), torch.zeros(2, 2, dtype=u8)
    kv8.KV8Cache(q, sf)
    wide = torch.zeros(32, 4 * D, dtype=u8).view(e4m3)
    for bad in ((q.view(torch.float8_e5m2), sf), (q, sf.int()), (q, sf[:1]), (q[:31], sf), (q, torch.zeros(2, 3, dtype=u8)),
                (wide[:, : 2 * D], sf), (q, torch.zeros(2, 4, dtype=u8)[:, :2]), (q[None], sf), (q[:0], sf[:0]),
                (q.view(-1), sf.view(-1)), (q[None, None], sf[None, None])):
        with pytest.raises(ValueError):
            kv8.KV8Cache(*bad)
    with pytest.raises(TypeError):
        kv8.KV8Cache(q, sf)[0]
    both = kv8.alloc(32, 2, layers=3, device="cpu")
    assert both[2] is both[2] and both[2].q.data_ptr() == both.q[2].data_ptr()


def attend_args(**over):
    a = dict(q=torch.zeros(2, 4 * D, dtype=torch.bfloat16), k_cache=kv8.alloc(32, 2, device="cpu"),
             v_cache=kv8.alloc(32, 2, device="cpu"), block_table=torch.zeros(2, 2, dtype=torch.int32),
             seq_lens=torch.ones(2, dtype=torch.int32), hq=4, hkv=2, scale=1.0)
    a.update(over)
    return a


DECODE_REFUSALS = {
    "group": dict(hq=18, q=torch.zeros(2, 18 * D, dtype=torch.bfloat16)),
    "heads": dict(hq=3),
    "q type": dict(q=torch.zeros(2, 4 * D)),
    "q width": dict(q=torch.zeros(2, 3 * D, dtype=torch.bfloat16)),
    "q rows": dict(q=torch.zeros(1, 4 * D, dtype=torch.bfloat16)),
    "lengths type": dict(seq_lens=torch.ones(2)),
    "table type": dict(block_table=torch.zeros(2, 2, dtype=torch.int64)),
    "table rows": dict(block_table=torch.zeros(1, 2, dtype=torch.int32)),
    "table layout": dict(block_table=torch.zeros(2, 2, dtype=torch.int32).t()),
    "bt_rows": dict(bt_rows=torch.zeros(3, dtype=torch.int32)),
    "splits": dict(splits=0),
    "tiles": dict(tiles_per_split=-1),
    "out width": dict(out=torch.zeros(2, 3 * D, dtype=torch.bfloat16)),
    "out rows": dict(out=torch.zeros(1, 4 * D, dtype=torch.bfloat16)),
    "one bf16 cache": dict(v_cache=torch.zeros(32, 2 * D, dtype=torch.bfloat16)),
    "slots of K and V": dict(k_cache=kv8.alloc(48, 2, device="cpu")),
}


@pytest.mark.parametrize("name", DECODE_REFUSALS)
def test_decode_refuses(name):
    with pytest.raises((ValueError, TypeError)):
        kv8.attn_decode(**attend_args(**DECODE_REFUSALS[name]))


PREFILL_REFUSALS = {
    "lengths type": dict(q_len=torch.ones(1)),
    "lengths count": dict(ctx_len=torch.ones(2, dtype=torch.int32)),
    "host lengths": dict(host_meta=([1, 1], [1, 1])),
    "q type": dict(q=torch.zeros(2, 4 * D)),
    "heads": dict(hq=5),
    "group": dict(hq=18, q=torch.zeros(2, 18 * D, dtype=torch.bfloat16)),
    "negative chunk": dict(host_meta=([-1], [1])),
    "out rows": dict(out=torch.zeros(1, 4 * D, dtype=torch.bfloat16)),
    "bf16 caches": dict(v_cache=torch.zeros(32, 2 * D, dtype=torch.bfloat16)),
    "table rows": dict(block_table=torch.zeros(0, 2, dtype=torch.int32)),
}


def test_prefill_nan_reaches_the_rows_that_see_it():
    n, ctx, hq, hkv = 20, 40, 4, 2
    kc, vc = random_cache(48, hkv, 1), random_cache(48, hkv, 2)
    bt, one = torch.tensor([[2, 0, 1]], dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = (torch.randn(n, hq * D, generator=torch.Generator().manual_seed(1)) / 60).to(torch.bfloat16)

    def run():
        return kv8.attn_prefill(q, kc, vc, bt, one - 1, one * n, one * ctx, None, hq, hkv, 0.1)

    clean = run()
    vc.q.view(torch.uint8)[0 + 30 - 16, D + 5] = 0x7F  # key 30 stands in page 0: rows 10 .. see it
    y = run()
    want = torch.zeros(n, hq, D, dtype=torch.bool)
    want[10:, 2:, 5] = True
    want = want.view(n, -1)
    assert torch.equal(y.isnan(), want) and torch.equal(y[~want], clean[~want])


@pytest.mark.parametrize("name", PREFILL_REFUSALS)
def test_prefill_refuses(name):
    a = attend_args()
    del a["seq_lens"]
    one = torch.ones(1, dtype=torch.int32)
    a.update(q_start=torch.zeros(1, dtype=torch.int32), q_len=one, ctx_len=one,
             tiles=torch.zeros(1, 2, dtype=torch.int32))
    a.update(PREFILL_REFUSALS[name])
    with pytest.raises((ValueError, TypeError)):
        kv8.attn_prefill(**a)


@pytest.mark.parametrize("q_lens,ctx_lens", [([1], [1]), ([17], [4113]), ([224], [8416]), ([5, 0, 300], [5, 0, 9000]),
                                             ([], []), ([2048] * 4, [2048] * 4), ([1], [131072])])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (64, 8)])
def test_prefill_plan(q_lens, ctx_lens, hq, hkv):
    items, rows, shares = kv8.prefill_plan(q_lens, ctx_lens, hq, hkv)
    per = 256 // (hq // hkv)
    assert rows == sum(q_lens) and items == sum(math.ceil(n / per) for n in q_lens)
    tiles = math.ceil(max(ctx_lens, default=0) / 128)
    assert 1 <= shares <= max(1, min(64, tiles))
