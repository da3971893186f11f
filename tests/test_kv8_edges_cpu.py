"""The 8-bit paged KV cache on CPU at the ends of its ranges, and the calls that
it refuses there."""

import pytest
import torch

from infera_b200.ops import kernels as K
from infera_b200.ops import kv8
from test_kv8_cpu import random_cache

D = 128


@pytest.mark.parametrize("e", [253, 254, 255])
def test_largest_scales(e):
    """Exponents end at 253, and 254 and 255 count as it: a row that joins such a page keeps its values."""
    hkv = 2
    kc, vc = [kv8.KV8Cache(random_cache(32, hkv, s).q, torch.full((2, hkv), e, dtype=torch.uint8)) for s in (1, 2)]
    old = vc.q.float()
    assert bool((vc.dequant()[16:] == (old * 2.0 ** 126)[16:]).all())  # (infinite above 2)
    qkv = torch.full((1, 8 * D), 2.0 ** 120, dtype=torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32)
    kv8.rope_kvwrite(qkv, zero, zero + 21, K.rope_cos_sin(2, D, 1e4), 4, hkv, D, kc, vc)
    for c in (kc, vc):
        assert bool((c.dequant()[21] == 2.0 ** 120).all()) and bool((c.sf[1] == 253).all())
    rest = [16 + o for o in range(16) if o != 5]
    assert torch.equal(vc.q.float()[rest], old[rest]) and torch.equal(vc.q.float()[:16], old[:16])


def attention_case(lens, hq, hkv, rows, seed=1):
    """(q, K, V, page table) of sequences on pages of their own, two pages to spare."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // 16) for n in lens]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=g).to(torch.int32)
    bt = torch.zeros(len(lens), max(need), dtype=torch.int32)
    for i, n in enumerate(need):
        bt[i, :n] = order[sum(need[:i]):sum(need[:i]) + n]
    q = (torch.randn(rows, hq * D, generator=g) / 60).to(torch.bfloat16)
    return q, random_cache(pool * 16, hkv, seed), random_cache(pool * 16, hkv, seed + 1), bt


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_attention_in_place():
    """The output may be the queries' own memory."""
    hq, hkv = 4, 2
    q, kc, vc, bt = attention_case([40, 1, 70], hq, hkv, 3)
    args = (kc, vc, bt, i32(40, 0, 70), hq, hkv, 0.1)
    want = kv8.attn_decode(q, *args)
    mine = q.clone()
    assert kv8.attn_decode(mine, *args, out=mine) is mine and torch.equal(mine, want)
    assert bool(want[0].any()) and not want[1].any()
    q, kc, vc, bt = attention_case([40, 70], hq, hkv, 25)
    args = (kc, vc, bt, i32(0, 20), i32(20, 5), i32(13, 70), None, hq, hkv, 0.1)
    want = kv8.attn_prefill(q, *args)
    kv8.attn_prefill(q, *args, out=q)
    assert torch.equal(q, want)


def test_bad_tables_and_lengths():
    """What the kernels find wrong is treated alike on CPU: a row that the table has not gives zeros (a negative one is
    not counted from the end), a page id outside the cache reads as zeros, a length ends where the table does."""
    hq, hkv = 4, 2
    q, kc, vc, bt = attention_case([70, 40], hq, hkv, 2)
    decode = lambda table, lens, **kw: kv8.attn_decode(q, kc, vc, table, i32(*lens), hq, hkv, 0.1, **kw)  # noqa: E731
    good = decode(bt, (70, 40))
    for bad in (-1, 2, -3):
        y = decode(bt, (70, 40), bt_rows=i32(0, bad))
        assert torch.equal(y[0], good[0]) and not y[1].any()
        yp = kv8.attn_prefill(q, kc, vc, bt, i32(0, 1), i32(1, 1), i32(70, 40), None, hq, hkv, 0.1, bt_rows=i32(bad, 0))
        assert not yp[0].any() and bool(yp[1].any())
    assert torch.equal(decode(bt, (1000, -7))[0], decode(bt, (16 * bt.shape[1], 0))[0])
    assert not decode(bt, (1000, -7))[1].any()
    pages = kc.sf.shape[0]
    blank = [kv8.KV8Cache(torch.cat([c.q, torch.zeros_like(c.q[:16])]), torch.cat([c.sf, torch.ones_like(c.sf[:1])]))
             for c in (kc, vc)]
    none = bt.clone()
    none[0, 1] = pages
    want = kv8.attn_decode(q, *blank, none, i32(70, 40), hq, hkv, 0.1)
    wantp = kv8.attn_prefill(q, *blank, none, i32(0), i32(2), i32(70), None, hq, hkv, 0.1)
    for bad in (pages, -1, 2 ** 28 + 1, 2 ** 31 - 1):
        none[0, 1] = bad
        assert torch.equal(decode(none, (70, 40)), want)
        assert torch.equal(kv8.attn_prefill(q, kc, vc, none, i32(0), i32(2), i32(70), None, hq, hkv, 0.1), wantp)


def test_prefill_refuses_on_cpu_what_it_refuses_on_the_gpu():
    hq, hkv = 4, 2
    q, kc, vc, bt = attention_case([70], hq, hkv, 4)
    for n, ctx, kw in ((4, 16 * bt.shape[1] + 1, {}), (5, 70, {}), (4, 70, dict(kv_splits=0)), (4, 70, dict(kv_splits=70000))):
        with pytest.raises(ValueError):
            kv8.attn_prefill(q, kc, vc, bt, i32(0), i32(n), i32(ctx), None, hq, hkv, 0.1, **kw)


def test_rows_that_share_memory():
    """Read, rows may start anywhere; written, they have to be apart."""
    hq, hkv = 4, 2
    q, kc, vc, bt = attention_case([30, 70], hq, hkv, 2)
    one = torch.zeros(1, hq * D, dtype=torch.bfloat16)
    shared = (one.expand(2, -1), torch.zeros(2 * hq * D, dtype=torch.bfloat16).as_strided((2, hq * D), (hq * D - 8, 1)))
    want = kv8.attn_decode(q[:1].repeat(2, 1), kc, vc, bt, i32(30, 70), hq, hkv, 0.1)
    assert torch.equal(kv8.attn_decode(q[:1].expand(2, -1), kc, vc, bt, i32(30, 70), hq, hkv, 0.1), want)
    for out in shared:
        with pytest.raises(ValueError, match="share memory"):
            kv8.attn_decode(q, kc, vc, bt, i32(30, 70), hq, hkv, 0.1, out=out)
        with pytest.raises(ValueError, match="share memory"):
            kv8.attn_prefill(q, kc, vc, bt, i32(0, 1), i32(1, 1), i32(30, 70), None, hq, hkv, 0.1, out=out)
    qkv, cs = torch.ones(1, 8 * D, dtype=torch.bfloat16).expand(2, -1), K.rope_cos_sin(4, D, 1e4)
    with pytest.raises(ValueError, match="share memory"):
        kv8.rope_kvwrite(qkv, i32(0, 1), i32(3, 4), cs, hq, hkv, D, kc, vc)
    for out in shared:
        with pytest.raises(ValueError, match="share memory"):
            kv8.rope_kvwrite(qkv, i32(0, 1), i32(3, 4), cs, hq, hkv, D, kc, vc, q_out=out)
    kv8.rope_kvwrite(qkv, i32(0, 1), i32(3, 4), cs, hq, hkv, D, kc, vc, q_out=torch.empty_like(q))


def test_one_cache_for_keys_and_values():
    """K and V of an append need memory of their own; attention may read one cache as both."""
    hq, hkv = 4, 2
    q, kc, vc, bt = attention_case([30], hq, hkv, 1)
    qkv, cs = torch.ones(1, 8 * D, dtype=torch.bfloat16), K.rope_cos_sin(4, D, 1e4)
    long = random_cache(96, hkv)
    for k, v in ((kc, kc), (kc, kv8.KV8Cache(kc.q, vc.sf)), (kc, kv8.KV8Cache(vc.q, kc.sf)),
                 (kv8.KV8Cache(long.q[:64], long.sf[:4]), kv8.KV8Cache(long.q[32:], long.sf[2:]))):
        with pytest.raises(ValueError, match="same memory"):
            kv8.rope_kvwrite(qkv, i32(0), i32(3), cs, hq, hkv, D, k, v)
    layers = kv8.alloc(32, hkv, layers=2, device="cpu")
    kv8.rope_kvwrite(qkv, i32(0), i32(3), cs, hq, hkv, D, layers[0], layers[1])
    assert bool(kv8.attn_decode(q, kc, kc, bt, i32(30), hq, hkv, 0.1).any())
