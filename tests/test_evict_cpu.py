"""Decode attention with accumulated weights, and eviction by them, on the CPU; and what is refused."""

import math

import paged_oracle as O
import pytest
import torch

from infera_b200.ops import evict, kv8
from infera_b200.ops import kernels as K

SCALE = 1 / math.sqrt(128)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_decode_adds_weights():
    lens, hq, hkv = [1, 17, 0, 50], 6, 2
    table, pool = O.page_table(lens, 1)
    k, v = O.caches(pool, hkv)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(4, (hq + 2 * hkv) * 128, generator=g).to(torch.bfloat16)
    mass = torch.rand(4, hkv, 64, generator=g)
    was = mass.clone().double()
    out = K.attn_decode(q, k, v, table, i32(lens), hq, hkv, SCALE, mass=mass)
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.all(out[b] == 0)
            continue
        kk, vv = (O.rows_of(x, table[b], n, hkv) for x in (k, v))
        want, bound, w, wb = O.attend(q[b:b + 1, : hq * 128], kk, vv, torch.ones(1, n, dtype=torch.bool), hq, hkv, SCALE, 0.0)
        O.close(out[b:b + 1], want, bound)
        was[b, :, :n] += w[0].view(hkv, -1, n).sum(1)
    O.close(mass, was, 2.0 ** -16 * was + 1e-30)


def test_rows_that_do_not_exist_or_come_twice():
    table, pool = O.page_table([20, 20], 1)
    k, v = O.caches(pool, 1)
    q = torch.randn(4, 128).to(torch.bfloat16)
    mass = torch.zeros(2, 1, 16)
    out = evict.attn_decode(q, k, v, table, i32([20, 20, 20, 999]), 1, 1, SCALE, mass, bt_rows=i32([1, 5, 1, 0]))
    assert torch.all(out[1] == 0) and bool(out[3].any())
    kk = O.rows_of(k, table[1], 20, 1)[:, 0]
    w = torch.softmax(kk @ q[0].double() * SCALE, 0)[:16]
    O.close(mass[1, 0], w, 2.0 ** -16 * w)
    kept, m, count = evict.select_keys(mass, i32([16, 16, 3]), 4, bt_rows=i32([1, 2, 0]))
    assert count.tolist() == [4, 0, 3] and kept[1, 0].tolist() == [-1] * 4 and kept[2, 0].tolist() == [0, 1, 2, -1]


@pytest.mark.parametrize("keep,recent,sink", [(1, 0, 0), (5, 2, 1), (8, 8, 0), (8, 0, 8), (30, 7, 3), (64, 4, 4)])
def test_selection(keep, recent, sink):
    g = torch.Generator().manual_seed(5)
    lens = [1, 30, 0, 64, 40, 5]
    mass = torch.rand(6, 2, 64, generator=g)
    mass[3] = mass[3].mul(8).round()  # many equal ones
    mass[4, 0, 3:9] = torch.tensor([float("nan"), float("inf"), -0.0, 0.0, float("-inf"), -1.0])
    mass[4, 1] = float("nan")
    was = mass.clone()
    kept, kept_mass, count = evict.select_keys(mass, i32(lens), keep, recent, sink)
    assert torch.equal(mass.nan_to_num(7), was.nan_to_num(7))
    for s, n in enumerate(lens):
        assert int(count[s]) == min(n, keep)
        for h in range(2):
            on = O.select(was[s, h, :n].tolist(), keep, recent, sink)
            assert kept[s, h].tolist() == on + [-1] * (keep - len(on))
            x = kept_mass[s, h].nan_to_num(7)
            assert torch.equal(x[: len(on)], was[s, h, on].nan_to_num(7)) and torch.all(x[len(on):] == 0)
    again = evict.select_keys(mass, i32(lens), keep, recent, sink, update=True)
    assert torch.equal(again[0], kept)
    for s, n in enumerate(lens):
        if n > keep:
            assert torch.equal(mass[s, :, :keep].nan_to_num(7), kept_mass[s].nan_to_num(7))
            assert torch.all(mass[s, :, keep:n] == 0)
        assert torch.equal(mass[s, :, n:].nan_to_num(7), was[s, :, n:].nan_to_num(7))


def test_evicted_cache_attends_to_the_kept_keys():
    lens, hq, hkv, keep = [100, 37], 4, 2, 40
    table, pool = O.page_table(lens, 6)
    k, v = O.caches(pool, hkv)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, hq * 128, generator=g).to(torch.bfloat16)
    mass = evict.alloc_mass(2, hkv, 112, device="cpu")
    K.attn_decode(q, k, v, table, i32(lens), hq, hkv, SCALE, mass=mass)
    k0, v0 = k.clone(), v.clone()
    kept, _, count = evict.select_keys(mass, i32(lens), keep, recent=8, sink=2, update=True)
    K.kv_compact(k, v, table, kept, count)
    out = K.attn_decode(q, k, v, table, count, hq, hkv, SCALE, mass=mass)
    for s, n in enumerate(lens):
        kk, vv = (O.rows_of(x, table[s], n, hkv) for x in (k0, v0))
        on = [kept[s, h, : int(count[s])].long() for h in range(hkv)]
        kk, vv = (torch.stack([x[on[h], h] for h in range(hkv)], 1) for x in (kk, vv))
        want, bound, _, _ = O.attend(q[s:s + 1], kk, vv, torch.ones(1, len(on[0]), dtype=torch.bool), hq, hkv, SCALE, 0.0)
        O.close(out[s:s + 1], want, bound)


def test_refusals():
    table, pool = O.page_table([20, 20], 1)
    k, v = O.caches(pool, 2)
    q = torch.randn(2, 512).to(torch.bfloat16)
    mass = evict.alloc_mass(2, 2, 32, device="cpu")
    good = dict(q=q, k_cache=k, v_cache=v, block_table=table, seq_lens=i32([20, 20]), hq=4, hkv=2, scale=SCALE, mass=mass)
    evict.attn_decode(**good)
    k8 = kv8.alloc(k.shape[0], 2, device="cpu")
    for change, error in [(dict(k_cache=k8, v_cache=k8), TypeError), (dict(hq=18), ValueError), (dict(hq=5), ValueError),
                          (dict(mass=mass.double()), ValueError), (dict(mass=mass[0]), ValueError),
                          (dict(mass=mass[:, :1]), ValueError), (dict(mass=mass.transpose(0, 1)[:, :, ::2]), ValueError),
                          (dict(k_cache=k.half(), v_cache=v.half()), ValueError), (dict(v_cache=v[:16]), ValueError),
                          (dict(seq_lens=torch.tensor([20, 20])), ValueError), (dict(splits=0), ValueError),
                          (dict(tiles_per_split=-1), ValueError), (dict(block_table=table[:1]), ValueError),
                          (dict(bt_rows=i32([0])), ValueError), (dict(q=q[:1]), ValueError),
                          (dict(out=torch.empty(1, 512, dtype=torch.bfloat16)), ValueError)]:
        with pytest.raises(error):
            evict.attn_decode(**{**good, **change})
    for change in [dict(keep=0), dict(recent=-1), dict(sink=3, recent=2), dict(seq_lens=i32([[1, 2]])),
                   dict(mass=mass.half()), dict(mass=mass[0]), dict(bt_rows=i32([0]))]:
        with pytest.raises(ValueError):
            evict.select_keys(**{**dict(mass=mass, seq_lens=i32([3, 4]), keep=4), **change})
