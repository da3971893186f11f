"""Decode attention with accumulated weights, and eviction by them, on the GPU against 64-bit forms."""

import math

import paged_oracle as O
import pytest
import torch

from infera_b200.ops import evict
from infera_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)
W_STEP = 2.0 ** -16  # a weight's two bf16 digits leave at most 2^-8 of 2^-8 of it


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def status():
    torch.cuda.synchronize()
    s = K.scratch().read_status_detail()
    K.scratch().clear_status()
    return s


def batch(lens, hq, hkv, seed=0, runs=False, pad=0):
    g = torch.Generator().manual_seed(seed)
    table, pool = O.page_table(lens, seed, runs)
    k, v = O.caches(pool, hkv, seed)
    q = torch.randn(len(lens), (hq + 2 * hkv) * 128 + pad, generator=g).to(torch.bfloat16)
    # places that no sequence has are NaN, as a recycled page may leave them
    own = torch.zeros(k.shape[0], dtype=torch.bool)
    for row, c in zip(table, lens):
        p = torch.arange(c)
        own[row[p // 16].long() * 16 + p % 16] = True
    k[~own], v[~own] = float("nan"), float("nan")
    mass = torch.rand(len(lens), hkv, table.shape[1] * 16, generator=g)
    return q, k, v, table, mass


def check(out, mass, q, k, v, table, was, lens, hq, hkv, scale=SCALE):
    was, bound_m = was.double(), 2.0 ** -23 * was.double() + 1e-37
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.all(out[b] == 0)
            continue
        kk, vv = (O.rows_of(x, table[b], n, hkv) for x in (k, v))
        want, bound, w, wb = O.attend(q[b:b + 1, : hq * 128], kk, vv, torch.ones(1, n, dtype=torch.bool), hq, hkv, scale, W_STEP)
        O.close(out[b:b + 1], want, bound, f"sequence {b}")
        was[b, :, :n] += w[0].view(hkv, -1, n).sum(1)
        # (sums of up to 8 weights and the mass, and exp2's 2^-22)
        bound_m[b, :, :n] += (wb + 2.0 ** -20 * w)[0].view(hkv, -1, n).sum(1)
    O.close(mass, was, bound_m, "mass")


LENS = {"one key": [1], "short": [100], "a tile": [128, 129, 127], "ragged": [5, 0, 700, 16, 1025, 300], "many": [40] * 70}


@pytest.mark.parametrize("plan", ["plan", (1, 0), (5, 0), (20, 1)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (32, 8), (16, 2), (3, 1), (14, 2)])
@pytest.mark.parametrize("name", LENS)
def test_decode(name, hq, hkv, plan):
    lens = LENS[name]
    q, k, v, table, mass = batch(lens, hq, hkv, seed=hq + len(lens))
    splits, tps = evict.decode_plan(len(lens), hkv, max(lens)) if plan == "plan" else plan
    got = mass.cuda()
    out = K.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, hkv, SCALE, splits=splits,
                        tiles_per_split=tps, mass=got)
    assert status()["code"] == 0
    check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, hkv)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("runs", [False, True])
def test_decode_scale_stride_and_growing_maxima(runs, scale):
    lens, hq, hkv = [900, 333], 8, 2
    q, k, v, table, mass = batch(lens, hq, hkv, 3, runs, pad=6)
    for p in range(lens[0]):
        k[int(table[0, p // 16]) * 16 + p % 16] *= p / 100
    for splits, tps in ((1, 0), (3, 3)):
        got, buf = mass.cuda(), torch.zeros(2, hq * 128 + 2, dtype=torch.bfloat16, device="cuda")
        out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, hkv, scale, got, splits, out=buf,
                                tiles_per_split=tps)
        assert torch.all(buf[:, hq * 128:] == 0)
        check(out.cpu()[:, : hq * 128], got.cpu(), q, k, v, table, mass, lens, hq, hkv, scale)


def test_decode_bad_pages_rows_and_lengths():
    lens, hq, hkv = [100, 300, 60], 4, 1
    q, k, v, table, mass = batch(lens, hq, hkv, 4)
    table[0, 2], table[1, 5] = -4, 2 ** 30 + 1
    args = [q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, hkv, SCALE]
    got = mass.cuda()
    out = evict.attn_decode(*args, got, 2)
    check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, hkv)
    assert status()["code"] == 0
    # a row that does not exist, one that came before, one beyond the mass
    got = mass.cuda()[:2].contiguous()
    out = evict.attn_decode(*args, got, 2, bt_rows=i32([1, 9, 1])).cpu()
    assert torch.all(out[1] == 0) and status()["code"] == 7
    check(out[:1], got.cpu()[1:], q, k, v, table[1:], mass[1:2], [100], hq, hkv)
    assert torch.equal(got.cpu()[0], mass[0])
    got = mass.cuda()[:2].contiguous()
    out = evict.attn_decode(*args, got, 2).cpu()
    assert status()["code"] == 7 and bool(out[2].any())
    # fewer places in the mass than keys; keys that no split covers; more than the table holds
    got = mass[:, :, :150].contiguous().cuda()
    out = evict.attn_decode(*args, got, 2).cpu()
    full = mass.clone()
    check(out, torch.cat([got.cpu(), torch.zeros(3, 1, mass.shape[2] - 150)], 2)[:1], q, k, v, table, full[:1], lens[:1], hq, hkv) \
        if mass.shape[2] <= 150 else None
    assert status()["code"] == 7
    got = mass.cuda()
    out = evict.attn_decode(*args, got, 1, tiles_per_split=1).cpu()
    assert status()["code"] == 6
    check(out[:1], got.cpu()[:1], q, k, v, table, mass[:1], lens[:1], hq, hkv)
    args[4] = i32([100, 300, 5000])
    evict.attn_decode(*args, mass.cuda(), 2)
    assert status()["code"] == 7


def test_decode_nan_where_it_is_seen():
    lens, hq = [200, 200], 4
    q, k, v, table, mass = batch(lens, hq, 1, 5)
    v[int(table[0, 3]) * 16 + 1, 9] = float("nan")
    k[int(table[1, 3]) * 16 + 1] = float("nan")
    got = mass.cuda()
    out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, 1, SCALE, got, 1).cpu()
    nan = out[0].isnan().view(hq, 128)
    assert nan[:, 9].all() and int(nan.sum()) == hq and bool(got[0].isfinite().all())
    assert out[1].isnan().all() and got[1, 0, :200].isnan().all() and bool(got[1, 0, 200:].isfinite().all())


def test_decode_captured_with_other_lengths_and_into_the_queries():
    lens, hq, hkv = [700, 300], 8, 2
    q, k, v, table, mass = batch(lens, hq, hkv, 6)
    dev = [x.cuda() for x in (k, v, table)]
    lens_d, got = i32(lens), [mass.cuda(), mass.cuda()]
    qs = [q.cuda(), q.cuda()]
    graphs = []
    for i in range(2):
        evict.attn_decode(q.cuda(), *dev, lens_d, hq, hkv, SCALE, mass.cuda(), 3, tiles_per_split=2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            evict.attn_decode(qs[i], *dev, lens_d, hq, hkv, SCALE, got[i], 3, out=qs[i], tiles_per_split=2)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for now in ([700, 300], [1, 129], [0, 650]):
        now[1] = min(now[1], 300)
        lens_d.copy_(i32(now))
        for i in range(2):
            got[i].copy_(mass), qs[i].copy_(q)
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            check(qs[i].cpu()[:, : hq * 128], got[i].cpu(), q, k, v, table, mass, now, hq, hkv)


# ---------------------------------------------------------------- selection


@pytest.mark.parametrize("keep,recent,sink", [(1, 0, 0), (7, 3, 2), (64, 64, 0), (64, 0, 64), (64, 8, 4), (3000, 100, 16)])
@pytest.mark.parametrize("lens,hkv", [([1, 64, 0, 65, 100], 2), ([5000, 2999, 3001], 2), ([40001], 8), ([2048] * 20, 4),
                                      ([50001] + [100] * 79, 1)])
def test_selection(lens, hkv, keep, recent, sink):
    g = torch.Generator().manual_seed(keep + len(lens))
    cap = max(lens) + 5
    mass = torch.exp(3 * torch.randn(len(lens), hkv, cap, generator=g))
    mass[:, 0] = (mass[:, 0] * 2).round()  # many equal ones
    mass[-1, -1, ::7] = 0
    mass[-1, -1, 1::97] = torch.tensor(float("nan"))
    mass[-1, -1, 2::89] = -mass[-1, -1, 2::89]
    mass[-1, -1, 3::400], mass[-1, -1, 4::400] = float("inf"), float("-inf")
    mass[-1, -1, ::50] = -0.0
    dev = mass.cuda()
    kept, kept_mass, count = (x.cpu() for x in evict.select_keys(dev, i32(lens), keep, recent, sink))
    same = lambda a, b: torch.equal(a.nan_to_num(1e30), b.nan_to_num(1e30))  # noqa: E731
    assert same(dev.cpu(), mass)
    for s, n in enumerate(lens):
        assert int(count[s]) == min(n, keep)
        for h in range(hkv):
            on = O.select(mass[s, h, :n].tolist(), keep, recent, sink)
            assert kept[s, h].tolist() == on + [-1] * (keep - len(on)), (s, h)
            assert same(kept_mass[s, h, : len(on)], mass[s, h, on]) and torch.all(kept_mass[s, h, len(on):] == 0)
    again = evict.select_keys(dev, i32(lens), keep, recent, sink, update=True)
    assert torch.equal(again[0].cpu(), kept)
    got = dev.cpu()
    for s, n in enumerate(lens):
        if n > keep:
            assert same(got[s, :, :keep], kept_mass[s]) and torch.all(got[s, :, keep:n] == 0)
        assert same(got[s, :, n if n > keep else 0:], mass[s, :, n if n > keep else 0:])
    assert status()["code"] == 0


def test_selection_of_bad_rows_and_lengths():
    mass = torch.rand(3, 2, 50, device="cuda")
    was = mass.clone()
    kept, m, count = evict.select_keys(mass, i32([40, 40, 99]), 10, bt_rows=i32([2, 3, 0]))
    assert count.tolist() == [10, 0, 10] and torch.all(kept[1] == -1) and torch.all(m[1] == 0)
    assert kept[2, 0].tolist() == O.select(was[0, 0].tolist(), 10, 0, 0) and status()["code"] == 7
    kept, _, count = evict.select_keys(mass, i32([40, 40]), 10, bt_rows=i32([1, 1]), update=True)
    assert count.tolist() == [10, 0] and torch.all(mass[1, :, 10:40] == 0) and status()["code"] == 7
    kept, _, count = evict.select_keys(mass, i32([]), 10)
    assert kept.shape == (0, 2, 10)


# ---------------------------------------------------------------- moving


@pytest.mark.parametrize("lens,hkv,keep", [([70], 1, 40), ([300, 41, 900], 2, 40), ([5000, 1200], 8, 1100),
                                           ([2100] * 30, 2, 2000)])
def test_kept_rows_move(lens, hkv, keep):
    g = torch.Generator().manual_seed(len(lens))
    table, pool = O.page_table(lens, 3)
    k, v = (torch.randn(pool * 16, hkv * 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    mass = torch.rand(len(lens), hkv, table.shape[1] * 16, generator=g).cuda()
    kept, _, count = evict.select_keys(mass, i32(lens), keep, recent=10, sink=3)
    want = []
    place = torch.arange(keep, device="cuda")
    for x in (k, v):
        y = x.clone()
        for s in range(len(lens)):
            c = int(count[s])
            t = table[s].cuda().long()
            for h in range(hkv):
                a, b = kept[s, h, :c].long(), place[:c]
                y[t[b // 16] * 16 + b % 16, h * 128:(h + 1) * 128] = x[t[a // 16] * 16 + a % 16, h * 128:(h + 1) * 128]
        want.append(y)
    K.kv_compact(k, v, table.cuda(), kept, count)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and status()["code"] == 0


def test_evict_and_decode_on():
    """Steps that add up weights, an eviction, and steps over what is left."""
    lens, hq, hkv, keep = [700, 64, 333], 8, 2, 200
    q, k, v, table, _ = batch(lens, hq, hkv, 11)
    dev = [x.cuda() for x in (k, v, table)]
    mass = evict.alloc_mass(3, hkv, table.shape[1] * 16)
    want = torch.zeros(mass.shape)
    for step in range(3):
        qs = torch.randn(3, hq * 128, generator=torch.Generator().manual_seed(step)).to(torch.bfloat16)
        was = mass.cpu()
        out = K.attn_decode(qs.cuda(), *dev, i32(lens), hq, hkv, SCALE, splits=2, mass=mass)
        check(out.cpu(), mass.cpu(), qs, k, v, table, was, lens, hq, hkv)
    want = mass.cpu()
    kept, _, count = evict.select_keys(mass, i32(lens), keep, recent=32, sink=4, update=True)
    K.kv_compact(*dev, kept, count)
    kept_c, new = kept.cpu().long(), count.tolist()
    assert new == [200, 64, 200]
    was = mass.cpu()
    out = K.attn_decode(q.cuda(), *dev, count, hq, hkv, SCALE, splits=2, mass=mass).cpu()
    for s in range(3):
        on = [kept_c[s, h, : new[s]] for h in range(hkv)]
        assert all(torch.equal(was[s, h, : new[s]], want[s, h, on[h]]) for h in range(hkv))
        kk, vv = (O.rows_of(x, table[s], lens[s], hkv) for x in (k, v))
        kk, vv = (torch.stack([x[on[h], h] for h in range(hkv)], 1) for x in (kk, vv))
        o, bound, _, _ = O.attend(q[s:s + 1, : hq * 128], kk, vv, torch.ones(1, new[s], dtype=torch.bool), hq, hkv, SCALE, W_STEP)
        O.close(out[s:s + 1], o, bound)
    assert status()["code"] == 0
