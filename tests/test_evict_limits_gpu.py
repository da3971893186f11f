"""Decode attention with accumulated weights and moves of rows at the ends of their ranges on the GPU."""

import math

import paged_oracle as O
import pytest
import torch
from test_evict_gpu import W_STEP, batch, check, i32, status

from infera_b200.ops import evict
from infera_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)


@pytest.mark.parametrize("hq", [1, 4, 8])
def test_values_near_the_largest(hq):
    """Sums of weighted values stay in range, however far the maximum lags and in however many shares a sequence is cut."""
    lens = [1500, 40]
    q, k, v, table, mass = batch(lens, hq, 1, 3)
    for s, n in enumerate(lens):
        for p in range(n):  # scores that grow by some 6 in log2 from tile to tile, under the lag
            at = int(table[s, p // 16]) * 16 + p % 16
            k[at, 0] = p / 128
            v[at, 20] = 3.3e38
            v[at, 21] = -3.3e38 if p % 3 else 3.3e38
            v[at, 22] = 3.3e38 if p % 50 == 7 else 1.0
    for h in range(hq):
        q[:, 128 * h] = 48
    for splits, tps in ((1, 0), (2, 0), (12, 1)):
        got = mass.cuda()
        out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, 1, SCALE, got, splits,
                                tiles_per_split=tps)
        check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, 1)
    assert status()["code"] == 0


@pytest.mark.parametrize("heads,layers,m", [(1, 3, 9), (2, 1, 70), (1, 2, 100)])
def test_a_table_row_named_twice_moves_once(heads, layers, m):
    """By the first sequence that names it, whether that one's rows move or its start is refused."""
    g = torch.Generator().manual_seed(m)
    table, pool = O.page_table([300, 200], 5)
    k, v = (torch.randn(layers, pool * 16, 256, generator=g).to(torch.bfloat16) for _ in range(2))
    src = torch.stack([torch.randperm(150, generator=g)[:m].sort().values for _ in range(4 * heads)]).to(torch.int32)
    src = src.view(4, heads, m) if heads > 1 else src
    for start in ([0, 7, 3, 11], [-1, 7, 3, 11]):
        want = [k, v]
        for s, row in ((0, 0), (1, 1)):  # (the third and fourth come after them)
            for h in range(heads):
                if start[s] >= 0:
                    w = 256 // heads
                    want = [O.moved(x, table[row], src.view(4, heads, m)[s, h].tolist(), start[s], w, h * w) for x in want]
        for dev in ("cuda", "cpu"):
            kc, vc = (x.clone().to(dev) for x in (k, v))
            K.kv_compact(kc, vc, table.to(dev), src.to(dev), torch.full((4,), m, dtype=torch.int32, device=dev),
                         start=torch.tensor(start, dtype=torch.int32, device=dev),
                         bt_rows=torch.tensor([0, 1, 0, 1], dtype=torch.int32, device=dev))
            assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1]), dev
        assert status()["code"] == 7


def test_fewer_places_in_the_mass_than_keys():
    """Weights of places that the mass has are added, up to its end and not into the next row; the output is whole."""
    lens, hq, hkv = [100, 300, 60, 151], 8, 2
    q, k, v, table, mass = batch(lens, hq, hkv, 4)
    for splits, tps in ((1, 0), (2, 0), (3, 1)):
        got = mass[:, :, :150].contiguous().cuda()
        out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, hkv, SCALE, got, splits,
                                tiles_per_split=tps).cpu()
        assert status()["code"] == 7
        for b, n in enumerate(lens):
            kk, vv = (O.rows_of(x, table[b], n, hkv) for x in (k, v))
            want, bound, w, wb = O.attend(q[b:b + 1, : hq * 128], kk, vv, torch.ones(1, n, dtype=torch.bool), hq, hkv, SCALE, W_STEP)
            O.close(out[b:b + 1], want, bound)
            cut = min(n, 150)
            was = mass[b, :, :150].double()
            bound_m = 2.0 ** -23 * was + 1e-37
            was[:, :cut] += w[0].view(hkv, -1, n).sum(1)[:, :cut]
            bound_m[:, :cut] += (wb + 2.0 ** -20 * w)[0].view(hkv, -1, n).sum(1)[:, :cut]
            O.close(got[b], was, bound_m, f"mass {b}")


@pytest.mark.parametrize("splits", [1, 2, 3])
def test_a_length_beyond_the_table_is_cut(splits):
    lens, hq, hkv = [100, 304, 60], 4, 1
    q, k, v, table, mass = batch(lens, hq, hkv, 4)
    got = mass.cuda()
    out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32([100, 5000, 60]), hq, hkv, SCALE, got, splits)
    assert status()["code"] == 7
    check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, hkv)


@pytest.mark.parametrize("plan", ["plan", (1, 0), (235, 1)])
def test_long_contexts_of_many_shares(plan):
    lens, hq, hkv = [30011, 9001], 4, 1
    q, k, v, table, mass = batch(lens, hq, hkv, 9)
    splits, tps = evict.decode_plan(2, hkv, max(lens)) if plan == "plan" else plan
    got = mass.cuda()
    out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, hkv, SCALE, got, splits,
                            tiles_per_split=tps)
    assert status()["code"] == 0
    check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, hkv)


def test_a_padded_batch():
    """Sequences of length 0 that pad a batch share one row of the table: a captured eviction step over them reports nothing
    and leaves the row, and what the others do, alone."""
    lens, hq, hkv, keep = [200, 90, 150, 64], 4, 2, 60
    q, k, v, table, mass = batch(lens, hq, hkv, 6)
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    rows = [2, 0, 1, 3, 3, 3]
    now = [lens[2], lens[0], lens[1], 0, 0, 0]
    qp = torch.cat([q[rows[:3]], q[:3]])
    dev = [qp.cuda(), k.cuda(), v.cuda(), table.cuda()]
    got, lens_d, rows_d = mass.cuda(), i32(now), i32(rows)
    start = i32([0] * 6)

    def step():
        out = evict.attn_decode(*dev, lens_d, hq, hkv, SCALE, got, 2, bt_rows=rows_d)
        kept, _, count = evict.select_keys(got, lens_d, keep, recent=8, sink=2, bt_rows=rows_d, update=True)
        K.kv_compact(dev[1], dev[2], dev[3], kept, count, start=start, bt_rows=rows_d)  # each KV head's columns by a list
        K.kv_compact(dev[1], dev[2], dev[3], whole, moved, start=start, bt_rows=rows_d)  # whole rows
        return out, kept, count

    whole, moved = i32([[3, 9]] * 6), i32([0] * 6)
    step()
    assert status()["code"] == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, kept, count = step()
    for x, y in zip((dev[1], dev[2], got), (k, v, mass)):
        x.copy_(y)
    graph.replay()
    assert status()["code"] == 0 and count.tolist() == [60, 60, 60, 0, 0, 0] and torch.all(kept[3:] == -1)
    assert torch.all(out[3:] == 0) and torch.equal(got[3].cpu(), mass[3])
    want_k, want_v = k, v
    for s in range(3):
        n, row = now[s], rows[s]
        kk, vv = (O.rows_of(x, table[row], n, hkv) for x in (k, v))
        want, bound, w, wb = O.attend(qp[s:s + 1, : hq * 128], kk, vv, torch.ones(1, n, dtype=torch.bool), hq, hkv, SCALE, W_STEP)
        O.close(out[s:s + 1], want, bound)
        was = mass[row, :, :n].double()
        full = was + w[0].view(hkv, -1, n).sum(1)
        bound_m = 2.0 ** -23 * was + (wb + 2.0 ** -20 * w)[0].view(hkv, -1, n).sum(1)
        for h in range(hkv):
            on = kept[s, h].tolist()
            assert on[:2] == [0, 1] and on[-8:] == list(range(n - 8, n)) and on == sorted(set(on))
            O.close(got[row, h, :60], full[h, on], bound_m[h, on])
            assert torch.all(got[row, h, 60:n] == 0)
            want_k, want_v = (O.moved(x, table[row], on, 0, 128, 128 * h) for x in (want_k, want_v))
    assert torch.equal(dev[1].cpu(), want_k) and torch.equal(dev[2].cpu(), want_v)


@pytest.mark.parametrize("hq", [1, 2, 4, 8, 3])
def test_infinite_values(hq):
    """An infinity among the values is the output's, of both signs a NaN, whatever the weight's digits are."""
    lens = [700, 300, 129]
    q, k, v, table, mass = batch(lens, hq, 1, 8)
    slot = lambda s, p: int(table[s, p // 16]) * 16 + p % 16  # noqa: E731
    inf = float("inf")
    for s, p, d, x in ((0, 3, 5, inf), (0, 650, 5, inf), (0, 130, 7, -inf), (0, 131, 9, inf), (0, 500, 9, -inf), (0, 699, 127, inf),
                       (1, 0, 0, -inf), (1, 299, 64, inf), (1, 150, 65, float("nan")), (2, 128, 66, inf), (2, 5, 67, 3e38)):
        v[slot(s, p), d] = x
    for splits, tps in ((1, 0), (2, 0), (6, 1)):
        got = mass.cuda()
        out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, 1, SCALE, got, splits,
                                tiles_per_split=tps)
        check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, 1)
    # a share far below the others in weight
    for p in range(600, 700):
        k[slot(0, p), 0] = 300
    for h in range(hq):
        q[:, 128 * h] = 8
    for splits, tps in ((1, 0), (2, 0), (6, 1)):
        got = mass.cuda()
        out = evict.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lens), hq, 1, SCALE, got, splits,
                                tiles_per_split=tps)
        check(out.cpu(), got.cpu(), q, k, v, table, mass, lens, hq, 1)
    assert status()["code"] == 0
