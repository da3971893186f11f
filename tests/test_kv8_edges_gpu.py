"""The 8-bit paged KV cache on a GPU at the ends of its ranges: queries with
one large dimension, the smallest and largest scales, page tables and split
counts that no engine makes."""

import math

import pytest
import torch

from infera_b200.ops import kernels as K
from infera_b200.ops import kv8
from test_kv8_gpu import (PROMPT, TOKEN, assert_close, check_decode, check_status, decode_case, i32, plain, poison,
                          random_cache)

pytestmark = pytest.mark.gpu

D = 128
DEV = "cuda"


@pytest.mark.parametrize("octaves", [7, 10, 13])
@pytest.mark.parametrize("splits", [1, 2])
def test_one_large_query_dim(octaves, splits):
    """A query element 2^octaves above the others, in a dimension that the keys are quiet in: the others count in full.
    Each of them is 1 + (8 a + 1) / 128, so 4 significant bits of it leave 1 / 128 over; without it a score of 8 to 24
    (all products are positive) is off by up to 2^-7 of itself, differently for each key, and weights by 2^-4. The
    second digit holds it exactly down to 2^-13 of the largest element, so the bounds are those of any query."""
    n, ctx, hq, hkv, scale = 40, 300, 8, 2, 0.16
    g = torch.Generator(device=DEV).manual_seed(octaves)
    _, kc, vc, bt, sl = decode_case([ctx], hq, hkv, seed=1)
    slots = kc.q.shape[0]
    k = torch.randn(slots, hkv, D, generator=g, device=DEV).abs() * 0.8 \
        * (0.5 + torch.rand(slots, hkv, 1, generator=g, device=DEV))
    k[..., 0] = 2.0 ** -9
    kc = kv8.KV8Cache(k.view(slots, -1).to(torch.float8_e4m3fn), torch.full_like(kc.sf, 127))
    vc = kv8.KV8Cache(vc.q.float().abs().to(torch.float8_e4m3fn), vc.sf)
    a = torch.randint(0, 16, (n, hq, D), generator=g, device=DEV)
    q = 1 + (8 * a + 1) / 128
    q[..., 0] = 2.0 ** octaves
    q = q.view(n, hq * D).to(torch.bfloat16)
    y = kv8.attn_prefill(q, kc, vc, bt, i32([0]), i32([n]), sl, None, hq, hkv, scale, host_meta=([n], [ctx]),
                         kv_splits=splits)
    check_status()
    assert_close(y, plain(q, kc, vc, bt[0], ctx - n + 1, hq, hkv, scale), PROMPT)
    y = kv8.attn_decode(q[:1], kc, vc, bt, sl, hq, hkv, scale, splits=splits, tiles_per_split=3)
    check_status()
    assert_close(y, plain(q[:1], kc, vc, bt[0], ctx, hq, hkv, scale), TOKEN)


def test_wide_range_of_query_elements():
    """Queries whose elements spread over 2^20, over random keys. A digit pair is off by at most 2^-21 of the row's
    largest element (2^-14 where that is 2^7 to 2^8), so a score by 2^-21 max|q| sum|k| scale, and a weight by twice
    that of itself; the rest as for any query."""
    n, ctx, hq, hkv, scale = 130, 700, 8, 2, 0.1
    g = torch.Generator(device=DEV).manual_seed(4)
    _, kc, vc, bt, sl = decode_case([ctx], hq, hkv, seed=2)
    q = torch.randn(n, hq, D, generator=g, device=DEV) / 60
    q = (q * torch.exp2(torch.randint(-20, 1, (n, hq, D), generator=g, device=DEV))).view(n, -1).to(torch.bfloat16)
    k = kc.dequant().view(-1, hkv, D).abs().sum(-1).amax()
    extra = 2 * float(2 ** -21 * q.abs().amax() * k * scale)
    assert extra < 2 ** -9
    y = kv8.attn_prefill(q, kc, vc, bt, i32([0]), i32([n]), sl, None, hq, hkv, scale, host_meta=([n], [ctx]))
    check_status()
    # weights in f16 2^-12, sums of the scores 2^-13, as in TOKEN; and the digits
    assert_close(y, plain(q, kc, vc, bt[0], ctx - n + 1, hq, hkv, scale), (2 ** -11 + extra, 2 ** -26))


@pytest.mark.parametrize("splits", [1, 3, 70])
@pytest.mark.parametrize("tps", [2 ** 28, 2 ** 30, 2 ** 31 - 1, 2 ** 33 + 1])
def test_decode_shares_of_any_size(splits, tps):
    """``splits * tiles_per_split`` has to cover the longest sequence and may be far above it, in more than 32 bits."""
    lens, hq, hkv = [300, 0, 1500], 8, 2
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=24)
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 0.1, splits=splits, tiles_per_split=tps)
    check_status()
    want = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 0.1, splits=splits, tiles_per_split=12)
    assert torch.equal(y, want)
    check_decode(lens, hq, hkv, y, q, kc, vc, bt, 0.1)


@pytest.mark.parametrize("runs", [False, True])
def test_far_page_ids_read_as_zeros(runs):
    """Page ids outside the cache, those among them whose first slot's number wraps to one of the cache (2^28 pages of 16
    slots are 2^32): zeros, alone and in runs of eight that one box would load."""
    ctx, n, hq, hkv = 700, 200, 8, 2
    q, kc, vc, bt, sl = decode_case([ctx], hq, hkv, seed=25, runs=runs)
    g = torch.Generator().manual_seed(1)
    q = (torch.randn(n, hq * D, generator=g) / 60).to(torch.bfloat16).to(DEV)
    pages = kc.sf.shape[0]
    none = bt.clone()
    swap = [slice(0, 8), slice(20, 23), slice(43, 44)] if runs else [slice(1, 4), slice(17, 18), slice(43, 44)]
    blank = [kv8.KV8Cache(torch.cat([c.q, torch.zeros_like(c.q[:16])]), torch.cat([c.sf, torch.ones_like(c.sf[:1])]))
             for c in (kc, vc)]
    for s in swap:
        none[0, s] = pages  # (the page of zeros of ``blank``)

    def both(k, v, table):
        y = kv8.attn_decode(q[:1], k, v, table, sl, hq, hkv, 0.1, splits=2, tiles_per_split=3)
        yp = kv8.attn_prefill(q, k, v, table, i32([0]), i32([n]), sl, None, hq, hkv, 0.1, host_meta=([n], [ctx]))
        check_status()
        return y, yp

    want = both(*blank, none)
    assert_close(want[0], plain(q[:1], *blank, none[0], ctx, hq, hkv, 0.1), TOKEN)
    assert_close(want[1], plain(q, *blank, none[0], ctx - n + 1, hq, hkv, 0.1), PROMPT)
    for far in (pages, -pages - 5, 2 ** 28, -2 ** 28, 2 ** 27 + 3, 2 ** 31 - 1 - pages):
        bad = bt.clone()
        for s in swap:
            bad[0, s] = (bt[0, s].long() + far).clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
        for a, b in zip(both(kc, vc, bad), want):
            assert torch.equal(a, b)


def test_largest_scales():
    """Exponents end at 253: 254 and 255 count as it, in attention and when rows join such a page."""
    hq, hkv = 4, 2
    q, kc, vc, bt, sl = decode_case([40], hq, hkv, seed=22)
    q = torch.zeros_like(q)  # all keys alike
    vq = torch.exp2(torch.randint(-9, -2, vc.q.shape, device=DEV).float()).to(torch.float8_e4m3fn)
    qkv = torch.full((2, 8 * D), 2.0 ** 120, dtype=torch.bfloat16)
    qkv[1] *= -3
    cs = K.rope_cos_sin(2, D, 1e4)
    slots = torch.tensor([int(bt[0, 0]) * 16 + 9, int(bt[0, 1]) * 16 + 3], dtype=torch.int32)
    zero = torch.zeros(2, dtype=torch.int32)
    outs, held = [], []
    for e in (253, 254, 255):
        k, v = kv8.KV8Cache(kc.q.clone(), torch.full_like(kc.sf, e)), kv8.KV8Cache(vq.clone(), torch.full_like(vc.sf, e))
        y = kv8.attn_decode(q, k, v, bt, sl, hq, hkv, 0.1)
        yp = kv8.attn_prefill(q, k, v, bt, i32([0]), i32([1]), sl, None, hq, hkv, 0.1, host_meta=([1], [40]))
        check_status()
        assert bool(y.isfinite().all()) and bool(y.any()) and bool(yp.isfinite().all()) and bool(yp.any())
        outs.append((y, yp))
        cpu = [c.to("cpu") for c in (k, v)]
        assert torch.equal(cpu[1].dequant(), kv8.KV8Cache(vq.cpu(), torch.full_like(vc.sf, 253).cpu()).dequant())
        kv8.rope_kvwrite(qkv.to(DEV), zero.to(DEV), slots.to(DEV), cs.to(DEV), hq, hkv, D, k, v)
        check_status()
        kv8.rope_kvwrite(qkv.clone(), zero, slots, cs, hq, hkv, D, *cpu)
        for x, c in ((k, cpu[0]), (v, cpu[1])):
            assert torch.equal(x.q.cpu().view(torch.uint8), c.q.view(torch.uint8))
            assert torch.equal(x.sf.cpu(), c.sf)
        rows = v.dequant().view(-1, hkv, D)[slots.long().to(DEV)]
        assert bool((rows[0] == 2.0 ** 120).all()) and bool((rows[1] == -3 * 2.0 ** 120).all())
        held.append((k, v))
    for o, h in zip(outs[1:], held[1:]):
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))
        for a, b in zip(h, held[0]):
            page = bt[0, :2].long()
            assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.sf[page], b.sf[page])


def test_largest_scales_of_whole_pages():
    """Several rows of a page at once, which another path of the append takes."""
    hkv = 2
    qkv = torch.randn(9, 8 * D, generator=torch.Generator().manual_seed(1)).mul(2.0 ** 119).to(torch.bfloat16)
    slots, pos = torch.arange(3, 12, dtype=torch.int32), torch.arange(9, dtype=torch.int32)
    cs = K.rope_cos_sin(16, D, 1e4)
    for e in (253, 254, 255):
        c = [kv8.KV8Cache(random_cache(16, hkv, 1).q, torch.full((1, hkv), e, dtype=torch.uint8, device=DEV))
             for _ in range(2)]
        cpu = [x.to("cpu") for x in c]
        kv8.rope_kvwrite(qkv.to(DEV), pos.to(DEV), slots.to(DEV), cs.to(DEV), 4, hkv, D, *c)
        check_status()
        kv8.rope_kvwrite(qkv.clone(), pos, slots, cs, 4, hkv, D, *cpu)
        for x, y in zip(c, cpu):
            assert torch.equal(x.q.cpu().view(torch.uint8), y.q.view(torch.uint8)) and torch.equal(x.sf.cpu(), y.sf)
        v = c[1].dequant()[3:12].double().cpu()
        want = qkv[:, 6 * D:].double()
        assert int(c[1].sf[0, 0]) == 253
        assert bool(((v - want).abs() <= torch.maximum(want.abs() * 2 ** -4, torch.tensor(2.0 ** 116))).all())


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("e", [1, 4, 6, 7])
def test_smallest_value_scales(e, splits):
    """Values of 2^(e-127) times a code, 2^-126 times a code at the least, are normal bf16 numbers like others. (What
    becomes smaller than 2^-126 on the way, in a share's output or in a product of the merge, may be lost: some 2^-126
    for each share.)"""
    lens, hq, hkv, scale = [300], 8, 2, 0.1
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=21)
    vc = kv8.KV8Cache(vc.q, torch.full_like(vc.sf, e))
    want = plain(q, kc, vc, bt[0], 300, hq, hkv, scale)
    want[1] += 2.0 ** -126 * 4 / TOKEN[0]
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, scale, splits=splits, tiles_per_split=3)
    check_status()
    assert_close(y, want, TOKEN)
    y = kv8.attn_prefill(q, kc, vc, bt, i32([0]), i32([1]), sl, None, hq, hkv, scale, host_meta=([1], lens),
                         kv_splits=splits)
    check_status()
    assert_close(y, want, PROMPT)


def test_decode_split_counts_its_own_pages():
    """A split's weights are held against the largest V scale of its own pages: keys of the next split whose values are
    2^30 times as large, and whose weights are nothing, cost the first split's output no digit."""
    hq, hkv, mine, n = 8, 2, 256, 512
    q, kc, vc, bt, sl = decode_case([n], hq, hkv, seed=23, spread=1)
    q = torch.zeros_like(q).view(1, hq, D)
    q[..., 0] = 1.0
    q = q.view(1, -1)
    far = bt[0, mine // 16:].long()
    codes = kc.q.view(torch.uint8).view(-1, 16, hkv, D)
    codes.zero_()
    codes[far, :, :, 0] = 0xFE  # -448
    vc.sf[far] += 30
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 1.0, splits=2, tiles_per_split=2)
    check_status()
    # e^-448 of a value below 2^46 is nothing beside the first split's
    assert_close(y, plain(q, kc, vc, bt[0], mine, hq, hkv, 1.0), TOKEN)


@pytest.mark.parametrize("splits", [1, 3])
def test_attention_in_place(splits):
    """The output may be the queries' own memory."""
    hq, hkv, lens = 32, 8, [700, 0, 300]
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=26)
    args = (kc, vc, bt, sl, hq, hkv, 0.1)
    want = kv8.attn_decode(q, *args, splits=splits, tiles_per_split=6)
    mine = q.clone()
    kv8.attn_decode(mine, *args, splits=splits, tiles_per_split=6, out=mine)
    assert torch.equal(mine, want)
    n = [600, 0, 7]
    q = (torch.randn(sum(n), hq * D, generator=torch.Generator().manual_seed(2)) / 60).to(torch.bfloat16).to(DEV)
    args = (kc, vc, bt, i32([0, 600, 600]), i32(n), sl, None, hq, hkv, 0.1)
    want = kv8.attn_prefill(q, *args, host_meta=(n, lens), kv_splits=splits)
    kv8.attn_prefill(q, *args, host_meta=(n, lens), kv_splits=splits, out=q)
    assert torch.equal(q, want)
    check_status()


def test_engine_holds_no_decode_workspace(monkeypatch):
    """8-bit attention's partials are each call's own: an engine with this cache sizes no bf16 decode workspace."""
    from infera_b200.engine.llm_engine import EngineConfig, LLMEngine
    from infera_b200.engine.request import SamplingParams

    def never(self, o_numel, lse_numel):
        raise AssertionError(f"a decode workspace of {o_numel} + {lse_numel} elements")

    monkeypatch.setattr(K.DeviceScratch, "ensure_decode", never)
    eng = LLMEngine(EngineConfig(model="tiny-dense-gpu", kv_cache_dtype="fp8", num_pages=64, max_num_seqs=4,
                                 max_batched_tokens=96), device="cuda:0")
    outs = eng.generate([[5, 6, 7], list(range(2, 150))], SamplingParams(max_tokens=5, ignore_eos=True))
    check_status()
    assert [len(o) for o in outs] == [5, 5]


@pytest.mark.parametrize("ql,ctx", [([17], [4113]), ([300], [300]), ([1], [2000]), ([3], [8100]),
                                    ([17, 256, 1, 300, 5], [17, 700, 90, 301, 1500]), ([20, 0, 40], [50, 0, 40])])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 8), (32, 8)])
def test_prefill_reads_its_lengths_back(ql, ctx, hq, hkv):
    """Without host lengths the call reads them from the device and makes the same plan: the same bits, in a wider buffer
    too, whose other columns and rows stay as they are."""
    g = torch.Generator().manual_seed(hq)
    _, kc, vc, bt, sl = decode_case(ctx, hq, hkv, seed=hq)
    poison(kc, vc, bt, ctx)
    T = sum(ql)
    q = (torch.randn(T, hq * D, generator=g) / 60).to(torch.bfloat16).to(DEV)
    start = [sum(ql[:i]) for i in range(len(ql))]
    args = (q, kc, vc, bt, i32(start), i32(ql), sl, None, hq, hkv, 0.1)
    y = kv8.attn_prefill(*args, host_meta=(ql, ctx))
    out = torch.full((T + 2, hq * D + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    kv8.attn_prefill(*args, out=out)
    check_status()
    assert torch.equal(out[:T, : hq * D], y) and bool((out[T:] == 3).all()) and bool((out[:, hq * D:] == 3).all())


@pytest.mark.parametrize("lens", [[8192, 8192], [8192, 100, 4097, 1], [1000] * 8])
@pytest.mark.parametrize("hq,hkv", [(64, 8), (10, 2), (8, 1)])
def test_decode_as_planned_for_more_than_four_heads(lens, hq, hkv):
    """The splits that an engine takes for five to eight query heads to a KV head: one wave of two CTAs per SM."""
    q, kc, vc, bt, sl = decode_case(lens, hq, hkv, seed=hq + len(lens))
    splits, tps = kv8.decode_plan(len(lens), hkv, max(lens), group=hq // hkv)
    assert splits == 1 or splits * len(lens) * hkv <= 2 * 148
    y = kv8.attn_decode(q, kc, vc, bt, sl, hq, hkv, 1 / math.sqrt(D), splits=splits, tiles_per_split=tps)
    check_status()
    for b, n in enumerate(lens):
        assert_close(y[b:b + 1], plain(q[b:b + 1], kc, vc, bt[b], n, hq, hkv, 1 / math.sqrt(D)), TOKEN)


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("model,over", [("tiny-dense-gpu", {"qk_norm": True}), ("tiny-moe-gqa-gpu", {})])
def test_models(model, over, graphs):
    """Models with q / k norms and with routed experts over an 8-bit cache: the first layer's K and V depend on tokens
    and positions alone. An element is off by half a step of e4m3 (2^-4 of it; 2^-10 of the scale below the normals,
    and the scale is at most 2^-7 of its page's largest element; once more where a page's scale grew), and by a step of
    bf16 where the two engines' products round differently."""
    from infera_b200.engine.llm_engine import EngineConfig, LLMEngine
    from infera_b200.engine.request import SamplingParams

    g = torch.Generator().manual_seed(3)
    ask = [torch.randint(2, 4096, (n,), generator=g).tolist() for n in (40, 300, 33)]
    got = []
    for kv in ("fp8", "bf16"):
        e = LLMEngine(EngineConfig(model=model, kv_cache_dtype=kv, num_pages=64, max_batched_tokens=96, max_num_seqs=4,
                                   use_cuda_graphs=graphs, model_overrides=dict(over)), device="cuda:0")
        e.generate(ask, SamplingParams(max_tokens=1, ignore_eos=True))
        check_status()
        k, v = e.runner.k_cache, e.runner.v_cache
        got.append((k[0].dequant(), v[0].dequant()) if kv == "fp8" else (k[0].float(), v[0].float()))
        if kv == "fp8":
            got[0] = tuple(t.clone() for t in got[0])
            outs = e.generate([p + [5, 6] for p in ask], SamplingParams(max_tokens=12, ignore_eos=True))
            check_status()
            assert [len(o) for o in outs] == [12, 12, 12]
    for x, y in zip(*got):
        used = y.abs().sum(-1) > 0
        assert int(used.sum()) >= 320 and torch.equal(used, x.abs().sum(-1) > 0)
        page = y.view(-1, 16, 2, D).abs().amax(dim=(1, 3))[:, None, :, None].expand(-1, 16, 2, D).reshape(y.shape)
        assert bool(((x - y).abs() <= y.abs() * (2 ** -4 + 2 ** -7) + (2 * 2 ** -10 * 2 ** -7 + 2 ** -20) * page).all())
