// Attention of drafted tokens that form a tree (speculative decoding) over the
// bf16 paged KV cache, on tcgen05. A sequence's last q_len keys are its nodes;
// node i sees the keys before them and node j where bit j of its mask is set.
//
//   S = Q K^T, O += W V,  w = 2^(c s - m) in bf16 (rounded, 2^-9 of itself, as
//   the prompt kernel's), the sum of the softmax over the fp32 weights
//
// The query heads of a KV head are packed: rows are (node, head) pairs. Tiles
// of 128 keys pass through shared memory once for 256 rows. Two softmax groups
// of 128 threads, a row each, with accumulators of their own in TMEM:
//   more than 128 rows   two query tiles, one a group, over every key tile
//                        (the tensor core works on one while the other's
//                        softmax runs)
//   up to 128 rows       one query tile; the groups take every other key tile
//                        and are joined at the end through shared memory, so
//                        the scores of a key tile are made while the softmax of
//                        the one before runs
//   warp 0       TMA producer: lane 0 K tiles, lane 1 V tiles
//   warp 1       MMA issuer
//   warps 2..9   the softmax groups; they also stage Q
// The weights of 64 keys lie over their scores in TMEM.
//
// Masks are looked at only in the tiles that hold nodes (the last ones). There
// the values' infinities and NaN are multiplied as zeros (a weight of zero does
// not cancel them) and written at the end to the rows that see them, and V rows
// behind the sequence, which a recycled page may have left as NaN, are zeroed.
//
// A CTA takes up to 256 rows of a (sequence, KV head) and a share of its key
// tiles, the same number for every sequence, so ragged batches stay balanced;
// rows with more than one share are merged by a second kernel.
#include <algorithm>

#include "kv8.cuh"
#include "tma_host.h"

namespace ib200 {
namespace atree {

using kv8::elect_one;
using kv8::known_pages;
using kv8::table_row;
using kv8::umma_bf16_if;
using kv8::umma_commit_if;
using kv8::umma_f16_ts_if;
using kv8::uniform;

constexpr int D = 128;
constexpr int PAGE = 16;
constexpr int BQ = 128;               // rows of a query tile
constexpr int BKV = 128;
constexpr int BLK = 128 * 128;        // bytes of 128 rows x 64 bf16
constexpr int KST = 3, VST = 2;       // stages of K tiles and of V tiles
constexpr int NUM_THREADS = 320;
constexpr int SMEM_BYTES = 1024 + (4 + 2 * KST + 2 * VST) * BLK + 2048;
constexpr int UNIT = 64;              // keys of a step of the softmax
constexpr uint32_t O_COL = 256;       // S0 (W0 over each unit's columns) [0,128) S1 [128,256) O0 O1
constexpr float kLagLog2 = 8.0f;      // the running maximum may lag by this much

struct Params {
  const __nv_bfloat16* q;
  int ldq;
  int T;                   // rows of q, mask and out
  const int* q_start;
  const int* q_len;
  const int* ctx_len;
  const int* mask;         // [T, words]
  int words;
  const __nv_bfloat16* v;
  int num_pages;
  const int* block_table;
  const int* bt_rows;
  int table_rows, max_pages, ld_table;
  int hq, hkv, G, tokens;  // tokens: of an item, 256 / G
  int blocks;              // items of the longest tree
  int splits, tiles_per_split;
  float c;                 // |scale| * log2(e)
  uint32_t q_flip, q_keep;
  float* o_part;           // [T, hq, splits, 128]
  float* lse_part;         // [T, hq, splits]
  __nv_bfloat16* out;
  int ldo;
  int* status;
};

// What both kernels know of a sequence. `tps` tiles are a share's, so that the
// shares cover it; `shares` of them have keys.
struct Seq {
  int start, n, ctx, base, tps, shares;  // base: its keys before the nodes
  const int* bt;
};
__device__ __forceinline__ Seq sequence(const Params& p, int s, int* status) {
  Seq q;
  q.start = p.q_start[s];
  const int want = max(p.q_len[s], 0);
  const int cover = min(p.blocks * p.tokens, 32 * p.words);
  q.n = min(want, cover);
  if (q.start < 0 || q.start > p.T) q.n = 0;
  q.n = min(q.n, p.T - q.start);
  q.ctx = max(p.ctx_len[s], 0);
  q.base = q.ctx - want;  // (may be negative: nodes without a key)
  q.bt = table_row(p.block_table, p.bt_rows != nullptr ? p.bt_rows[s] : s, p.table_rows, p.ld_table, s, status);
  if (q.bt == nullptr) q.ctx = 0;
  if (threadIdx.x == 0) {
    if (q.n < want) record_status_detail(status, kStatusBadIndex, 9, s, want);
    if (q.ctx > p.max_pages * PAGE) record_status_detail(status, kStatusBadIndex, 1, s, q.ctx);
  }
  q.ctx = min(q.ctx, p.max_pages * PAGE);
  const int tiles = (q.ctx + BKV - 1) / BKV;
  q.tps = max(p.tiles_per_split, (tiles + p.splits - 1) / p.splits);
  q.shares = (tiles + q.tps - 1) / q.tps;
  return q;
}

__device__ __forceinline__ uint64_t f2pack(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void f2unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Which of the 64 keys from key `k` on a row sees: those before the nodes, and
// node j where bit j of its mask is set.
__device__ __forceinline__ uint64_t seen_of(const int* mask, int words, int k, int base, int ctx) {
  if (ctx <= k) return 0;
  const uint64_t there = ctx - k >= 64 ? ~0ull : (1ull << (ctx - k)) - 1;
  const int off = k - base;  // the node at key k
  if (off <= -64) return there;
  uint64_t bits;
  if (off >= 0) {
    const int w = off >> 5, sh = off & 31;
    const uint32_t a = w < words ? mask[w] : 0, b = w + 1 < words ? mask[w + 1] : 0, c = w + 2 < words ? mask[w + 2] : 0;
    bits = static_cast<uint64_t>(__funnelshift_r(a, b, sh)) | static_cast<uint64_t>(__funnelshift_r(b, c, sh)) << 32;
  } else {
    const uint64_t low = static_cast<uint32_t>(mask[0]) | (words > 1 ? static_cast<uint64_t>(static_cast<uint32_t>(mask[1])) << 32 : 0);
    bits = low << -off | ((1ull << -off) - 1);
  }
  return bits & there;
}

// Writes what is not finite among the values of a CTA's nodes to the rows that
// see it, a warp per node. Rare, so nothing here is tuned.
__device__ __noinline__ void write_not_finite(const Params& p, const Seq& sq, int first, int n, int kvh, int z, int k_lo,
                                              int k_hi) {
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n; i += NUM_THREADS / 32) {
    const int row = sq.start + first + i;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};  // of dims 4 lane .. 4 lane + 3: an infinity, a NaN, or 0
    for (int k = max(k_lo, max(sq.base, 0)); k < min(k_hi, sq.ctx); ++k) {
      const int j = k - sq.base, page = sq.bt[k / PAGE];
      if (j >= 32 * p.words || (p.mask[static_cast<size_t>(row) * p.words + (j >> 5)] >> (j & 31) & 1) == 0) continue;
      if (page < 0 || page >= p.num_pages) continue;
      const uint2 u = *reinterpret_cast<const uint2*>(
          p.v + ((static_cast<size_t>(page) * PAGE + k % PAGE) * p.hkv + kvh) * D + 4 * lane);
      const float x[4] = {bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y)};
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (!(fabsf(x[d]) <= 3.4e38f)) sum[d] += x[d];
    }
    for (int g = 0; g < p.G; ++g)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if (sum[d] == 0.f) continue;
        const int head = kvh * p.G + g;
        if (sq.shares > 1)
          p.o_part[((static_cast<size_t>(row) * p.hq + head) * p.splits + z) * D + 4 * lane + d] = sum[d];
        else
          p.out[static_cast<size_t>(row) * p.ldo + head * D + 4 * lane + d] = __float2bfloat16(sum[d]);
      }
  }
}

// ONE: up to 128 rows, whose key tiles the two groups share.
template <bool ONE>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    tree_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ CUtensorMap tmK8, const __grid_constant__ CUtensorMap tmV8,
                const __grid_constant__ Params p) {
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.x, seq = blockIdx.y, G = p.G;
  const int block = blockIdx.z % p.blocks, z = blockIdx.z / p.blocks;
  const Seq sq = sequence(p, seq, p.status);
  const int first = block * p.tokens;                 // the item's first node
  const int n_nodes = min(p.tokens, sq.n - first);
  if (n_nodes <= 0) return;
  const int n_rows = n_nodes * G;
  const int j_lo = z * sq.tps;
  const int nk = min((sq.ctx + BKV - 1) / BKV - j_lo, sq.tps);  // key tiles of this share
  if (nk <= 0) {
    if (z == 0)  // no keys at all
      for (int i = threadIdx.x; i < n_rows * (D / 8); i += NUM_THREADS) {
        const int row = sq.start + first + i / (D / 8) / G, head = kvh * G + i / (D / 8) % G;
        reinterpret_cast<uint4*>(p.out + static_cast<size_t>(row) * p.ldo + head * D)[i % (D / 8)] = make_uint4(0u, 0u, 0u, 0u);
      }
    return;
  }
  // key tiles of the two groups
  const int rows1 = ONE ? n_rows : max(0, n_rows - BQ);
  const int nt0 = ONE ? (nk + 1) / 2 : nk, nt1 = ONE ? nk / 2 : (rows1 > 0 ? nk : 0);
  const int n_pages = (sq.ctx + PAGE - 1) / PAGE;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                    // tile t: dims 0..63, dims 64..127
  uint8_t* sK = sQ + 4 * BLK;            // [KST] dims 0..63, dims 64..127
  uint8_t* sV = sK + 2 * KST * BLK;      // [VST]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * VST * BLK);
  uint64_t* q_ready = bars;
  uint64_t* k_full = bars + 1;           // [KST]
  uint64_t* k_empty = k_full + KST;      // [KST]
  uint64_t* v_full = k_empty + KST;      // [VST]
  uint64_t* v_empty = v_full + VST;      // [VST]
  uint64_t* s_full = v_empty + VST;      // [2 groups]
  uint64_t* p_full = s_full + 2;         // [2 groups][2 units]
  uint64_t* o_done = p_full + 4;         // [2][2]: a phase of [t][0] per first unit's W V; [t][1]: the last one's
  uint64_t* joined = o_done + 4;         // ONE: the second group's part is in shared memory
  uint64_t* drain = joined + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* not_finite = abort_flag + 1;
  float2* s_ml = reinterpret_cast<float2*>(tmem_slot + 4);  // ONE: [128] maximum and sum of the second group

  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_ready, 256);
    for (int s = 0; s < KST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) mbar_init(&s_full[t], 1);
    for (int s = 0; s < 4; ++s) {
      mbar_init(&p_full[s], 128);
      mbar_init(&o_done[s], 1);
    }
    mbar_init(joined, 128);
    mbar_init(drain, 1);
    *abort_flag = 0;
    *not_finite = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmK8);
    tma_prefetch_desc(&tmV8);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  if (warp == 0) {
    if (lane < 2) {
      const bool is_v = lane == 1;
      const int stages = is_v ? VST : KST;
      const CUtensorMap* tm1 = is_v ? &tmV : &tmK;
      const CUtensorMap* tm8 = is_v ? &tmV8 : &tmK8;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      uint8_t* dst0 = is_v ? sV : sK;
      // another item of the sequence reads these keys too, or none
      const uint64_t pol = p.blocks > 1 ? policy_evict_last() : policy_evict_first();
      int issued = 0, st = 0, ph = 1;
      int nxt[8];
      load_tile_pages(sq.bt, j_lo, n_pages, nxt);
      for (int j = 0; j < nk; ++j) {
        int cur[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cur[i] = nxt[i];
        known_pages(cur, p.num_pages);
        if (j + 1 < nk) load_tile_pages(sq.bt, j_lo + j + 1, n_pages, nxt);
        if (!mbar_wait(&empty[st], static_cast<uint32_t>(ph), abort_flag, p.status, kStatusTimeoutEmpty)) break;
        uint8_t* dst = dst0 + st * 2 * BLK;
        bool run = true;
#pragma unroll
        for (int pg = 1; pg < BKV / PAGE; ++pg) run = run && cur[pg] == cur[0] + pg;
        const int n = min(BKV / PAGE, n_pages - (j_lo + j) * (BKV / PAGE));  // pages that the sequence has here
        mbar_expect_tx(&full[st], 2 * n * PAGE * 128);
        if (run && n == BKV / PAGE) {
          tma_load_2d(dst, tm8, &full[st], kvh * D, cur[0] * PAGE, pol);
          tma_load_2d(dst + BLK, tm8, &full[st], kvh * D + 64, cur[0] * PAGE, pol);
        } else {
#pragma unroll
          for (int pg = 0; pg < BKV / PAGE; ++pg)
            if (pg < n) {
              tma_load_2d(dst + pg * PAGE * 128, tm1, &full[st], kvh * D, cur[pg] * PAGE, pol);
              tma_load_2d(dst + BLK + pg * PAGE * 128, tm1, &full[st], kvh * D + 64, cur[pg] * PAGE, pol);
            }
        }
        ++issued;
        if (++st == stages) {
          st = 0;
          ph ^= 1;
        }
      }
      for (int i = max(0, issued - stages); i < issued; ++i)
        mbar_wait(&full[i % stages], static_cast<uint32_t>((i / stages) & 1), nullptr, nullptr, 0, kWaitLimitNs / 4);
    }
  } else if (warp == 1) {
    const uint32_t on = elect_one();
    const uint32_t idesc_s = make_idesc_bf16(128, BKV);
    const uint32_t idesc_o = make_idesc_bf16(128, D, true);  // B = V with adjacent dims (MN-major)
    const uint64_t q_desc = make_sw128_desc(smem_u32(sQ), 16, 1024);
    const uint64_t k_desc = make_sw128_desc(smem_u32(sK), 16, 1024);
    const uint64_t v_desc = make_sw128_desc(smem_u32(sV), BLK, 1024);
    const int n1 = uniform(nt1);
    bool ok = mbar_wait_warp(q_ready, 0, abort_flag, p.status, kStatusTimeoutFull);
    // (descriptor addresses are in units of 16 bytes)
    auto wait_k = [&](int j) {
      ok = ok && mbar_wait_warp(&k_full[j % KST], static_cast<uint32_t>((j / KST) & 1), abort_flag, p.status,
                                kStatusTimeoutFull);
    };
    auto wait_v = [&](int j) {
      ok = ok && mbar_wait_warp(&v_full[j % VST], static_cast<uint32_t>((j / VST) & 1), abort_flag, p.status,
                                kStatusTimeoutFull);
    };
    auto scores = [&](int j, int t) {  // S_t of key tile j
      tc_fence_after();
      const uint64_t kd = k_desc + (j % KST) * (2 * BLK / 16), qd = q_desc + (ONE ? 0 : t) * (2 * BLK / 16);
#pragma unroll
      for (int s = 0; s < 8; ++s)
        umma_bf16_if(on, tmem + t * 128, qd + ((s >> 2) * BLK + (s & 3) * 32) / 16, kd + ((s >> 2) * BLK + (s & 3) * 32) / 16,
                     idesc_s, s > 0 ? 1u : 0u);
      umma_commit_if(on, &s_full[t]);
    };
    auto values = [&](int j, int t, int jt, bool end) {  // O_t += W_t V of key tile j, the group's jt-th
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!ok) break;
        ok = mbar_wait_warp(&p_full[t * 2 + half], static_cast<uint32_t>(jt & 1), abort_flag, p.status,
                            kStatusTimeoutTmemEmpty);
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = v_desc + (j % VST) * (2 * BLK / 16);
#pragma unroll
        for (int s = 0; s < 4; ++s)
          // W_t packs keys 16s .. 16s + 15 of the unit into columns 8s .. 8s + 7 of its S
          umma_f16_ts_if(on, tmem + O_COL + t * 128, tmem + t * 128 + half * UNIT + s * 8,
                         vd + (half * UNIT * 128 + s * 2048) / 16, idesc_o, (jt > 0 || half > 0 || s > 0) ? 1u : 0u);
        if (half == 0 || end) umma_commit_if(on, &o_done[t * 2 + half]);
      }
    };
    if constexpr (ONE) {
      for (int j = 0; j <= nk && ok; ++j) {
        if (j < nk) {
          wait_k(j);
          if (!ok) break;
          scores(j, j & 1);
          umma_commit_if(on, &k_empty[j % KST]);
        }
        if (j > 0) {
          wait_v(j - 1);
          values(j - 1, (j - 1) & 1, (j - 1) >> 1, j + 1 >= nk);
          if (!ok) break;
          umma_commit_if(on, &v_empty[(j - 1) % VST]);
        }
      }
    } else {
      for (int j = -1; j < nk && ok; ++j) {
        if (j + 1 < nk) wait_k(j + 1);
        if (j >= 0) wait_v(j);
        if (!ok) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (t == 1 && n1 == 0) break;
          if (j >= 0) values(j, t, j, j + 1 == nk);
          if (j + 1 < nk && ok) scores(j + 1, t);
        }
        if (!ok) break;
        if (j + 1 < nk) umma_commit_if(on, &k_empty[(j + 1) % KST]);
        if (j >= 0) umma_commit_if(on, &v_empty[j % VST]);
      }
    }
    umma_commit_if(on, drain);
    mbar_wait_warp(drain, 0, nullptr, p.status, kStatusTimeoutFull);
  } else {
    const int t = (warp - 2) >> 2;
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const int pr = (ONE ? 0 : t * BQ) + r;               // the row, and whether it exists
    const bool live = pr < n_rows;
    const int node = first + (live ? pr / G : 0), head = kvh * G + (live ? pr % G : 0);
    const int row = sq.start + node;
    const int nt = t ? nt1 : nt0;
    // stage this row (rows that do not exist are zero)
    if (!ONE || t == 0) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + static_cast<size_t>(row) * p.ldq + head * D);
      uint4 v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = live ? src[i] : make_uint4(0u, 0u, 0u, 0u);
      uint8_t* dst = sQ + t * 2 * BLK;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] = make_uint4((v[i].x ^ p.q_flip) & p.q_keep, (v[i].y ^ p.q_flip) & p.q_keep, (v[i].z ^ p.q_flip) & p.q_keep,
                          (v[i].w ^ p.q_flip) & p.q_keep);
        *reinterpret_cast<uint4*>(dst + (i >> 3) * BLK + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = v[i];
      }
      fence_proxy_async_smem();
    }
    mbar_arrive(q_ready);
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    const uint32_t o_addr = lane_addr + O_COL + t * 128;
    const int* mask = p.mask + static_cast<size_t>(row) * p.words;
    const bool awake = __any_sync(0xffffffffu, live);    // a warp without rows only keeps step
    float m_run = -INFINITY;
    float l_run = 0.f;
    bool ok = true;
    // the jt-th key tile of the group
    for (int jt = 0; jt < nt && ok; ++jt) {
      const int j = ONE ? 2 * jt + t : jt;
      const int k0 = (j_lo + j) * BKV;
      const bool edge = k0 + BKV > sq.base;              // the tile has nodes, or ends behind the sequence
      if (!mbar_wait_warp(&s_full[t], static_cast<uint32_t>(jt & 1), abort_flag, p.status, kStatusTimeoutTmemFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (edge && (ONE || t == 0)) {
        // V row r of the tile: zeroed behind the sequence, and where a node's is not finite. (S of this tile was
        // issued after the W V that freed the stage: the barrier is in this tile's phase or past it.)
        if (!mbar_wait_warp(&v_full[j % VST], static_cast<uint32_t>((j / VST) & 1), abort_flag, p.status,
                            kStatusTimeoutFull)) {
          ok = false;
          break;
        }
        const int key = k0 + r;
        uint8_t* src = sV + (j % VST) * 2 * BLK + r * 128;
        if (key >= sq.ctx) {
#pragma unroll
          for (int i = 0; i < 16; ++i) *reinterpret_cast<uint4*>(src + (i >> 3) * BLK + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        } else if (key >= sq.base) {
#pragma unroll 4
          for (int i = 0; i < 16; ++i) {
            uint4* at = reinterpret_cast<uint4*>(src + (i >> 3) * BLK + (((i & 7) ^ (r & 7)) << 4));
            uint32_t u[4] = {at->x, at->y, at->z, at->w};
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((u[k] & 0x7f80u) == 0x7f80u) u[k] &= 0xffff0000u, bad = true;
              if ((u[k] & 0x7f800000u) == 0x7f800000u) u[k] &= 0xffffu, bad = true;
            }
            if (bad) {
              *at = make_uint4(u[0], u[1], u[2], u[3]);
              *not_finite = 1;
            }
          }
        }
        fence_proxy_async_smem();
      }
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int u = 2 * jt + half;
        if (awake) {
          const uint32_t s_addr = lane_addr + t * 128 + half * UNIT;
          uint32_t v[UNIT];
          tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
          tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
          tmem_ld_wait();
          if (edge) {
            const uint64_t seen = seen_of(mask, p.words, k0 + half * UNIT, sq.base, sq.ctx);
            const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
#pragma unroll
            for (int i = 0; i < UNIT; ++i)
              if (((i < 32 ? lo : hi) >> (i & 31) & 1) == 0) v[i] = __float_as_uint(-INFINITY);
          }
          float mx[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            mx[g] = __uint_as_float(v[16 * g]);
#pragma unroll
            for (int i = 1; i < 15; i += 2)
              mx[g] = max3(mx[g], __uint_as_float(v[16 * g + i]), __uint_as_float(v[16 * g + i + 1]));
            mx[g] = fmaxf(mx[g], __uint_as_float(v[16 * g + 15]));
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.c;
          // a stale maximum is kept unless the new one is above it by more than 2^8
          const bool grow = top > m_run + kLagLog2;
          if (__any_sync(0xffffffffu, grow)) {
            const float m_use = grow ? top : m_run;
            const float alpha = m_run == -INFINITY ? 0.f : exp2f(m_run - m_use);  // nothing before it: zeros
            l_run *= alpha;
            if (u > 0) {
              // O_t *= alpha once the W V of the unit before has landed (that of
              // a tile's second unit has, S of this tile was issued after it);
              // none is issued until this unit's W is published
              if (half == 1 && !mbar_wait_warp(&o_done[t * 2], static_cast<uint32_t>(jt & 1), abort_flag, p.status,
                                               kStatusTimeoutTmemFull)) {
                ok = false;
                break;
              }
              tc_fence_after();
#pragma unroll 1
              for (int c0 = 0; c0 < 128; c0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st32(o_addr + c0, o);
              }
            }
            m_run = m_use;
          }
          const float m_ref = m_run == -INFINITY ? 0.f : m_run;
          // w = 2^(c s - m) as bf16 pairs over the S columns just read
          const uint64_t c2 = f2pack(p.c, p.c), b2 = f2pack(-m_ref, -m_ref);
          uint64_t l2[2] = {f2pack(0.f, 0.f), f2pack(0.f, 0.f)};
#pragma unroll
          for (int i = 0; i < UNIT; i += 2) {
            float x0, x1;
            f2unpack(ffma2(f2pack(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), c2, b2), x0, x1);
            x0 = exp2f(x0);
            x1 = exp2f(x1);
            l2[(i >> 1) & 1] = fadd2(l2[(i >> 1) & 1], f2pack(x0, x1));
            v[i / 2] = pack_bf16(x0, x1);
          }
          tmem_st32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
          float a, b;
          f2unpack(fadd2(l2[0], l2[1]), a, b);
          l_run += a + b;
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(&p_full[t * 2 + half]);
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    // the last W V of the group has landed (its second unit's commit is the first phase of o_done[t][1])
    if (nt > 0 && ok) ok = mbar_wait_warp(&o_done[t * 2 + 1], 0, abort_flag, p.status, kStatusTimeoutTmemFull);
    tc_fence_after();
    float f0 = 1.f, f1 = 0.f;  // factors of this group's part and of the second's
    float* other = reinterpret_cast<float*>(sK);  // [128 rows][128], 16-byte pieces of a row in an order of its own
    if constexpr (ONE) {
      if (nt1 > 0) {
        if (t == 1) {
          // every tile has been used: the ring of K is free
          if (ok) {
#pragma unroll 1
            for (int c0 = 0; c0 < 128; c0 += 32) {
              uint32_t o[32];
              tmem_ld32(o_addr + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(other + r * 128 + (((c0 / 4 + i) ^ (r & 31)) * 4)) =
                    make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
            s_ml[r] = make_float2(m_run, l_run);
          }
          mbar_arrive(joined);
        } else if (ok) {
          ok = mbar_wait_warp(joined, 0, abort_flag, p.status, kStatusTimeoutTmemFull) && *abort_flag == 0;
          ok = __all_sync(0xffffffffu, ok);
          const float2 ml = s_ml[r];
          const float m = fmaxf(m_run, ml.x);
          f0 = m_run == -INFINITY ? 0.f : exp2f(m_run - m);
          f1 = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
          l_run = l_run * f0 + ml.y * f1;
          m_run = m;
        }
      }
    }
    if (ok && nt > 0 && (!ONE || t == 0)) {
      const size_t part = (static_cast<size_t>(row) * p.hq + head) * p.splits + z;
      const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;   // a NaN stays one
      const bool merge = sq.shares > 1;
      if (merge && live) p.lse_part[part] = l_run == 0.f ? -INFINITY : m_run + log2f(l_run);
#pragma unroll 1
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(o_addr + c0, o);
        tmem_ld_wait();
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(l_run == 0.f ? 0.f : __uint_as_float(o[i]) * f0 * inv);
        if (ONE && f1 != 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 w = *reinterpret_cast<const float4*>(other + r * 128 + (((c0 / 4 + i) ^ (r & 31)) * 4));
            const float x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) o[4 * i + k] = __float_as_uint(__uint_as_float(o[4 * i + k]) + x[k] * f1 * inv);
          }
        }
        if (merge) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(p.o_part + part * D + c0 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else {
          __nv_bfloat16* orow = p.out + static_cast<size_t>(row) * p.ldo + head * D + c0;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w;
            w.x = pack_bf16(__uint_as_float(o[i + 0]), __uint_as_float(o[i + 1]));
            w.y = pack_bf16(__uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
            w.z = pack_bf16(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5]));
            w.w = pack_bf16(__uint_as_float(o[i + 6]), __uint_as_float(o[i + 7]));
            *reinterpret_cast<uint4*>(orow + i) = w;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
  if (*not_finite != 0) write_not_finite(p, sq, first, n_nodes, kvh, z, j_lo * BKV, (j_lo + nk) * BKV);
}

// Merge the key shares of a (node, head) row.
template <int W>
__global__ void __launch_bounds__(kv8::MERGE_WARPS * 32) tree_merge_kernel(const __grid_constant__ Params p) {
  pdl_trigger();
  pdl_wait();
  const Seq sq = sequence(p, blockIdx.y, nullptr);
  const int at = blockIdx.x * (kv8::MERGE_WARPS / W) + (threadIdx.x >> 5) / W;
  const int node = at / p.hq, head = at % p.hq;
  if (sq.shares <= 1 || node >= sq.n) return;  // (W > 1: the same for the whole block)
  const int row = sq.start + node;
  const size_t part = (static_cast<size_t>(row) * p.hq + head) * p.splits;
  kv8::merge_shares<W>(p.o_part + part * D, p.lse_part + part, sq.shares,
                       p.out + static_cast<size_t>(row) * p.ldo + head * D);
}

}  // namespace atree
}  // namespace ib200

using namespace ib200;

// q [T, ldq] bf16 (head h at columns h*128); caches bf16 [num_slots, hkv*128];
// q_start / q_len / ctx_len [n_seqs], ctx_len with the nodes; mask int32 [T,
// words]; max_nodes: the most nodes of a sequence. Each sequence's 128-key tiles
// in shares of tiles_per_split, or of what `splits` shares need. o_part /
// lse_part: fp32 [T*hq*splits*128] / [T*hq*splits], used where a sequence has
// more than one share.
extern "C" int ib_attn_tree(const void* q, int T, int ldq, const void* k_cache, const void* v_cache, long long num_slots,
                            const int* q_start, const int* q_len, const int* ctx_len, const int* mask, int words,
                            int n_seqs, int max_nodes, const int* block_table, const int* bt_rows, int table_rows,
                            int max_pages, int ld_table, int hq, int hkv, float scale, int splits, int tiles_per_split,
                            float* o_part, float* lse_part, void* out, int ldo, int* status, cudaStream_t stream) {
  using namespace ib200::atree;
  if (T <= 0 || n_seqs <= 0 || max_nodes <= 0) return 0;
  if (hkv <= 0 || hq % hkv != 0 || hq / hkv > 16 || splits < 1 || tiles_per_split < 1 || words < 1 || words > 8 ||
      max_nodes > 32 * words || n_seqs > 65535 || (ldq % 8) != 0 || (ldo % 8) != 0 || num_slots < PAGE ||
      num_slots % PAGE != 0 || max_pages < 0 || max_pages > (1 << 27) - 1 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return -1;
  if (splits > 1 && (o_part == nullptr || lse_part == nullptr || (reinterpret_cast<uintptr_t>(o_part) & 15) != 0))
    return -1;
  try {
    const int kvw = hkv * D;
    CUtensorMap tk, tv, tk8, tv8;
    const auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (!cached_tmap_2d(&tk, k_cache, bf, 2, num_slots, kvw, kvw, 16, 64) ||
        !cached_tmap_2d(&tv, v_cache, bf, 2, num_slots, kvw, kvw, 16, 64) ||
        !cached_tmap_2d(&tk8, k_cache, bf, 2, num_slots, kvw, kvw, 128, 64) ||
        !cached_tmap_2d(&tv8, v_cache, bf, 2, num_slots, kvw, kvw, 128, 64))
      return -2;
    Params p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.ldq = ldq;
    p.T = T;
    p.q_start = q_start;
    p.q_len = q_len;
    p.ctx_len = ctx_len;
    p.mask = mask;
    p.words = words;
    p.v = static_cast<const __nv_bfloat16*>(v_cache);
    p.num_pages = static_cast<int>(num_slots / PAGE);
    p.block_table = block_table;
    p.bt_rows = bt_rows;
    p.table_rows = table_rows;
    p.max_pages = max_pages;
    p.ld_table = ld_table;
    p.hq = hq;
    p.hkv = hkv;
    p.G = hq / hkv;
    const bool one = max_nodes * p.G <= BQ;
    p.tokens = (one ? BQ : 2 * BQ) / p.G;
    p.blocks = (max_nodes + p.tokens - 1) / p.tokens;
    p.splits = splits;
    p.tiles_per_split = tiles_per_split;
    p.c = fmaxf(fabsf(scale) * 1.4426950408889634f, 1.2e-38f);  // positive: masked scores are -inf times it
    p.q_flip = scale < 0.f ? 0x80008000u : 0u;
    p.q_keep = scale == 0.f ? 0u : ~0u;
    p.o_part = o_part;
    p.lse_part = lse_part;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.ldo = ldo;
    p.status = status;
    if (static_cast<long long>(p.blocks) * splits > 65535) return -1;
    static bool attr_set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t e;
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
      e = cudaFuncSetAttribute(tree_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(tree_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
      if (e != cudaSuccess) return static_cast<int>(e);
      if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    e = launch_pdl(one ? tree_kernel<true> : tree_kernel<false>, dim3(hkv, n_seqs, p.blocks * splits), NUM_THREADS,
                   SMEM_BYTES, stream, tk, tv, tk8, tv8, p);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (splits > 1) {
      const long long rows = static_cast<long long>(max_nodes) * hq;
      if (kv8::merge_warps(rows * n_seqs, splits) > 1)
        e = launch_pdl(tree_merge_kernel<kv8::MERGE_WARPS>, dim3(static_cast<unsigned>(rows), n_seqs),
                       kv8::MERGE_WARPS * 32, 0, stream, p);
      else
        e = launch_pdl(tree_merge_kernel<1>, dim3(static_cast<unsigned>((rows + kv8::MERGE_WARPS - 1) / kv8::MERGE_WARPS), n_seqs),
                       kv8::MERGE_WARPS * 32, 0, stream, p);
    }
    return static_cast<int>(e);
  } catch (...) {  // (no memory for a tensor map's entry)
    return -3;
  }
}
