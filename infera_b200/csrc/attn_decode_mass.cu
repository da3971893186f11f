// Paged decode attention over the bf16 KV cache (one query token per sequence,
// GQA) that also adds up what each key received, on tcgen05:
//
//   o[h]          = sum_j w[h, j] v_j,  w[h, j] = 2^(c s[h, j] - m[h]) / l[h],  s = q K^T
//   mass[kvh, j] += sum over the KV head's query heads h of w[h, j]
//
// A weight is known only when the last key has been seen, so the pass over K
// and V keeps the raw scores (4 bytes a key and query head, against 512 of K
// and V a key and KV head). A second kernel merges the shares and turns the
// scores into weights; where a sequence is one share and short, its CTA does
// that itself at its end.
//
//   S^T[128 keys, 16]  = K_tile . Q^T     (A = K, K-major)
//   O^T[128 dims, 16]  = V_tile^T . W     (A = V, MN-major)
//
// The 16 columns of O^T hold two bf16 digits of the weights of up to 8 heads,
// w = hi + lo: a weight is off by at most 2^-16 of itself instead of bf16's
// 2^-8, and the digits cost no matrix instruction.
//
// One CTA handles (sequence, KV head, share) and walks its keys in tiles of 128
// (8 pages), 32 KB of K and 32 KB of V in a ring of three slots that both take
// in turn; two CTAs to an SM:
//   warp 0      TMA producer
//   warp 1      MMA issuer
//   warps 2..5  thread <-> key row for the softmax; they also stage Q
// A tile first only asks whether any score is above its head's running maximum
// by more than the lag (one compare a score, one barrier with an OR); the
// maxima are reduced and O^T is rescaled in TMEM when one is, in the first tile
// and rarely after it. V rows behind the sequence are zeroed in shared memory:
// what a recycled page holds there may be a NaN, which a zero weight does not
// cancel.
//
// Bound by HBM: 512 bytes a key and KV head. Captured calls of 32 sequences of
// 8192 keys (64 heads over 8) take 189 to 193 us, 175 of them (6.2 TB/s, 0.97 of
// the copy rate) for the first kernel and 15 for the second, which reads 67 MB of
// scores from L2; of 61 ragged ones up to 12000 keys on scattered pages (32 over
// 8) 256 us, 240 (0.94) and 15; of one of 100 keys 7.3 us. Finishing in the CTA
// that ends last in a (sequence, KV head), by a counter, was slower: it streams
// nothing meanwhile, 12 KB of scores a round trip (287 and 201 us). One sequence of
// 100000 keys on one KV head (8 heads, 261 shares) takes 45 us, where its bytes need 8:
// one CTA merges the shares in a loop; on 8 KV heads (64 heads, 36 shares) 78 of 65.
#include "kv8.cuh"
#include "tma_host.h"

namespace ib200 {
namespace dmass {

using kv8::elect_one;
using kv8::known_pages;
using kv8::max_over_warp;
using kv8::scaled;
using kv8::table_row;
using kv8::umma_bf16_if;
using kv8::umma_commit_if;

constexpr int D = 128;
constexpr int PAGE = 16;
constexpr int BKV = 128;
constexpr int BLK = 128 * 128;       // 128 rows x 128 B: one 64-dim half of a 128-key tile
constexpr int TILE = 2 * BLK;        // K or V of 128 keys
constexpr int SLOTS = 3;
constexpr int NQ = 16;               // columns of S^T and O^T
constexpr int QBLK = NQ * 128;       // 16 rows x 128 B
constexpr int PBLK = BKV * NQ * 2;   // weights of a tile
constexpr int NUM_THREADS = 192;
constexpr int SMEM_BYTES = 1024 + SLOTS * TILE + 2 * QBLK + 2 * PBLK + 1024;
constexpr uint32_t TMEM_COLS = 64;   // S0 [0,16) S1 [16,32) O [32,48)
constexpr uint32_t O_COL = 32;
constexpr float kLagLog2 = 8.0f;     // the running maximum may lag by this much
// Weights that meet V, and their sums, carry a factor of 2^-32, which divides out: 2^24 of the lagging ones times bf16's
// largest value are numbers of 32 bits.
constexpr float kDown = 1.0f / 4294967296.0f;
constexpr int FIN_THREADS = 256;
constexpr int FIN_KEYS = 1024;       // keys of a block of the second kernel

struct Params {
  const __nv_bfloat16* q;
  int ldq;
  const __nv_bfloat16* v;
  int num_pages;
  const int* block_table;
  const int* bt_rows;
  const int* seq_lens;
  int table_rows, max_pages, ld_table;
  int hq, hkv, G;
  int splits, tiles_per_split;  // split s covers tiles [s * this, (s + 1) * this) of every sequence
  float c;                      // |scale| * log2(e)
  uint32_t q_flip, q_keep;      // sign flips of q pairs (scale < 0), all bits or none kept (scale 0)
  float* scores;                // [B, hkv, keys, GP] raw scores
  long long keys;
  float* o_part;                // [B, hq, splits, D], not divided by the sum
  float2* ml;                   // [B, hq, splits] maximum (log2 units) and sum (with kDown); (-inf, 0): no keys
  float* mass;                  // [mass_rows, hkv, cap]
  int mass_rows;
  long long cap;
  __nv_bfloat16* out;
  int ldo;
  bool fused;                   // one share, whose CTA finishes
  int* status;
};

// Keys of sequence b that exist (as far as its page table goes) and its row of
// the tables; both kernels use the same, only the first reports.
struct Seq {
  int len, row;
  const int* bt;
};
__device__ __forceinline__ Seq sequence(const Params& p, int b, int* status) {
  const int row = p.bt_rows != nullptr ? p.bt_rows[b] : b;
  int len = max(p.seq_lens[b], 0);
  if (len > p.max_pages * PAGE) {  // more keys than the page table has places for
    if (threadIdx.x == 0) record_status_detail(status, kStatusBadIndex, 1, b, len);
    len = p.max_pages * PAGE;
  }
  const int* bt = table_row(p.block_table, row, p.table_rows, p.ld_table, b, status);
  return {bt == nullptr ? 0 : len, row, bt};
}

// Barrier of the four softmax warps that ORs a predicate. Every one of them
// passes the same number of these, whatever a bounded wait in between gave.
__device__ __forceinline__ bool barrier_or(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(pred))
      : "memory");
  return r != 0;
}
// byte offset of element (row, k) of a 16-row K-major block pair [k < 64 | k >= 64], 128-byte swizzle
__device__ __forceinline__ uint32_t q_offset(int row, int k) {
  const int half = k >> 6, kk = k & 63;
  return static_cast<uint32_t>(half * QBLK + row * 128 + ((((kk >> 3) ^ (row & 7))) << 4) + (kk & 7) * 2);
}
// MN-major descriptor without swizzle: cores of 16 bytes (columns) x 8 keys,
// `mn` bytes between cores along the columns, `k` along the keys.
__device__ __forceinline__ uint64_t make_mn_desc(uint32_t smem_addr, uint32_t mn, uint32_t k) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((k >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>((mn >> 4) & 0x3FFFu) << 32;
  d |= 1ull << 46;
  return d;
}

// The scores stay in L2 for the second kernel (67 MB for 32 sequences of 8192 keys and 64 heads).
template <int N>
__device__ __forceinline__ void store_scores(float* dst, const float (&x)[N], uint64_t policy) {
  if constexpr (N == 1) {
    asm volatile("st.global.L2::cache_hint.f32 [%0], %1, %2;" ::"l"(dst), "f"(x[0]), "l"(policy) : "memory");
  } else if constexpr (N == 2) {
    asm volatile("st.global.L2::cache_hint.v2.f32 [%0], {%1, %2}, %3;" ::"l"(dst), "f"(x[0]), "f"(x[1]), "l"(policy)
                 : "memory");
  } else {
#pragma unroll
    for (int h = 0; h < N; h += 4)
      asm volatile("st.global.L2::cache_hint.v4.f32 [%0], {%1, %2, %3, %4}, %5;" ::"l"(dst + h), "f"(x[h]), "f"(x[h + 1]),
                   "f"(x[h + 2]), "f"(x[h + 3]), "l"(policy)
                   : "memory");
  }
}

// ---- from parts and scores to the output and the mass, by CTAs of N threads
//   o = sum_s O_s 2^(m_s - M) / L,  L = sum_s l_s 2^(m_s - M)
//   mass[j] += sum_h 2^(c s[h, j] - M[h]) / L[h]

// Keys of a sequence that the splits cover.
__device__ __forceinline__ int covered(const Params& p, const Seq& sq) {
  return static_cast<int>(
      min(static_cast<long long>(sq.len), static_cast<long long>(p.splits) * p.tiles_per_split * BKV));
}
// M and 1 / L of the group's heads (L with the factor kDown).
template <int N>
__device__ __forceinline__ void make_sums(const Params& p, int b, int kvh, float* s_m, float* s_inv) {
  const int lane = threadIdx.x & 31;
  for (int h = threadIdx.x >> 5; h < p.G; h += N / 32) {
    const float2* ml = p.ml + (static_cast<size_t>(b) * p.hq + kvh * p.G + h) * p.splits;
    float m = -INFINITY, l = 0.f;
    for (int s = lane; s < p.splits; s += 32) m = fmaxf(m, __ldcg(ml + s).x);
    m = max_over_warp(m);
    if (m == -INFINITY) m = 0.f;
    for (int s = lane; s < p.splits; s += 32) {
      const float2 v = __ldcg(ml + s);
      if (v.x != -INFINITY) l += v.y * exp2f(v.x - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
      s_m[h] = m;
      s_inv[h] = l == 0.f ? 0.f : 1.f / l;
    }
  }
}
template <int N>
__device__ __forceinline__ void merge_parts(const Params& p, int b, int kvh, const float* s_m, const float* s_inv) {
  for (int i = threadIdx.x; i < p.G * (D / 4); i += N) {
    const int h = i / (D / 4), d = (i % (D / 4)) * 4;
    const size_t base = (static_cast<size_t>(b) * p.hq + kvh * p.G + h) * p.splits;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
      const float m = __ldcg(p.ml + base + s).x;
      if (m == -INFINITY) continue;  // a share without keys wrote nothing
      const float w = exp2f(m - s_m[h]);
      const float4 o = __ldcg(reinterpret_cast<const float4*>(p.o_part + (base + s) * D + d));
      a[0] += scaled(o.x, w);
      a[1] += scaled(o.y, w);
      a[2] += scaled(o.z, w);
      a[3] += scaled(o.w, w);
    }
    const float inv = s_inv[h];
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + static_cast<size_t>(b) * p.ldo + (kvh * p.G + h) * D + d);
    dst[0] = pack_bf16(a[0] * inv, a[1] * inv);
    dst[1] = pack_bf16(a[2] * inv, a[3] * inv);
  }
}
// The weights of keys k0 .. k0 + n, four a thread at a time. Called by all threads.
template <int GP, int N>
__device__ __forceinline__ void add_mass(const Params& p, const Seq& sq, int b, int kvh, int k0, int n, const float* s_m,
                                         const float* s_inv) {
  const int G = p.G, len = covered(p, sq), stop = min(len - k0, n) + k0;
  if (sq.row >= p.mass_rows || stop > p.cap) {
    if (threadIdx.x == 0)
      record_status_detail(p.status, kStatusBadIndex, 6, b, sq.row >= p.mass_rows ? sq.row : len);
    if (sq.row >= p.mass_rows) return;
  }
  if (p.bt_rows != nullptr) {  // a row that an earlier sequence of the batch has: that one's weights alone are added
    bool twice = false;
    for (int i = threadIdx.x; i < b; i += N) twice = twice || p.bt_rows[i] == sq.row;
    if (__syncthreads_or(twice)) {
      if (threadIdx.x == 0) record_status_detail(p.status, kStatusBadIndex, 7, b, sq.row);
      return;
    }
  }
  float m[GP], inv[GP];
#pragma unroll
  for (int h = 0; h < GP; ++h) {
    m[h] = h < G ? s_m[h] : 0.f;
    inv[h] = h < G ? s_inv[h] * kDown : 0.f;
  }
  const float* scores = p.scores + (static_cast<size_t>(b) * p.hkv + kvh) * static_cast<size_t>(p.keys) * GP;
  float* mass = p.mass + (static_cast<size_t>(sq.row) * p.hkv + kvh) * static_cast<size_t>(p.cap);
  const int end = static_cast<int>(min(static_cast<long long>(stop), p.cap));
  constexpr int KEYS = 4;
  for (int at = k0 + static_cast<int>(threadIdx.x); at < end; at += KEYS * N) {
    float x[KEYS][GP], was[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {  // all loads under way at once
      const int k = at + i * N;
      if (k >= end) break;
      const float* src = scores + static_cast<size_t>(k) * GP;
      if constexpr (GP == 1) {
        x[i][0] = __ldcg(src);
      } else if constexpr (GP == 2) {
        *reinterpret_cast<float2*>(&x[i][0]) = __ldcg(reinterpret_cast<const float2*>(src));
      } else {
#pragma unroll
        for (int h = 0; h < GP; h += 4)
          *reinterpret_cast<float4*>(&x[i][h]) = __ldcg(reinterpret_cast<const float4*>(src + h));
      }
      was[i] = mass[k];
    }
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int k = at + i * N;
      if (k >= end) break;
      float w = 0.f;
#pragma unroll
      for (int h = 0; h < GP; ++h)
        if (h < G) w = fmaf(exp2f(fmaf(x[i][h], p.c, -m[h])), inv[h], w);
      mass[k] = was[i] + w;
    }
  }
}
// The end of a sequence of one share. All threads, after the scores were written.
template <int GP>
__device__ __forceinline__ void end_share(const Params& p, const Seq& sq, int b, int kvh) {
  __shared__ float s_m[8], s_inv[8];
  __threadfence_block();
  __syncthreads();
  make_sums<NUM_THREADS>(p, b, kvh, s_m, s_inv);
  __syncthreads();
  add_mass<GP, NUM_THREADS>(p, sq, b, kvh, 0, sq.len, s_m, s_inv);
}

// The sum of what is not finite in one column (`v`, in a page's first row) of the values of keys k_lo .. k_hi: an
// infinity, a NaN, or 0. An infinity times two digits of different sign, or one of 0, is a NaN in the product. Rare, so
// nothing here is tuned.
__device__ __noinline__ float values_not_finite(const __nv_bfloat16* v, int width, int num_pages, const int* bt, int k_lo,
                                                int k_hi) {
  float sum = 0.f;
  for (int k0 = k_lo; k0 < k_hi && !isnan(sum); k0 += 8) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + i, page = k < k_hi ? bt[k / PAGE] : -1;
      x[i] = static_cast<unsigned>(page) >= static_cast<unsigned>(num_pages)
                 ? 0.f
                 : __bfloat162float(v[(static_cast<size_t>(page) * PAGE + k % PAGE) * width]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(fabsf(x[i]) <= FLT_MAX)) sum += x[i];
  }
  return sum;
}

template <int GP>  // query heads per KV head, rounded up to 1, 2, 4 or 8
__global__ void __launch_bounds__(NUM_THREADS, 2)
    decode_mass_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const __grid_constant__ CUtensorMap tmK8, const __grid_constant__ CUtensorMap tmV8,
                       const Params p) {
  constexpr int NC = (2 * GP + 7) / 8;  // 16-byte pieces of a key's digits
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.x, b = blockIdx.y, split = blockIdx.z;
  const int G = p.G;
  const Seq sq = sequence(p, b, p.status);
  const int len = sq.len;
  const int n_tiles = (len + BKV - 1) / BKV;
  if (split == p.splits - 1 && n_tiles > p.splits * static_cast<long long>(p.tiles_per_split) && threadIdx.x == 0)
    record_status_detail(p.status, kStatusBadArgs, 5, b, len);  // keys that no split takes
  const int t0 = static_cast<int>(min(static_cast<long long>(n_tiles), static_cast<long long>(split) * p.tiles_per_split));
  const int t1 = static_cast<int>(min(static_cast<long long>(n_tiles), static_cast<long long>(t0) + p.tiles_per_split));
  if (t0 >= t1) {  // nothing in this split
    if (threadIdx.x < G)
      p.ml[(static_cast<size_t>(b) * p.hq + kvh * G + threadIdx.x) * p.splits + split] = make_float2(-INFINITY, 0.f);
    if (p.splits == 1)
      for (int i = threadIdx.x; i < G * D; i += blockDim.x)
        p.out[static_cast<size_t>(b) * p.ldo + kvh * G * D + i] = __float2bfloat16(0.f);
    return;
  }
  const int nt = t1 - t0;
  const int n_pages = (len + PAGE - 1) / PAGE;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sKV = smem;                      // slot i % SLOTS: load i = K (even) or V (odd) of tile i / 2
  uint8_t* sQ = sKV + SLOTS * TILE;
  uint8_t* sP = sQ + 2 * QBLK;              // [2] columns: digit d of head h at d * GP + h
  uint64_t* bars = reinterpret_cast<uint64_t*>(sP + 2 * PBLK);
  uint64_t* full = bars;                    // [SLOTS]
  uint64_t* empty = full + SLOTS;           // [SLOTS]
  uint64_t* s_full = empty + SLOTS;         // [2]
  uint64_t* p_full = s_full + 2;            // [2] one per P buffer
  uint64_t* pv_done = p_full + 2;           // [2] PV of tile j commits to pv_done[j & 1]
  uint64_t* q_ready = pv_done + 2;
  uint64_t* drain = q_ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* red = reinterpret_cast<float*>(tmem_slot + 4);  // [4][GP] tile maxima, then sums

  const int warp = kv8::uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_ready, 128);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmK8);
    tma_prefetch_desc(&tmV8);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = kv8::uniform(*tmem_slot);

  if (warp == 0) {
    // The whole warp runs along and the elected lane issues, so that the operands stay in uniform registers: a lane of
    // its own issued the 32 boxes of a tile of scattered pages too slowly (61 ragged sequences 268 us against 260).
    const uint32_t on = elect_one();
    const uint64_t pol = policy_evict_first();
    int issued = 0, st = 0, ph = 1;
    bool ok = true;
    int nxt[8];
    load_tile_pages(sq.bt, t0, n_pages, nxt);
    for (int j = 0; j < nt && ok; ++j) {
      int cur[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) cur[i] = static_cast<int>(kv8::uniform(nxt[i]));
      known_pages(cur, p.num_pages);
      if (j + 1 < nt) load_tile_pages(sq.bt, t0 + j + 1, n_pages, nxt);  // in flight while we wait
      // eight consecutive pages are one 128-row box per half (the swizzle
      // repeats every 8 rows: the same image as eight page boxes)
      bool run = true;
#pragma unroll
      for (int pg = 1; pg < BKV / PAGE; ++pg) run = run && cur[pg] == cur[0] + pg;
      const int n = min(BKV / PAGE, n_pages - (t0 + j) * (BKV / PAGE));  // pages that the sequence has here
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        if (!ok) break;
        ok = mbar_wait_warp(&empty[st], static_cast<uint32_t>(ph), abort_flag, p.status, kStatusTimeoutEmpty);
        if (!ok) break;
        const CUtensorMap* tm1 = v ? &tmV : &tmK;
        uint8_t* dst = sKV + st * TILE;
        kv8::mbar_expect_tx_if(on, &full[st], 2 * n * PAGE * 128);
        if (run && n == BKV / PAGE) {
          const CUtensorMap* tm8 = v ? &tmV8 : &tmK8;
          kv8::tma_load_2d_if(on, dst, tm8, &full[st], kvh * D, cur[0] * PAGE, pol);
          kv8::tma_load_2d_if(on, dst + BLK, tm8, &full[st], kvh * D + 64, cur[0] * PAGE, pol);
        } else {
#pragma unroll
          for (int pg = 0; pg < BKV / PAGE; ++pg)
            if (pg < n) {
              kv8::tma_load_2d_if(on, dst + pg * PAGE * 128, tm1, &full[st], kvh * D, cur[pg] * PAGE, pol);
              kv8::tma_load_2d_if(on, dst + BLK + pg * PAGE * 128, tm1, &full[st], kvh * D + 64, cur[pg] * PAGE, pol);
            }
        }
        ++issued;
        if (++st == SLOTS) {
          st = 0;
          ph ^= 1;
        }
      }
    }
    for (int i = max(0, issued - SLOTS); i < issued; ++i)
      mbar_wait_warp(&full[i % SLOTS], static_cast<uint32_t>((i / SLOTS) & 1), nullptr, nullptr, 0, kWaitLimitNs / 4);
  } else if (warp == 1) {
    const uint32_t on = elect_one();
    const uint32_t idesc_s = make_idesc_bf16(128, NQ);
    const uint32_t idesc_o = make_idesc_bf16(128, NQ, true, true);
    const uint64_t q_desc = make_sw128_desc(smem_u32(sQ), 16, 1024);
    const uint64_t k_desc = make_sw128_desc(smem_u32(sKV), 16, 1024);
    const uint64_t v_desc = make_sw128_desc(smem_u32(sKV), BLK, 1024);  // MN-major: BLK to dims 64..127
    const uint64_t p_desc = make_mn_desc(smem_u32(sP), 128, 256);
    bool ok = mbar_wait_warp(q_ready, 0, abort_flag, p.status, kStatusTimeoutFull);
    // (descriptor addresses are in units of 16 bytes)
    for (int j = 0; j <= nt && ok; ++j) {
      if (j < nt) {
        const int i = 2 * j, st = i % SLOTS;
        ok = mbar_wait_warp(&full[st], static_cast<uint32_t>((i / SLOTS) & 1), abort_flag, p.status, kStatusTimeoutFull);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < 8; ++s)
          umma_bf16_if(on, tmem + ((j & 1) ? NQ : 0), k_desc + (st * TILE + (s >> 2) * BLK + (s & 3) * 32) / 16,
                       q_desc + ((s >> 2) * QBLK + (s & 3) * 32) / 16, idesc_s, s > 0 ? 1u : 0u);
        umma_commit_if(on, &s_full[j & 1]);
        umma_commit_if(on, &empty[st]);
      }
      if (j > 0) {
        const int jj = j - 1, i = 2 * jj + 1, st = i % SLOTS;
        ok = mbar_wait_warp(&p_full[jj & 1], static_cast<uint32_t>((jj >> 1) & 1), abort_flag, p.status,
                            kStatusTimeoutTmemEmpty) &&
             mbar_wait_warp(&full[st], static_cast<uint32_t>((i / SLOTS) & 1), abort_flag, p.status, kStatusTimeoutFull);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < 8; ++s)  // 16 keys each: two groups of 8
          umma_bf16_if(on, tmem + O_COL, v_desc + (st * TILE + s * 2048) / 16, p_desc + ((jj & 1) * PBLK + s * 512) / 16,
                       idesc_o, (jj > 0 || s > 0) ? 1u : 0u);
        umma_commit_if(on, &pv_done[jj & 1]);
        umma_commit_if(on, &empty[st]);
      }
    }
    umma_commit_if(on, drain);
    mbar_wait_warp(drain, 0, nullptr, p.status, kStatusTimeoutFull);
  } else {
    const int t = threadIdx.x - 64;   // 0..127
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;     // key row of S, dim row of O
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    bool ok = true;
    // stage Q: columns without a head, and without a digit of one, are zero
    for (int i = t; i < (2 * QBLK + 2 * PBLK) / 16; i += 128) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    barrier_or(false);
    for (int idx = t; idx < G * 64; idx += 128) {
      const int h = idx >> 6, d = (idx & 63) * 2;
      const uint32_t v =
          *reinterpret_cast<const uint32_t*>(p.q + static_cast<size_t>(b) * p.ldq + (kvh * G + h) * D + d);
      *reinterpret_cast<uint32_t*>(sQ + q_offset(h, d)) = (v ^ p.q_flip) & p.q_keep;
    }
    fence_proxy_async_smem();
    mbar_arrive(q_ready);

    // a head's scores are c * x, its running maximum m; a score above `limit`
    // is above the maximum by more than the lag
    float m_run[GP], limit[GP], l_part[GP];
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      m_run[h] = 0.f;
      limit[h] = h < G ? -INFINITY : INFINITY;
      l_part[h] = 0.f;
    }
    // the PV of tile jj has completed: its commit is completion (jj >> 1) + 1
    // of pv_done[jj & 1], and no later PV on that barrier can have been issued
    auto wait_pv = [&](int jj) {
      if (ok) ok = mbar_wait_warp(&pv_done[jj & 1], static_cast<uint32_t>((jj >> 1) & 1), abort_flag, p.status,
                                  kStatusTimeoutTmemFull);
      tc_fence_after();
    };
    const uint64_t keep = policy_evict_last();
    float* scores = p.scores + (static_cast<size_t>(b) * p.hkv + kvh) * static_cast<size_t>(p.keys) * GP;
    for (int j = 0; j < nt; ++j) {
      if (ok) ok = mbar_wait_warp(&s_full[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag, p.status,
                                  kStatusTimeoutTmemFull);
      tc_fence_after();
      uint32_t sv[16];
      tmem_ld16(lane_addr + ((j & 1) ? NQ : 0), sv);
      const int key = (t0 + j) * BKV + r;
      const bool last = (t0 + j + 1) * BKV > len;  // only here are rows masked
      const bool valid = !last || key < len;
      tmem_ld_wait();
      float x[GP];
      bool above = false;
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        x[h] = valid ? __uint_as_float(sv[h]) : -INFINITY;
        above = above || x[h] > limit[h];
      }
      if (valid) store_scores(scores + static_cast<size_t>(key) * GP, x, keep);
      if (barrier_or(above)) {
        // uniform over the CTA: every thread derives the same maxima
#pragma unroll
        for (int h = 0; h < GP; ++h) {
          const float mx = max_over_warp(x[h]);
          if (lane == 0) red[q4 * GP + h] = mx;
        }
        barrier_or(false);
        float f[GP];
#pragma unroll
        for (int h = 0; h < GP; ++h) {
          const float tmax = fmaxf(fmaxf(red[h], red[GP + h]), fmaxf(red[2 * GP + h], red[3 * GP + h]));
          f[h] = 1.f;
          if (tmax > limit[h]) {
            const float m = tmax * p.c;
            f[h] = limit[h] == -INFINITY ? 0.f : exp2f(m_run[h] - m);  // nothing before it: all zeros
            m_run[h] = m;
            limit[h] = (m + kLagLog2) / p.c;
            l_part[h] *= f[h];
          }
        }
        if (j > 0) {  // O^T *= f once the PV of the tile before has landed
          wait_pv(j - 1);
          uint32_t ov[16];
          tmem_ld16(lane_addr + O_COL, ov);
          tmem_ld_wait();
#pragma unroll
          for (int n = 0; n < 2 * GP; ++n) ov[n] = __float_as_uint(__uint_as_float(ov[n]) * f[n % GP]);
          tmem_st16(lane_addr + O_COL, ov);
          tmem_st_wait();
        }
        barrier_or(false);  // red is read
      }
      uint32_t d[4 * NC];  // digits by column, two to a word
#pragma unroll
      for (int i = 0; i < 4 * NC; ++i) d[i] = 0u;
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const float w = exp2f(fmaf(x[h], p.c, -m_run[h])) * kDown;
        l_part[h] += w;
        const __nv_bfloat16 hi = __float2bfloat16(w);
        const __nv_bfloat16 lo = __float2bfloat16(w - __bfloat162float(hi));
        d[h / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(hi)) << (16 * (h & 1));
        d[(GP + h) / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(lo)) << (16 * ((GP + h) & 1));
      }
      // P buffer j & 1 was last read by the PV of tile j - 2
      if (j >= 2) wait_pv(j - 2);
      uint8_t* pbuf = sP + (j & 1) * PBLK + (r >> 3) * 256 + (r & 7) * 16;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        *reinterpret_cast<uint4*>(pbuf + c * 128) = make_uint4(d[4 * c], d[4 * c + 1], d[4 * c + 2], d[4 * c + 3]);
      if (last) {
        const int i = 2 * j + 1, st = i % SLOTS;
        if (ok) ok = mbar_wait_warp(&full[st], static_cast<uint32_t>((i / SLOTS) & 1), abort_flag, p.status,
                                    kStatusTimeoutFull);
        if (!valid) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4* row = reinterpret_cast<uint4*>(sKV + st * TILE + half * BLK + r * 128);
#pragma unroll
            for (int k = 0; k < 8; ++k) row[k] = make_uint4(0, 0, 0, 0);
          }
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(&p_full[j & 1]);
    }
    wait_pv(nt - 1);
    uint32_t ov[16];
    tmem_ld16(lane_addr + O_COL, ov);
    tmem_ld_wait();
    // sum of the softmax: the per-key partials over the 128 rows
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      float v = l_part[h];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) red[q4 * GP + h] = v;
    }
    barrier_or(false);
    float wild = 0.f;  // (every head sees every key)
    bool odd = false;
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      const float o = __uint_as_float(ov[h]) + __uint_as_float(ov[GP + h]);
      odd = odd || (h < G && isnan(o) && !isnan(red[h] + red[GP + h] + red[2 * GP + h] + red[3 * GP + h]));
    }
    if (odd && ok) wild = values_not_finite(p.v + kvh * D + r, p.hkv * D, p.num_pages, sq.bt, t0 * BKV, min(len, t1 * BKV));
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      if (h >= G || !ok) break;
      const float l = red[h] + red[GP + h] + red[2 * GP + h] + red[3 * GP + h];
      float o = __uint_as_float(ov[h]) + __uint_as_float(ov[GP + h]);
      if (wild != 0.f) o = wild;
      const int head = kvh * G + h;
      const size_t slot = (static_cast<size_t>(b) * p.hq + head) * p.splits + split;
      if (r == 0) p.ml[slot] = make_float2(l == 0.f ? -INFINITY : m_run[h], l);
      if (p.splits == 1)
        p.out[static_cast<size_t>(b) * p.ldo + head * D + r] = __float2bfloat16(l == 0.f ? 0.f : o / l);
      else
        p.o_part[slot * D + r] = o;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, TMEM_COLS);
  }
  if (p.fused) end_share<GP>(p, sq, b, kvh);
}

// Block 0 of a (sequence, KV head) merges the shares, the others take FIN_KEYS
// keys each.
template <int GP>
__global__ void __launch_bounds__(FIN_THREADS) finish_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.y, b = blockIdx.z;
  const Seq sq = sequence(p, b, nullptr);
  const bool merge = blockIdx.x == 0;
  const int k0 = (static_cast<int>(blockIdx.x) - 1) * FIN_KEYS;
  if (merge ? p.splits == 1 : k0 >= covered(p, sq)) return;
  __shared__ float s_m[8], s_inv[8];
  make_sums<FIN_THREADS>(p, b, kvh, s_m, s_inv);
  __syncthreads();
  if (merge)
    merge_parts<FIN_THREADS>(p, b, kvh, s_m, s_inv);
  else
    add_mass<GP, FIN_THREADS>(p, sq, b, kvh, k0, FIN_KEYS, s_m, s_inv);
}

template <int GP>
int launch(const CUtensorMap (&tm)[4], const Params& p, int B, cudaStream_t stream) {
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(decode_mass_kernel<GP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  cudaError_t e = launch_pdl(decode_mass_kernel<GP>, dim3(p.hkv, B, p.splits), NUM_THREADS, SMEM_BYTES, stream, tm[0],
                             tm[1], tm[2], tm[3], p);
  if (e != cudaSuccess || p.fused) return static_cast<int>(e);
  const unsigned blocks = static_cast<unsigned>(1 + (p.keys + FIN_KEYS - 1) / FIN_KEYS);
  return static_cast<int>(launch_pdl(finish_kernel<GP>, dim3(blocks, p.hkv, B), FIN_THREADS, 0, stream, p));
}

}  // namespace dmass
}  // namespace ib200

using namespace ib200;

// q [B, ldq] bf16 (head h at columns h*128); caches bf16 [num_slots, hkv*128];
// block_table [table_rows] rows of max_pages places (pitch ld_table), row
// bt_rows[b] (null: b), which is also the sequence's row of mass, fp32
// [mass_rows, hkv, cap]; split s covers the 128-key tiles [s*tiles_per_split,
// (s+1)*tiles_per_split) of every sequence; scores: fp32 scratch of B*hkv*keys*GP
// (GP = hq/hkv rounded up to 1, 2, 4 or 8; keys: at least what the splits cover or the
// table holds, the lesser), ml of 2*B*hq*splits, o_part of B*hq*splits*128 (only
// touched when splits > 1). fused (splits 1): the first kernel's CTAs finish, else a
// second kernel.
extern "C" int ib_attn_decode_mass(const void* q, int ldq, const void* k_cache, const void* v_cache,
                                   long long num_slots, const int* block_table, const int* bt_rows,
                                   const int* seq_lens, int table_rows, int max_pages, int ld_table, int B, int hq,
                                   int hkv, int splits, int tiles_per_split, float scale, float* scores,
                                   long long keys, float* ml, float* o_part, float* mass, int mass_rows,
                                   long long cap, int fused, void* out, int ldo, int* status, cudaStream_t stream) {
  using namespace ib200::dmass;
  if (B <= 0) return 0;
  if (hkv <= 0 || hkv > 65535 || hq % hkv != 0 || hq / hkv > 8 || splits < 1 || tiles_per_split < 1 || (ldq % 2) != 0 ||
      B > 65535 || splits > 65535 || num_slots < PAGE || num_slots % PAGE != 0 || max_pages < 0 || max_pages > (1 << 26) ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 3) != 0 || (ldo % 2) != 0 || cap < 0 ||
      keys < 1 || (reinterpret_cast<uintptr_t>(scores) & 15) != 0 || scores == nullptr || ml == nullptr ||
      (reinterpret_cast<uintptr_t>(ml) & 7) != 0)
    return -1;
  if (splits > 1 && (o_part == nullptr || fused != 0 || (reinterpret_cast<uintptr_t>(o_part) & 15) != 0)) return -1;
  if (keys < std::min(static_cast<long long>(splits) * tiles_per_split * BKV, static_cast<long long>(max_pages) * PAGE))
    return -1;
  try {
    const int kvw = hkv * D;
    CUtensorMap tm[4];
    const auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (!cached_tmap_2d(&tm[0], k_cache, bf, 2, num_slots, kvw, kvw, 16, 64) ||
        !cached_tmap_2d(&tm[1], v_cache, bf, 2, num_slots, kvw, kvw, 16, 64) ||
        !cached_tmap_2d(&tm[2], k_cache, bf, 2, num_slots, kvw, kvw, 128, 64) ||
        !cached_tmap_2d(&tm[3], v_cache, bf, 2, num_slots, kvw, kvw, 128, 64))
      return -2;
    Params p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.ldq = ldq;
    p.v = static_cast<const __nv_bfloat16*>(v_cache);
    p.num_pages = static_cast<int>(num_slots / PAGE);
    p.block_table = block_table;
    p.bt_rows = bt_rows;
    p.seq_lens = seq_lens;
    p.table_rows = table_rows;
    p.max_pages = max_pages;
    p.ld_table = ld_table;
    p.hq = hq;
    p.hkv = hkv;
    p.G = hq / hkv;
    p.splits = splits;
    p.tiles_per_split = tiles_per_split;
    p.c = fmaxf(fabsf(scale) * 1.4426950408889634f, 1.2e-38f);  // positive: masked scores are -inf times it
    p.q_flip = scale < 0.f ? 0x80008000u : 0u;
    p.q_keep = scale == 0.f ? 0u : ~0u;
    p.scores = scores;
    p.keys = keys;
    p.o_part = o_part;
    p.ml = reinterpret_cast<float2*>(ml);
    p.mass = mass;
    p.mass_rows = mass_rows;
    p.fused = fused != 0;
    p.cap = cap;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.ldo = ldo;
    p.status = status;
    if (p.G <= 1) return launch<1>(tm, p, B, stream);
    if (p.G <= 2) return launch<2>(tm, p, B, stream);
    return p.G <= 4 ? launch<4>(tm, p, B, stream) : launch<8>(tm, p, B, stream);
  } catch (...) {  // (no memory for a tensor map's entry)
    return -3;
  }
}
