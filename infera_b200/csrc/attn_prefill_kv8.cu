// Causal flash attention for chunks of new tokens over the 8-bit paged KV
// cache, on tcgen05.
//
//   S = Q K^T     kind::f8f6f4: K's codes are an operand as they lie in memory.
//                 q * 2^s = hi + lo, hi in e4m3 and lo in e5m2 (s brings the
//                 row's largest element to [2^7, 2^8)). bf16 has 8 significant
//                 bits; hi rounded to 4 leaves -8 .. 8 units of the last place,
//                 which the 3 bits of e5m2 hold, and its exponents reach 2^-16:
//                 exact for elements down to 2^-13 of the row's largest, and
//                 off by at most 2^-21 of that one below (as a second e4m3
//                 digit, whose steps end at 2^-9, 2^-9 and 2^-17). S is eight
//                 32-wide products into one accumulator: the tensor core's time
//                 of a bf16 product
//   O += W V      kind::f16: V's codes converted to f16 (exact) once per tile
//                 of keys, W rounded to f16 in TMEM (11 significant bits)
//
// Scales (a power of two for 16 keys and a head): K's joins the softmax scale
// of its 16 columns of S, V's goes into the weight's exponent:
// w = 2^(s - m) * 2^(vsf - R + 6), R the largest V exponent so far, m the
// running maximum, which may lag by 2^8, so w <= 2^14 in f16. The sum of the
// softmax takes the fp32 weights without V's scale.
//
// The query heads of a KV head are packed: a CTA takes 256 rows of
// (token, head) pairs, 256 / G tokens, as two tiles of 128 rows that share
// every tile of 128 keys, so short chunks fill the tensor core's rows and a
// cached byte is read once per 256 rows and converted once.
//   warp 0       TMA producer: lane 0 K tiles, lane 1 V tiles
//   warp 1       MMA issuer: W0 V(j), S0(j+1), W1 V(j), S1(j+1)
//   warps 2..9   softmax, one thread per row and tile; they also stage Q
//   warps 10,11  V codes to f16; warp 10 also the scales of the key tiles' pages
// The tensor core works on one query tile while the other's softmax runs. The
// softmax takes a key tile in two units of 64 keys, whose scores a thread holds
// in registers (one read of TMEM gives the maximum and the weights), and
// publishes each unit's weights, so W V of the first overlaps the softmax of
// the second.
// Tiles of keys that some row does not see yet (the last ones) keep what is
// masked apart: there R counts the pages that a row sees, row by row, and a
// value that is NaN is multiplied as zero (a weight of zero would not cancel
// it) and written at the end to the rows that see it. Both loops that do so
// exist twice, for such tiles and for the others, which pay nothing for it
// (6 % of a long prompt with one loop).
// A CTA walks its item's key tiles or one share of them (few rows over a long
// context); shares are merged by a combine kernel. Items are found from q_len
// on the device, the ones with the most keys first.
//
// Bound by two things. A tile of 256 rows x 128 keys takes 2.1 us, the chain S,
// softmax, W V of each query tile, where the tensor core needs 1.46 at the
// measured rate. And a CTA takes one item or share, one CTA to an SM, so each
// exposes its start (Q staged, first tiles loaded) and its end, and the last
// round of CTAs leaves SMs idle. Captured calls of 1024 rows of 64 heads (over 8)
// and 32768 keys take 1113 to 1150 us (942 to 973 TFLOP/s, 0.55 to 0.57 of the
// library's bf16 rate; 917 us at 2.1 us a tile on all SMs), of six ragged prompts
// of 64 heads 230 us (0.43; 156), of 224 rows of 32 heads over 8416 keys 56 us
// (30), of 17 rows over 4113 keys 16.2 to 16.7 us. Eager calls on changing inputs
// take 1165 to 1191, 234 to 240, 59 and 24 us. Slower: sixteen softmax warps, an
// MMA warp for each query tile, exponentials on the FMA pipe.
#include <limits.h>

#include <type_traits>

#include "kv8.cuh"
#include "tma_host.h"

namespace ib200 {
namespace pq8 {

using namespace kv8;

constexpr int BQ = 128;               // rows of a query tile
constexpr int BKV = 128;
constexpr int BLK = 128 * 128;        // bytes of 128 rows x 128 codes, and of 128 rows x 64 f16
constexpr int KST = 3, VST = 2;       // stages of K tiles and of V tiles
constexpr int CVT = 64;               // threads that convert V
constexpr int NUM_THREADS = 320 + CVT;
constexpr int SMEM_BYTES = 1024 + (4 + KST + VST + 4) * BLK + 2048;
constexpr int UNIT = 64;              // keys of a step of the softmax
constexpr uint32_t O_COL = 256;       // S0 (W0 over each unit's columns) [0,128) S1 [128,256) O0 O1
constexpr float kLagLog2 = 8.0f;
constexpr int kTopLog2 = 6;           // weight of a key at the running maximum, V exponent at R
constexpr int kLeastLog2 = -60;       // V exponents further below R count as this far

struct Params {
  const __nv_bfloat16* q;
  int ldq;
  int T;                   // rows of q and out
  const int* q_start;
  const int* q_len;
  const int* ctx_len;
  int n_seqs;
  const uint8_t* ksf;
  const uint8_t* vsf;
  const uint8_t* vq;
  int num_pages;
  const int* block_table;
  const int* bt_rows;
  int table_rows, max_pages, ld_table;
  int hq, hkv, G, tokens;  // tokens: of an item, 256 / G
  int splits;
  float scale_log2;        // |scale| * log2(e)
  float q_sign;
  float* o_part;           // [T, hq, splits, 128]
  float* lse_part;         // [T, hq, splits]
  __nv_bfloat16* out;
  int ldo;
  int* status;
};

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

// The top bits of the bytes of four codes that are NaN (seven ones below the sign).
__device__ __forceinline__ uint32_t nan_codes(uint32_t u) { return (u & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u; }

// The item `at` when the sequences' items follow one another, those with the
// most keys first (of the first 32 sequences; the others follow as they come),
// and a sequence's from its last tokens to its first: the longest items start
// first, so that none is left for the end. Called by whole warps.
struct Found {
  int seq, block, q_len, ctx, q_start, table;  // block: the item's place in its sequence
};
__device__ __forceinline__ Found locate_item(const Params& p, int at) {
  const int lane = threadIdx.x & 31, per = p.tokens;
  int before = 0;
  for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
    const int s = s0 + lane, some = min(32, p.n_seqs - s0);
    const bool in = lane < some;
    const int len = in ? p.q_len[s] : 0, ctx = in ? p.ctx_len[s] : 0;
    // what only the found sequence's lane needs, in flight with the lengths
    const int start = in ? p.q_start[s] : 0, table = in && p.bt_rows != nullptr ? p.bt_rows[s] : s;
    const int n = (max(len, 0) + per - 1) / per, key = s0 == 0 ? ctx : 0;
    int ahead = 0, total = 0;  // items of the sequences before this lane's
    for (int l = 0; l < some; ++l) {
      const int nl = __shfl_sync(0xffffffffu, n, l), kl = __shfl_sync(0xffffffffu, key, l);
      if (kl > key || (kl == key && l < lane)) ahead += nl;
      total += nl;
    }
    const uint32_t has = __ballot_sync(0xffffffffu, at >= before + ahead && at < before + ahead + n);
    if (has != 0) {
      const int l = __ffs(has) - 1;
      return {s0 + l, __shfl_sync(0xffffffffu, n - 1 - (at - before - ahead), l), __shfl_sync(0xffffffffu, len, l),
              __shfl_sync(0xffffffffu, ctx, l), __shfl_sync(0xffffffffu, start, l),
              __shfl_sync(0xffffffffu, table, l)};
    }
    before += total;
  }
  return {-1, 0, 0, 0, 0, 0};
}

// What a CTA works on: tokens of a sequence and the key tiles of its share.
struct Item {
  int row_first, n_tokens, pos_first, ctx, j_lo, nk;
  const int* bt;
};

// Writes the NaN among the values of a CTA's last tiles, whose keys not every
// row sees, to the rows that see them, a warp per token. Values that are NaN
// are rare, so nothing here is tuned, and it stays out of the kernel's way: the
// item comes from shared memory.
__device__ __noinline__ void write_nan(const Params& p, const Item& it) {
  const int lane = threadIdx.x & 31, kvh = blockIdx.x, z = blockIdx.z;
  const int k_lo = max(it.j_lo, max(0, it.pos_first + 1) / BKV) * BKV, k_hi = (it.j_lo + it.nk) * BKV;
  for (int token = threadIdx.x >> 5; token < it.n_tokens; token += NUM_THREADS / 32) {
    const int row = it.row_first + token;
    if (row < 0 || row >= p.T) continue;
    const int end = min(min(it.pos_first + token + 1, it.ctx), k_hi);
    uint32_t bad = 0;  // of dims 4 lane .. 4 lane + 3
    for (int k = k_lo; k < end; ++k) {
      const int page = it.bt[k / PAGE];
      if (page < 0 || page >= p.num_pages) continue;
      const size_t at = (static_cast<size_t>(page) * PAGE + k % PAGE) * p.hkv + kvh;
      bad |= nan_codes(reinterpret_cast<const uint32_t*>(p.vq + at * D)[lane]);
    }
    if (bad == 0) continue;
    for (int i = 0; i < 4 * p.G; ++i) {
      if ((bad >> (8 * (i & 3)) & 0x80u) == 0) continue;
      const int head = kvh * p.G + i / 4, d = 4 * lane + (i & 3);
      if (p.splits > 1)
        p.o_part[((static_cast<size_t>(row) * p.hq + head) * p.splits + z) * D + d] = NAN;
      else
        p.out[static_cast<size_t>(row) * p.ldo + head * D + d] = __float2bfloat16(NAN);
    }
  }
}

// The row of q and out of chunk row `at`, INT_MIN behind the last. Called by
// whole warps.
__device__ __forceinline__ int locate_row(const int* q_len, const int* q_start, int n_seqs, int at) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += 32) {
    const bool in = s0 + lane < n_seqs;
    const int n = in ? max(q_len[s0 + lane], 0) : 0;
    const int start = in ? q_start[s0 + lane] : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const uint32_t has = __ballot_sync(0xffffffffu, at < before + sum);
    if (has != 0) {
      const int l = __ffs(has) - 1;
      return at - before + __shfl_sync(0xffffffffu, start - (sum - n), l);
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return INT_MIN;
}

__global__ void __launch_bounds__(NUM_THREADS, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ CUtensorMap tmK8, const __grid_constant__ CUtensorMap tmV8,
                   const __grid_constant__ Params p) {
  pdl_trigger();
  pdl_wait();
  __shared__ Item s_item;
  __shared__ volatile int s_nan;  // a value was NaN in a tile that not every row sees whole
  const int kvh = blockIdx.x, z = blockIdx.z, S = p.splits, G = p.G;
  const Found it = locate_item(p, blockIdx.y);
  const int seq = it.seq, qlen = it.q_len;
  if (seq < 0) return;
  int ctx = max(it.ctx, 0);
  const int first = it.block * p.tokens;              // the item's first token in the chunk
  const int n_rows = min(p.tokens, qlen - first) * G;
  const int pos_first = ctx - qlen + first;
  const int row_first = it.q_start + first;
  const int* bt = table_row(p.block_table, it.table, p.table_rows, p.ld_table, seq, p.status);
  if (bt == nullptr) ctx = 0;
  if (ctx > p.max_pages * PAGE) {  // more keys than the page table has places for
    if (threadIdx.x == 0) record_status_detail(p.status, kStatusBadIndex, 1, seq, ctx);
    ctx = p.max_pages * PAGE;
  }
  // rows of the two query tiles and the units of keys that their last tokens see
  int rows_t[2], nuv_t[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    rows_t[t] = max(0, min(BQ, n_rows - t * BQ));
    const int last = pos_first + (t * BQ + rows_t[t] - 1) / G;
    nuv_t[t] = rows_t[t] > 0 ? max(0, (min(last + 1, ctx) + UNIT - 1) / UNIT) : 0;
  }
  const int n_kv = (max(nuv_t[0], nuv_t[1]) + 1) / 2;   // tiles of 128 keys
  const int chunk = (n_kv + S - 1) / S;
  const int j_lo = z * chunk;
  const int nk = min(n_kv - j_lo, chunk);
  if (nk <= 0) {  // no keys in this share, or none at all
    for (int i = threadIdx.x; i < n_rows; i += blockDim.x) {
      const int row = row_first + i / G, head = kvh * G + i % G;
      if (row < 0 || row >= p.T) continue;
      if (S > 1) p.lse_part[(static_cast<size_t>(row) * p.hq + head) * S + z] = -INFINITY;
      else
        for (int d = 0; d < D; ++d) p.out[static_cast<size_t>(row) * p.ldo + head * D + d] = __float2bfloat16(0.f);
    }
    return;
  }
  int nu_t[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) nu_t[t] = max(0, min(nuv_t[t] - 2 * j_lo, 2 * chunk));
  const int n_pages = (ctx + PAGE - 1) / PAGE;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                    // tile t: digits hi, lo
  uint8_t* sK = sQ + 4 * BLK;            // [KST]
  uint8_t* sV8 = sK + KST * BLK;         // [VST] codes
  uint8_t* sV = sV8 + VST * BLK;         // [2] f16: dims 0..63, dims 64..127
  float4* sSf = reinterpret_cast<float4*>(sV + 4 * BLK);  // [4][8 pages] 2^ke, weight exponent, its inverse, ve
  int* sR = reinterpret_cast<int*>(sSf + 32);             // [4] R of the tile
  uint64_t* bars = reinterpret_cast<uint64_t*>(sR + 4);
  uint64_t* q_ready = bars;
  uint64_t* k_full = bars + 1;           // [KST]
  uint64_t* k_empty = k_full + KST;      // [KST]
  uint64_t* v8_full = k_empty + KST;     // [VST]
  uint64_t* v8_empty = v8_full + VST;    // [VST]
  uint64_t* v_full = v8_empty + VST;     // [2]
  uint64_t* v_empty = v_full + 2;        // [2]
  uint64_t* s_full = v_empty + 2;        // [2 query tiles]
  uint64_t* p_full = s_full + 2;         // [2 query tiles][2 units]
  uint64_t* o_done = p_full + 4;         // [2][2]: a phase of [t][0] per first unit's W V; [t][1]: the last one's
  uint64_t* sf_full = o_done + 4;        // [4]
  uint64_t* drain = sf_full + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_ready, 256);
    for (int s = 0; s < KST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(&v8_full[s], 1);
      mbar_init(&v8_empty[s], CVT);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&v_full[t], CVT);
      mbar_init(&v_empty[t], 1);
      mbar_init(&s_full[t], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&p_full[s], 128);
      mbar_init(&o_done[s], 1);
      mbar_init(&sf_full[s], 8);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    s_nan = 0;
    s_item = {row_first, n_rows / G, pos_first, ctx, j_lo, nk, bt};
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
      uint64_t* full = is_v ? v8_full : k_full;
      uint64_t* empty = is_v ? v8_empty : k_empty;
      uint8_t* dst0 = is_v ? sV8 : sK;
      const uint64_t pol = policy_evict_last();  // the other items of the sequence read these keys too
      int issued = 0, st = 0, ph = 1;
      int nxt[8];
      load_tile_pages(bt, j_lo, n_pages, nxt);
      for (int j = 0; j < nk; ++j) {
        int cur[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cur[i] = nxt[i];
        known_pages(cur, p.num_pages);
        if (j + 1 < nk) load_tile_pages(bt, j_lo + j + 1, n_pages, nxt);
        if (!mbar_wait(&empty[st], static_cast<uint32_t>(ph), abort_flag, p.status, kStatusTimeoutEmpty)) break;
        uint8_t* dst = dst0 + st * BLK;
        bool run = true;
#pragma unroll
        for (int pg = 1; pg < BKV / PAGE; ++pg) run = run && cur[pg] == cur[0] + pg;
        const int n = min(BKV / PAGE, n_pages - (j_lo + j) * (BKV / PAGE));  // pages that the sequence has here
        mbar_expect_tx(&full[st], n * PAGE * 128);
        if (run && n == BKV / PAGE) {
          tma_load_2d(dst, tm8, &full[st], kvh * D, cur[0] * PAGE, pol);
        } else {
#pragma unroll
          for (int pg = 0; pg < BKV / PAGE; ++pg)
            if (pg < n) tma_load_2d(dst + pg * PAGE * 128, tm1, &full[st], kvh * D, cur[pg] * PAGE, pol);
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
    const uint32_t idesc_hi = make_idesc_e4m3(128, BKV);
    const uint32_t idesc_lo = idesc_hi | (1u << 7);  // A in e5m2
    // f16 operands (formats 0), B = V with adjacent dims (MN-major)
    const uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
    const uint64_t q_desc = make_sw128_desc(smem_u32(sQ), 16, 1024);
    const uint64_t k_desc = make_sw128_desc(smem_u32(sK), 16, 1024);
    const uint64_t v_desc = make_sw128_desc(smem_u32(sV), BLK, 1024);
    const int n0 = uniform(nu_t[0]), n1 = uniform(nu_t[1]);
    const int nj = (max(n0, n1) + 1) / 2;
    bool ok = mbar_wait_warp(q_ready, 0, abort_flag, p.status, kStatusTimeoutFull);
    // (descriptor addresses are in units of 16 bytes)
    for (int j = -1; j < nj && ok; ++j) {
      const int st = (j + 1) % KST;
      if (j + 1 < nj) ok = mbar_wait_warp(&k_full[st], static_cast<uint32_t>(((j + 1) / KST) & 1), abort_flag,
                                          p.status, kStatusTimeoutFull);
      if (j >= 0 && ok) ok = mbar_wait_warp(&v_full[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag, p.status,
                                            kStatusTimeoutFull);
      if (!ok) break;
      const uint64_t kd = k_desc + st * (BLK / 16);
      const uint64_t vd = v_desc + (j & 1) * (2 * BLK / 16);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int n = t ? n1 : n0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (j < 0 || 2 * j + half >= n || !ok) break;
          ok = mbar_wait_warp(&p_full[t * 2 + half], static_cast<uint32_t>(j & 1), abort_flag, p.status,
                              kStatusTimeoutTmemEmpty);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < 4; ++s)
            // W_t packs keys 16s .. 16s + 15 of the unit into columns 8s .. 8s + 7 of its S
            umma_f16_ts_if(on, tmem + O_COL + t * 128, tmem + t * 128 + half * UNIT + s * 8,
                           vd + (half * UNIT * 128 + s * 2048) / 16, idesc_pv, (j > 0 || half > 0 || s > 0) ? 1u : 0u);
          if (half == 0 || 2 * j + 2 == n) umma_commit_if(on, &o_done[t * 2 + half]);
        }
        if (2 * (j + 1) < n && ok) {
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < 8; ++s)
            umma_e4m3_if(on, tmem + t * 128, q_desc + (t * 2 * BLK + (s >> 2) * BLK + (s & 3) * 32) / 16,
                         kd + (s & 3) * 32 / 16, s < 4 ? idesc_hi : idesc_lo, s > 0 ? 1u : 0u);
          umma_commit_if(on, &s_full[t]);
        }
      }
      if (!ok) break;
      if (j + 1 < nj) umma_commit_if(on, &k_empty[st]);
      if (j >= 0) umma_commit_if(on, &v_empty[j & 1]);
    }
    umma_commit_if(on, drain);
    mbar_wait_warp(drain, 0, nullptr, p.status, kStatusTimeoutFull);
  } else if (warp >= 10) {
    // V codes to f16, and each key tile's scales one tile ahead
    const int ct = threadIdx.x - 320;
    const bool scales = ct < 8;
    int R = 0;
    uint32_t ke = 0, ve = 0;  // exponents as loaded, for the next publish
    auto page_of = [&](int j) -> int {
      const int lp = (j_lo + j) * (BKV / PAGE) + ct;
      return j < nk && lp < n_pages ? __ldg(bt + lp) : -1;
    };
    auto load = [&](int page) {  // waited for at the publish, a tile later
      const bool in = page >= 0 && page < p.num_pages;
      const size_t at = static_cast<size_t>(in ? page : 0) * p.hkv + kvh;
      ke = in ? __ldg(p.ksf + at) : 0u;
      ve = in ? __ldg(p.vsf + at) : 0u;
    };
    // The scales of tile j go to one of four places: the softmax of tile j - 4
    // is done with it when the W V of tile j - 3 is (which the caller waited for).
    auto publish = [&](int j) {
      const int e = exponent_of(ve);
      R = max(R, __reduce_max_sync(0xffu, e));
      const int d = max(e - R, kLeastLog2) + kTopLog2;
      sSf[(j & 3) * 8 + ct] = make_float4(two_to(exponent_of(ke) - 127), static_cast<float>(d),
                                          two_to(-d), static_cast<float>(e));
      if (ct == 0) sR[j & 3] = R;
      mbar_arrive(&sf_full[j & 3]);
    };
    int page_next = -1;
    if (scales) {
      load(page_of(0));
      page_next = page_of(1);
      publish(0);
      load(page_next);
      page_next = page_of(2);
    }
    __syncwarp();
    for (int j = 0; j < nk; ++j) {
      const int st = j % VST, vb = j & 1;
      if (!mbar_wait_warp(&v_empty[vb], static_cast<uint32_t>(((j >> 1) & 1) ^ 1), abort_flag, p.status,
                          kStatusTimeoutEmpty))
        break;
      if (scales && j + 1 < nk) {
        publish(j + 1);
        load(page_next);
        page_next = page_of(j + 3);
      }
      __syncwarp();
      if (!mbar_wait_warp(&v8_full[st], static_cast<uint32_t>((j / VST) & 1), abort_flag, p.status,
                          kStatusTimeoutFull))
        break;
      const uint8_t* src = sV8 + st * BLK;
      uint8_t* dst = sV + vb * 2 * BLK;
      const int live = ctx - (j_lo + j) * BKV;  // rows behind the sequence are zero: a stale code may be a NaN
      auto convert = [&](auto edge) {
#pragma unroll 4
      for (int i = 0; i < 1024 / CVT; ++i) {
        const int idx = ct + i * CVT;
        const int r = idx >> 3;
        const int ch = (idx & 7) ^ (r & 7);     // dims 16 ch .. 16 ch + 15
        uint4 v = *reinterpret_cast<const uint4*>(src + idx * 16);
        if (r >= live) v = make_uint4(0u, 0u, 0u, 0u);
        uint32_t u[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[8];
        if constexpr (decltype(edge)::value) {
          const uint32_t x = nan_codes(u[0]), y = nan_codes(u[1]), z = nan_codes(u[2]), w = nan_codes(u[3]);
          if ((x | y | z | w) != 0) {  // zero here, see write_nan
            u[0] &= ~((x >> 7) * 255u);
            u[1] &= ~((y >> 7) * 255u);
            u[2] &= ~((z >> 7) * 255u);
            u[3] &= ~((w >> 7) * 255u);
            s_nan = 1;
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[2 * k] = h2_bits(from_e4m3x2_h(u[k] & 0xffffu));
          h[2 * k + 1] = h2_bits(from_e4m3x2_h(u[k] >> 16));
        }
        // dims below 64 store their first 8 first, the others their second: the
        // eight lanes of a row then write eight different 16-byte columns
        const bool up = ch >= 4;
        uint8_t* row = dst + (up ? BLK : 0) + r * 128;
        const int c = (ch & 3) * 2;
        const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), b = make_uint4(h[4], h[5], h[6], h[7]);
        *reinterpret_cast<uint4*>(row + (((c + (up ? 1 : 0)) ^ (r & 7)) << 4)) = up ? b : a;
        *reinterpret_cast<uint4*>(row + (((c + (up ? 0 : 1)) ^ (r & 7)) << 4)) = up ? a : b;
      }
      };
      if ((j_lo + j) * BKV + BKV - 1 > pos_first)
        convert(std::true_type{});
      else
        convert(std::false_type{});
      fence_proxy_async_smem();
      mbar_arrive(&v8_empty[st]);
      mbar_arrive(&v_full[vb]);
    }
  } else {
    const int t = (warp - 2) >> 2;
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const int rows = t ? rows_t[1] : rows_t[0];   // selects: no dynamically indexed local arrays
    const int nut = t ? nu_t[1] : nu_t[0];
    const int pr = t * BQ + min(r, max(rows, 1) - 1);
    const int token = pr / G, head = kvh * G + pr - token * G;
    const int row = row_first + token;
    const bool write = r < rows && row >= 0 && row < p.T;
    const int pos = min(pos_first + token, ctx - 1);    // the last key that this row sees
    const int pos0 = min(pos_first + t * BQ / G, ctx - 1);
    // stage this row's digits (rows that do not exist are zero)
    float c_row;
    {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + static_cast<size_t>(write ? row : 0) * p.ldq + head * D);
      uint4 v[16];
      uint32_t mb = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = write ? src[i] : make_uint4(0u, 0u, 0u, 0u);  // (out may be q)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) mb = max(mb, max((u[k] << 16) & 0x7fffffffu, u[k] & 0x7fff0000u));
      }
      const int s = min(100, 134 - static_cast<int>(mb >> 23));
      const float f = two_to(s) * p.q_sign;
      c_row = p.scale_log2 * two_to(-s);
      uint8_t* hi = sQ + t * 2 * BLK;
      uint8_t* lo = hi + BLK;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        uint32_t dh[4], dl[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4& w = v[i + (k >> 1)];
          const uint32_t ua = (k & 1) ? w.z : w.x, ub = (k & 1) ? w.w : w.y;
          float x[4] = {bf16_lo(ua), bf16_hi(ua), bf16_lo(ub), bf16_hi(ub)};
#pragma unroll
          for (int m = 0; m < 4; ++m) x[m] = fabsf(x[m]) <= 3.4e38f ? x[m] * f : NAN;
          const uint32_t a = to_e4m3x2(x[0], x[1]), b = to_e4m3x2(x[2], x[3]);
          const float2 fa = from_e4m3x2(a), fb = from_e4m3x2(b);
          dh[k] = a | b << 16;
          dl[k] = to_e5m2x2(x[0] - fa.x, x[1] - fa.y) | to_e5m2x2(x[2] - fb.x, x[3] - fb.y) << 16;
        }
        *reinterpret_cast<uint4*>(hi + sw_offset(r, i * 8)) = make_uint4(dh[0], dh[1], dh[2], dh[3]);
        *reinterpret_cast<uint4*>(lo + sw_offset(r, i * 8)) = make_uint4(dl[0], dl[1], dl[2], dl[3]);
      }
      fence_proxy_async_smem();
      mbar_arrive(q_ready);
    }
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    const uint32_t o_addr = lane_addr + O_COL + t * 128;
    float m_run = -INFINITY;
    float l_run = 0.f;
    int R_run = 0;
    bool ok = true;
    // One unit; EDGE: of a tile that not every row sees whole.
    auto unit = [&](auto edge, int u) -> bool {
      constexpr bool EDGE = decltype(edge)::value;
      const int j = u >> 1, half = u & 1;
      if ((half == 0 && !mbar_wait_warp(&sf_full[j & 3], static_cast<uint32_t>((j >> 2) & 1), abort_flag, p.status,
                                        kStatusTimeoutFull)) ||
          (half == 0 && !mbar_wait_warp(&s_full[t], static_cast<uint32_t>(j & 1), abort_flag, p.status,
                                        kStatusTimeoutTmemFull))) {
        return false;
      }
      tc_fence_after();
      const uint32_t s_addr = lane_addr + t * 128 + half * UNIT;
      const float4* sf = sSf + (j & 3) * 8 + half * 4;
      const int kbase = (j_lo + j) * BKV + half * UNIT;
      uint32_t v[UNIT];
      tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
      tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
      int R = sR[j & 3];
      float4 f[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) f[g] = sf[g];
      if constexpr (EDGE) {  // R of the pages that this row sees
        R = R_run;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (kbase + 16 * g <= pos) R = max(R, static_cast<int>(f[g].w));
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = min(max(static_cast<int>(f[g].w) - R, kLeastLog2), 0) + kTopLog2;
          f[g].y = static_cast<float>(d);
          f[g].z = two_to(-d);
        }
      }
      tmem_ld_wait();
      if constexpr (EDGE) {
        const int lim = pos - kbase;  // key c of the unit is visible iff c <= lim
#pragma unroll
        for (int i = 0; i < UNIT; ++i)
          if (i > lim) v[i] = __float_as_uint(-INFINITY);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float a = __uint_as_float(v[16 * g]), b = __uint_as_float(v[16 * g + 1]);
#pragma unroll
        for (int i = 2; i < 16; i += 4) {
          a = max3(a, __uint_as_float(v[16 * g + i]), __uint_as_float(v[16 * g + i + 1]));
          if (i + 2 < 16) b = max3(b, __uint_as_float(v[16 * g + i + 2]), __uint_as_float(v[16 * g + i + 3]));
        }
        mx = fmaxf(mx, fmaxf(a, b) * f[g].x);
      }
      mx *= c_row;
      // a stale maximum is kept unless the new one is above it by more than 2^8
      const bool grow = mx > m_run + kLagLog2;
      if (__any_sync(0xffffffffu, grow || R != R_run)) {
        const float m_use = grow ? mx : m_run;
        const float alpha = m_run == -INFINITY ? 0.f : exp2f(m_run - m_use);  // nothing before it: zeros
        l_run *= alpha;
        if (u > 0) {
          // O_t *= alpha once the W V of the unit before has landed (that of a
          // tile's second unit has, S of this tile was issued after it); none
          // is issued until this unit's W is published
          if (half == 1 && !mbar_wait_warp(&o_done[t * 2], static_cast<uint32_t>(j & 1), abort_flag, p.status,
                                           kStatusTimeoutTmemFull)) {
            return false;
          }
          tc_fence_after();
          const float fo = alpha * two_to(max(R_run - R, -126));
#pragma unroll 1
          for (int c0 = 0; c0 < 128; c0 += 32) {
            uint32_t o[32];
            tmem_ld32(o_addr + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fo);
            tmem_st32(o_addr + c0, o);
          }
        }
        m_run = m_use;
        R_run = R;
      }
      const float m_ref = m_run == -INFINITY ? 0.f : m_run;
      // w = 2^(s - m + V's exponent) as f16 pairs over the S columns just
      // read; the sum without V's exponent
      uint64_t l2 = f2pack(0.f, 0.f);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        // positive, so that masked scores stay -inf
        const float c = fmaxf(c_row * f[g].x, 1.2e-38f), b = f[g].y - m_ref;
        const uint64_t c2 = f2pack(c, c), b2 = f2pack(b, b);
        uint64_t sum2 = f2pack(0.f, 0.f);
#pragma unroll
        for (int i = 16 * g; i < 16 * g + 16; i += 2) {
          float x0, x1;
          f2unpack(ffma2(f2pack(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), c2, b2), x0, x1);
          x0 = exp2f(x0);
          x1 = exp2f(x1);
          sum2 = fadd2(sum2, f2pack(x0, x1));
          v[i / 2] = h2_bits(__floats2half2_rn(x0, x1));
        }
        l2 = ffma2(sum2, f2pack(f[g].z, f[g].z), l2);
      }
      tmem_st32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
      float a, b;
      f2unpack(l2, a, b);
      l_run += a + b;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t * 2 + half]);
      return true;
    };
    int u = 0;
    const int whole = min(nut, 2 * ((pos0 + 1) / BKV - j_lo));
    for (; u < whole && ok; ++u) ok = unit(std::false_type{}, u);
    for (; u < nut && ok; ++u) ok = unit(std::true_type{}, u);
    ok = __all_sync(0xffffffffu, ok);
    const size_t part = (static_cast<size_t>(row) * p.hq + head) * S + z;
    if (nut <= 0) {
      if (write) {
        if (S > 1)
          p.lse_part[part] = -INFINITY;
        else
          for (int i = 0; i < D / 8; ++i)
            reinterpret_cast<uint4*>(p.out + static_cast<size_t>(row) * p.ldo + head * D)[i] = make_uint4(0u, 0u, 0u, 0u);
      }
    } else if (ok && mbar_wait_warp(&o_done[t * 2 + ((nut - 1) & 1)],
                                    (nut & 1) ? static_cast<uint32_t>(((nut - 1) >> 1) & 1) : 0u, abort_flag, p.status,
                                    kStatusTimeoutTmemFull)) {
      tc_fence_after();
      const float inv = l_run == 0.f ? 0.f : 1.0f / l_run * (1.f / (1 << kTopLog2));   // a NaN stays one
      const float back = two_to(max(R_run, 1) - 127);
      if (S > 1 && write) p.lse_part[part] = l_run == 0.f ? -INFINITY : m_run + log2f(l_run);
#pragma unroll 1
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(o_addr + c0, o);
        tmem_ld_wait();
        if (!write) continue;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv * back);
        if (S > 1) {
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
  if (s_nan != 0) write_nan(p, s_item);
}

// Merge the key shares of a query row.
template <int W>
__global__ void __launch_bounds__(MERGE_WARPS * 32) prefill_merge_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  const int row = locate_row(p.q_len, p.q_start, p.n_seqs, blockIdx.x);
  const int head = blockIdx.y * (MERGE_WARPS / W) + (threadIdx.x >> 5) / W;
  if (row < 0 || row >= p.T || head >= p.hq) return;
  const size_t part = (static_cast<size_t>(row) * p.hq + head) * p.splits;
  merge_shares<W>(p.o_part + part * D, p.lse_part + part, p.splits,
                  p.out + static_cast<size_t>(row) * p.ldo + head * D);
}

}  // namespace pq8
}  // namespace ib200

using namespace ib200;

// q [T, ldq] bf16 (head h at columns h*128); kq / vq e4m3 [num_slots, hkv*128]
// and ksf / vsf [num_slots/16, hkv]; q_start / q_len / ctx_len [n_seqs];
// block_table [table_rows] rows of max_pages places (pitch ld_table), row
// bt_rows[s] (null: s). n_items: sum of ceil(q_len / (256 / G)); n_rows: sum of q_len. splits
// > 1: each item's key tiles in that many shares, o_part / lse_part fp32
// [T*hq*splits*128] / [T*hq*splits].
extern "C" int ib_attn_prefill_kv8(const void* q, int T, int ldq, const void* kq, const void* ksf, const void* vq,
                                   const void* vsf, long long num_slots, const int* q_start, const int* q_len,
                                   const int* ctx_len, int n_seqs, int n_items, int n_rows, const int* block_table,
                                   const int* bt_rows, int table_rows, int max_pages, int ld_table, int hq, int hkv,
                                   float scale, int splits, float* o_part, float* lse_part, void* out, int ldo, int* status,
                                   cudaStream_t stream) {
  using namespace ib200::pq8;
  if (T <= 0 || n_seqs <= 0 || n_items <= 0) return 0;
  if (hkv <= 0 || hq % hkv != 0 || hq / hkv > 8 || splits < 1 || splits > 65535 || n_items > 65535 ||
      (ldq % 8) != 0 || (ldo % 8) != 0 || num_slots < PAGE || num_slots % PAGE != 0 || max_pages < 0 || hq > 65535 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return -1;
  if (splits > 1 && (o_part == nullptr || lse_part == nullptr || (reinterpret_cast<uintptr_t>(o_part) & 15) != 0))
    return -1;
  const int kvw = hkv * D;
  CUtensorMap tk, tv, tk8, tv8;
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  if (!cached_tmap_2d(&tk, kq, u8, 1, num_slots, kvw, kvw, 16, 128)) return -2;
  if (!cached_tmap_2d(&tv, vq, u8, 1, num_slots, kvw, kvw, 16, 128)) return -2;
  if (!cached_tmap_2d(&tk8, kq, u8, 1, num_slots, kvw, kvw, 128, 128)) return -2;
  if (!cached_tmap_2d(&tv8, vq, u8, 1, num_slots, kvw, kvw, 128, 128)) return -2;
  Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.ldq = ldq;
  p.T = T;
  p.q_start = q_start;
  p.q_len = q_len;
  p.ctx_len = ctx_len;
  p.n_seqs = n_seqs;
  p.ksf = static_cast<const uint8_t*>(ksf);
  p.vsf = static_cast<const uint8_t*>(vsf);
  p.vq = static_cast<const uint8_t*>(vq);
  p.num_pages = static_cast<int>(num_slots / PAGE);
  p.block_table = block_table;
  p.bt_rows = bt_rows;
  p.table_rows = table_rows;
  p.max_pages = max_pages;
  p.ld_table = ld_table;
  p.hq = hq;
  p.hkv = hkv;
  p.G = hq / hkv;
  p.tokens = 256 / p.G;
  p.splits = splits;
  p.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  p.q_sign = scale < 0.f ? -1.f : (scale == 0.f ? 0.f : 1.f);
  p.o_part = o_part;
  p.lse_part = lse_part;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.status = status;
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    cudaFuncSetAttribute(prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  launch_pdl(prefill_kernel, dim3(hkv, n_items, splits), NUM_THREADS, SMEM_BYTES, stream, tk, tv, tk8, tv8, p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  if (splits > 1) {
    if (merge_warps(static_cast<long long>(n_rows) * hq, splits) > 1)
      launch_pdl(prefill_merge_kernel<MERGE_WARPS>, dim3(n_rows, hq), MERGE_WARPS * 32, 0, stream, p);
    else
      launch_pdl(prefill_merge_kernel<1>, dim3(n_rows, (hq + MERGE_WARPS - 1) / MERGE_WARPS), MERGE_WARPS * 32, 0,
                 stream, p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
}
