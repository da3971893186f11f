// Paged decode attention (one query token per sequence, GQA) over the 8-bit
// KV cache on tcgen05: the cached e4m3 codes are the tensor core's operands as
// they lie in memory, nothing is converted per cached byte.
//
//   S^T[128 keys, 16]  = K_tile . Q^T     (kind::f8f6f4, A = K codes, K-major)
//   O^T[128 dims, N]   = V_tile^T . W     (A = V codes, MN-major)
//
// Both operands of an f8f6f4 product are 8-bit, so the bf16 query and the
// weights are split into e4m3 digits that stand in columns of their own:
//   q * 2^s = hi + lo / 16            bf16 has 8 significant bits, a digit 4; s
//                                     brings the head's largest element to
//                                     [2^7, 2^8): exact for elements down to
//                                     2^-13 of it, and off by at most 2^-21 of
//                                     it below, where digits are subnormal
//   w       = hi + mid / 32 + lo / 1024  a weight rounded to f16 (11 bits; bf16
//                                     has 8): each digit is rounded to nearest,
//                                     so what is left of it is at most half a
//                                     step, 5 bits further; the last one ends
//                                     at 2^-19
// The 16 columns of S hold both digits of up to 8 heads, so the split costs no
// matrix instruction, and the N columns of O three digits of them.
//
// Scales (one power of two per page and head): K's multiplies a key's scores.
// V's goes into the weight: w = 2^(s - m) * 2^6 * 2^(vsf - R), with R the
// largest V exponent of the split's pages so far and m the running maximum
// that may lag by 2^2, so that w <= 2^8 < 448; a weight is off by at most
// max(2^-12 w, 2^-20), the latter 2^-26 of the largest one. The sum of the
// softmax takes the fp32 weight. When m or R grows, O^T is rescaled in TMEM.
//
// A tile costs few instructions per score, because 4 warps have to keep up
// with 32 KB of K and V: a tile first only asks whether any score is above its
// head's running maximum by more than the lag (one compare per score, one
// barrier with an OR); the maxima themselves are reduced when one is, in the
// first tile and rarely after it. The digits are made in packed f16, and a
// key's digits of all heads are one or two 16-byte stores (the weights' tile
// has the columns adjacent, an MN-major operand).
//
// One CTA handles (sequence, KV head, KV split) and walks its share of the
// sequence in tiles of 128 keys (8 pages), 32 KB for K and V:
//   warp 0      TMA producer: lane 0 K tiles, lane 1 V tiles
//   warp 1      MMA issuer
//   warps 2..5  thread <-> key row for the softmax; they also stage Q
// Pages that a sequence does not have are not loaded. V rows of the last tile
// behind the sequence are zeroed in shared memory: a stale code there may be a
// NaN, which a zero weight does not cancel (stale K rows only give masked
// scores).
// Split partials (output normalised by its own sum, LSE in log2 units) are
// merged by a combine kernel.
//
// Bound by HBM: two 8-bit codes per key, dim and KV head. Captured calls of 32
// sequences of 8192 keys (64 heads over 8) take 87 to 89 us (6.1 TB/s, 0.93 of
// the copy rate), of 61 ragged ones on scattered pages (32 over 8) 124 to 126 us
// (0.90: boxes of 2 KB), of one of 120001 keys 44 us (0.85, with its start and
// the merge of 53 shares), of one of 100 keys 5.5 us. Eager calls on changing
// inputs take 89 to 94 (0.87), 127 to 135 (0.83), 43 to 45 and, bound by the
// host, 16 us.
#include "kv8.cuh"
#include "tma_host.h"

namespace ib200 {
namespace dq8 {

using namespace kv8;

constexpr int BKV = 128;
constexpr int BLK = 128 * 128;      // 128 rows x 128 codes
constexpr int NS = 16;              // columns of S
constexpr int QBLK = NS * 128;
constexpr int NUM_THREADS = 192;
constexpr float kLagLog2 = 2.0f;    // the running maximum may lag by this much
constexpr int kTopLog2 = 6;         // weight of a key at the running maximum

// Stages of K and V tiles, and CTAs per SM. Three CTAs of two stages hide a
// tile's chain (S, softmax, W V) better than two of three where a tile has few
// heads: 61 ragged sequences on scattered pages (4 heads) 125 us against 132,
// 1 x 120001 43.5 against 45.5. Eight heads need the registers of two CTAs,
// and the third stage: 32 x 8192 scattered 96 us against 112 with two.
__host__ __device__ constexpr int stages(int gp) { return gp <= 4 ? 2 : 3; }
// columns of O^T: three digits of GP heads
__host__ __device__ constexpr int cols_o(int gp) { return 3 * gp <= 16 ? 16 : 32; }
__host__ __device__ constexpr int smem_bytes(int gp) {
  return 1024 + stages(gp) * 2 * BLK + QBLK + 2 * cols_o(gp) * 128 + 2048;
}
constexpr int SF_TILES = 16;        // tiles whose page exponents are staged at a time: a page per softmax thread
constexpr uint32_t TMEM_COLS = 64;  // S0 [0,16) S1 [16,32) O [32,64)
constexpr uint32_t O_COL = 32;

struct Params {
  const __nv_bfloat16* q;
  int ldq;
  const uint8_t* ksf;
  const uint8_t* vsf;
  int num_pages;
  const int* block_table;
  const int* bt_rows;
  const int* seq_lens;
  int table_rows, max_pages, ld_table;  // rows of the block table, places of a row, and its pitch
  int hq, hkv, G;
  int splits;
  int tiles_per_split;  // split s covers tiles [s * this, (s + 1) * this) of every sequence
  float scale_log2;  // |scale| * log2(e)
  float q_sign;      // sign of the scale (0: every score is 0)
  float* o_part;    // [B, hq, splits, D]
  float* lse_part;  // [B, hq, splits]
  __nv_bfloat16* out;
  int ldo;
  int* status;
};

// The leading e4m3 digits of two f16 values (|x| <= 256), and the rest of the
// values after it, 32 times larger (exact in f16).
__device__ __forceinline__ uint32_t digit2(__half2& x) {
  const __half2_raw raw = x;
  const uint32_t d = __nv_cvt_halfraw2_to_fp8x2(raw, __NV_SATFINITE, __NV_E4M3);
  x = __hmul2(__hsub2(x, from_e4m3x2_h(d)), __float2half2_rn(32.f));
  return d;
}
// Barrier of the four softmax warps that ORs a predicate. Every one of them
// passes the same number of these, whatever a bounded wait in between gave,
// so none is left waiting.
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

template <int GP>  // query heads per KV head, rounded up to 1, 2, 4 or 8
__global__ void __launch_bounds__(NUM_THREADS, GP <= 4 ? 3 : 2)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmK8, const __grid_constant__ CUtensorMap tmV8,
                  const Params p) {
  constexpr int STAGES = stages(GP);
  constexpr int NO = cols_o(GP);
  constexpr int NC = NO / 16;           // 16-byte pieces of a key's digits
  constexpr int PBLK = NO * 128;
  constexpr int ND = 3 * GP;            // digits of a key's weights
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.x, b = blockIdx.y, split = blockIdx.z;
  const int G = p.G;
  const int table = p.bt_rows != nullptr ? p.bt_rows[b] : b;
  int len = max(p.seq_lens[b], 0);
  if (len > p.max_pages * PAGE) {  // more keys than the page table has places for
    if (threadIdx.x == 0) record_status_detail(p.status, kStatusBadIndex, 1, b, len);
    len = p.max_pages * PAGE;
  }
  const int* bt = table_row(p.block_table, table, p.table_rows, p.ld_table, b, p.status);
  if (bt == nullptr) len = 0;
  const int n_tiles = (len + BKV - 1) / BKV;
  if (split == p.splits - 1 && n_tiles > p.splits * static_cast<long long>(p.tiles_per_split) && threadIdx.x == 0)
    record_status_detail(p.status, kStatusBadArgs, 5, b, len);  // keys that no split takes
  // (in 64 bits: the caller's product may pass 32)
  const int t0 = static_cast<int>(min(static_cast<long long>(n_tiles), static_cast<long long>(split) * p.tiles_per_split));
  const int t1 = static_cast<int>(min(static_cast<long long>(n_tiles), static_cast<long long>(t0) + p.tiles_per_split));
  if (t0 >= t1) {  // nothing in this split
    if (p.splits > 1) {
      if (threadIdx.x < G)
        p.lse_part[(static_cast<size_t>(b) * p.hq + kvh * G + threadIdx.x) * p.splits + split] = -INFINITY;
    } else {
      for (int i = threadIdx.x; i < G * D; i += blockDim.x)
        p.out[static_cast<size_t>(b) * p.ldo + kvh * G * D + i] = __float2bfloat16(0.f);
    }
    return;
  }
  const int nt = t1 - t0;
  const int n_pages = (len + PAGE - 1) / PAGE;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sKV = smem;                        // stage s: K, V
  uint8_t* sQ = smem + STAGES * 2 * BLK;      // rows: hi digits of GP heads, lo digits
  uint8_t* sP = sQ + QBLK;                    // [2] columns: digit d of head h at d * GP + h
  uint64_t* bars = reinterpret_cast<uint64_t*>(sP + 2 * PBLK);
  uint64_t* k_full = bars;
  uint64_t* v_full = k_full + STAGES;
  uint64_t* k_empty = v_full + STAGES;
  uint64_t* v_empty = k_empty + STAGES;
  uint64_t* s_full = v_empty + STAGES;        // [2]
  uint64_t* p_full = s_full + 2;              // [2] one per P buffer
  uint64_t* pv_done = p_full + 2;             // [2] PV of tile j commits to pv_done[j & 1]
  uint64_t* q_ready = pv_done + 2;
  uint64_t* drain = q_ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* red = reinterpret_cast<float*>(tmem_slot + 4);     // [4][GP] tile maxima, then sums
  int* redv = reinterpret_cast<int*>(red + 4 * GP);         // [4] V exponents
  float* qsc = reinterpret_cast<float*>(redv + 4);          // [GP] scale_log2 * 2^-s
  uint16_t* sSf = reinterpret_cast<uint16_t*>(qsc + GP);    // [2][128] exponents (K low byte, V high) of a batch's pages

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
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
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane < 2) {
      const bool is_v = lane == 1;
      const CUtensorMap* tm1 = is_v ? &tmV : &tmK;
      const CUtensorMap* tm8 = is_v ? &tmV8 : &tmK8;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      uint8_t* dst0 = sKV + (is_v ? BLK : 0);
      const uint64_t pol = policy_evict_first();
      int issued = 0;
      int nxt[8];
      load_tile_pages(bt, t0, n_pages, nxt);
      for (int j = 0; j < nt; ++j) {
        const int st = j % STAGES;
        int cur[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cur[i] = nxt[i];
        known_pages(cur, p.num_pages);
        if (j + 1 < nt) load_tile_pages(bt, t0 + j + 1, n_pages, nxt);  // in flight while we wait
        if (!mbar_wait(&empty[st], static_cast<uint32_t>(((j / STAGES) & 1) ^ 1), abort_flag, p.status,
                       kStatusTimeoutEmpty))
          break;
        uint8_t* dst = dst0 + st * 2 * BLK;
        // eight consecutive pages are one 128-row box (the swizzle repeats
        // every 8 rows: the same image as eight page boxes)
        bool run = true;
#pragma unroll
        for (int pg = 1; pg < BKV / PAGE; ++pg) run = run && cur[pg] == cur[0] + pg;
        const int n = min(BKV / PAGE, n_pages - (t0 + j) * (BKV / PAGE));  // pages that the sequence has here
        mbar_expect_tx(&full[st], n * PAGE * 128);
        if (run && n == BKV / PAGE) {
          tma_load_2d(dst, tm8, &full[st], kvh * D, cur[0] * PAGE, pol);
        } else {
#pragma unroll
          for (int pg = 0; pg < BKV / PAGE; ++pg)
            if (pg < n) tma_load_2d(dst + pg * PAGE * 128, tm1, &full[st], kvh * D, cur[pg] * PAGE, pol);
        }
        ++issued;
      }
      for (int i = max(0, issued - STAGES); i < issued; ++i)
        mbar_wait(&full[i % STAGES], static_cast<uint32_t>((i / STAGES) & 1), nullptr, nullptr, 0, kWaitLimitNs / 4);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc_s = make_idesc_e4m3(128, NS);
      const uint32_t idesc_o = make_idesc_e4m3(128, NO) | (1u << 15) | (1u << 16);  // both MN-major
      const uint32_t q_addr = smem_u32(sQ);
      const uint32_t p_addr = smem_u32(sP);
      bool ok = mbar_wait(q_ready, 0, abort_flag, p.status, kStatusTimeoutFull);
      tc_fence_after();
      auto issue_pv = [&](int jj) -> bool {
        const int st = jj % STAGES;
        if (!mbar_wait(&p_full[jj & 1], static_cast<uint32_t>((jj >> 1) & 1), abort_flag, p.status,
                       kStatusTimeoutTmemEmpty))
          return false;
        if (!mbar_wait(&v_full[st], static_cast<uint32_t>((jj / STAGES) & 1), abort_flag, p.status,
                       kStatusTimeoutFull))
          return false;
        tc_fence_after();
        const uint32_t v_addr = smem_u32(sKV + st * 2 * BLK + BLK);
        const uint32_t pb = p_addr + static_cast<uint32_t>((jj & 1) * PBLK);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          // 32 keys: four groups of 8 rows, 1024 bytes apart (the stride);
          // all 128 dims are one 128-byte row, so the leading offset is unused
          const uint64_t ad = make_sw128_desc(v_addr + s * 4096, BLK, 1024);
          const uint64_t bd = make_mn_desc(pb + s * 4 * NC * 128, 128, NC * 128);
          umma_e4m3(tmem + O_COL, ad, bd, idesc_o, (jj > 0 || s > 0) ? 1u : 0u);
        }
        umma_commit(&pv_done[jj & 1]);
        umma_commit(&v_empty[st]);
        return true;
      };
      for (int j = 0; j < nt && ok; ++j) {
        const int st = j % STAGES;
        if (!mbar_wait(&k_full[st], static_cast<uint32_t>((j / STAGES) & 1), abort_flag, p.status,
                       kStatusTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t k_addr = smem_u32(sKV + st * 2 * BLK);
#pragma unroll
        for (int s = 0; s < 4; ++s)
          umma_e4m3(tmem + ((j & 1) ? NS : 0), make_sw128_desc(k_addr + s * 32, 16, 1024),
                    make_sw128_desc(q_addr + s * 32, 16, 1024), idesc_s, s > 0 ? 1u : 0u);
        umma_commit(&s_full[j & 1]);
        umma_commit(&k_empty[st]);
        if (j > 0 && !issue_pv(j - 1)) {
          ok = false;
          break;
        }
      }
      if (ok) issue_pv(nt - 1);
      umma_commit(drain);
      mbar_wait(drain, 0, nullptr, p.status, kStatusTimeoutFull);
    }
  } else {
    const int t = threadIdx.x - 64;   // 0..127
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;     // key row of S, dim row of O
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    bool ok = true;
    // exponents of the split's pages, of 16 tiles at a time: one page per thread
    const int end_page = min(n_pages, t1 * (BKV / PAGE));
    auto page_of = [&](int j) -> int {
      const int lp = (t0 + j) * (BKV / PAGE) + t;
      return lp < end_page ? __ldg(bt + lp) : -1;
    };
    auto load_sf = [&](int page) -> uint32_t {
      int ke, ve;
      page_exponents(p.ksf, p.vsf, p.num_pages, p.hkv, kvh, page, ke, ve);
      return static_cast<uint32_t>(ke | ve << 8);
    };
    uint32_t sf_next = load_sf(page_of(0));  // this thread's page of the next batch
    int page_next = -1;

    // stage Q: unused rows of Q are zero
    for (int i = t; i < QBLK / 16; i += 128) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    barrier_or(false);
    for (int h = q4; h < G; h += 4) {
      const uint32_t* src =
          reinterpret_cast<const uint32_t*>(p.q + static_cast<size_t>(b) * p.ldq + (kvh * G + h) * D) + lane * 2;
      const uint32_t u0 = src[0], u1 = src[1];
      float x[4] = {bf16_lo(u0), bf16_hi(u0), bf16_lo(u1), bf16_hi(u1)};
      float mx = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
      const uint32_t mb = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));
      const int s = min(100, 134 - static_cast<int>(mb >> 23));
      const float f = two_to(s) * p.q_sign;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = fabsf(x[i]) <= 3.4e38f ? x[i] * f : NAN;
      const uint32_t h01 = to_e4m3x2(x[0], x[1]), h23 = to_e4m3x2(x[2], x[3]);
      const float2 a = from_e4m3x2(h01), c = from_e4m3x2(h23);
      *reinterpret_cast<uint32_t*>(sQ + sw_offset(h, lane * 4)) = h01 | (h23 << 16);
      *reinterpret_cast<uint32_t*>(sQ + sw_offset(GP + h, lane * 4)) =
          to_e4m3x2((x[0] - a.x) * 16.f, (x[1] - a.y) * 16.f) |
          (to_e4m3x2((x[2] - c.x) * 16.f, (x[3] - c.y) * 16.f) << 16);
      if (lane == 0) qsc[h] = fmaxf(p.scale_log2 * two_to(-s), 1.2e-38f);  // positive: masked scores are -inf times it
    }
    fence_proxy_async_smem();
    mbar_arrive(q_ready);
    barrier_or(false);  // qsc

    // a head's scores are c * x, its running maximum m; a score above `limit`
    // is above the maximum by more than the lag
    float m_run[GP], limit[GP], l_part[GP], c_h[GP];
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      m_run[h] = 0.f;
      limit[h] = h < G ? -INFINITY : INFINITY;
      l_part[h] = 0.f;
      c_h[h] = h < G ? qsc[h] : 0.f;
    }
    int R = 1;  // largest V exponent of the batches so far
    // the PV of tile jj has completed: its commit is completion (jj >> 1) + 1
    // of pv_done[jj & 1], and no later PV on that barrier can have been issued
    auto wait_pv = [&](int jj) {
      if (ok) ok = mbar_wait_warp(&pv_done[jj & 1], static_cast<uint32_t>((jj >> 1) & 1), abort_flag, p.status,
                                  kStatusTimeoutTmemFull);
      tc_fence_after();
    };
    // O^T *= f, a factor per head, once the PV of tile jj has landed
    auto rescale = [&](int jj, const float (&f)[GP]) {
      wait_pv(jj);
      uint32_t ov[NO];
      if constexpr (NO == 16)
        tmem_ld16(lane_addr + O_COL, ov);
      else
        tmem_ld32(lane_addr + O_COL, ov);
      tmem_ld_wait();
#pragma unroll
      for (int n = 0; n < ND; ++n) ov[n] = __float_as_uint(__uint_as_float(ov[n]) * f[n % GP]);
      if constexpr (NO == 16)
        tmem_st16(lane_addr + O_COL, ov);
      else
        tmem_st32(lane_addr + O_COL, ov);
      tmem_st_wait();
    };
    for (int j = 0; j < nt; ++j) {
      const int in_batch = j % SF_TILES;
      uint16_t* sf = sSf + ((j / SF_TILES) & 1) * 128;
      if (in_batch == 0) {
        sf[t] = static_cast<uint16_t>(sf_next);
        const uint32_t v = __reduce_max_sync(0xffffffffu, sf_next >> 8);
        if (lane == 0) redv[q4] = static_cast<int>(v);
        barrier_or(false);
        const int batch_v = max(max(redv[0], redv[1]), max(redv[2], redv[3]));
        if (batch_v > R) {
          if (j > 0) {
            float f[GP];
#pragma unroll
            for (int h = 0; h < GP; ++h) f[h] = two_to(max(R - batch_v, -126));
            rescale(j - 1, f);
          }
          R = batch_v;
        }
        page_next = page_of(j + SF_TILES);
      } else if (in_batch == 4) {
        sf_next = load_sf(page_next);
      }
      if (ok) ok = mbar_wait_warp(&s_full[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag, p.status,
                                  kStatusTimeoutTmemFull);
      tc_fence_after();
      uint32_t sv[16];
      tmem_ld16(lane_addr + ((j & 1) ? NS : 0), sv);
      const uint32_t e = sf[in_batch * (BKV / PAGE) + (r >> 4)];
      const float kf = two_to(static_cast<int>(e & 255) - 127);
      const float vf = two_to(max(kTopLog2 + static_cast<int>(e >> 8) - R, -126));
      const bool last = (t0 + j + 1) * BKV > len;  // only here are rows masked
      const bool valid = !last || (t0 + j) * BKV + r < len;
      tmem_ld_wait();
      float x[GP];
      bool above = false;
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        x[h] = fmaf(__uint_as_float(sv[GP + h]), 0.0625f, __uint_as_float(sv[h])) * kf;
        if (!valid) x[h] = -INFINITY;
        above = above || x[h] > limit[h];
      }
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
            const float m = tmax * c_h[h];
            f[h] = limit[h] == -INFINITY ? 0.f : exp2f(m_run[h] - m);  // nothing before it: all zeros
            m_run[h] = m;
            limit[h] = (m + kLagLog2) / c_h[h];
            l_part[h] *= f[h];
          }
        }
        if (j > 0) rescale(j - 1, f);
        barrier_or(false);  // red is read
      }
      uint32_t d[NO / 4];  // digit bytes by column
#pragma unroll
      for (int i = 0; i < NO / 4; ++i) d[i] = 0u;
#pragma unroll
      for (int h = 0; h < GP; h += 2) {
        const float p0 = exp2f(fmaf(x[h], c_h[h], -m_run[h]));
        l_part[h] += p0;
        float p1 = 0.f;
        if (h + 1 < GP) {
          p1 = exp2f(fmaf(x[h + (GP > 1)], c_h[h + (GP > 1)], -m_run[h + (GP > 1)]));
          l_part[h + (GP > 1)] += p1;
        }
        __half2 w = __floats2half2_rn(p0 * vf, p1 * vf);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const int n = k * GP + h;
          const uint32_t u = k < 2 ? digit2(w) : __nv_cvt_halfraw2_to_fp8x2(w, __NV_SATFINITE, __NV_E4M3);
          d[n / 4] |= (GP > 1 ? u : (u & 0xffu)) << (8 * (n % 4));
        }
      }
      // P buffer j & 1 was last read by the PV of tile j - 2
      if (j >= 2) wait_pv(j - 2);
      uint8_t* pbuf = sP + (j & 1) * PBLK + (r >> 3) * (NC * 128) + (r & 7) * 16;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        *reinterpret_cast<uint4*>(pbuf + c * 128) = make_uint4(d[4 * c], d[4 * c + 1], d[4 * c + 2], d[4 * c + 3]);
      if (last) {
        // no stale V code behind the sequence reaches the product
        const int st = j % STAGES;
        if (ok) ok = mbar_wait_warp(&v_full[st], static_cast<uint32_t>((j / STAGES) & 1), abort_flag, p.status,
                                    kStatusTimeoutFull);
        if (!valid) {
          uint4* row = reinterpret_cast<uint4*>(sKV + st * 2 * BLK + BLK + r * 128);
#pragma unroll
          for (int i = 0; i < 8; ++i) row[i] = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(&p_full[j & 1]);
    }
    wait_pv(nt - 1);
    uint32_t ov[NO];
    if constexpr (NO == 16)
      tmem_ld16(lane_addr + O_COL, ov);
    else
      tmem_ld32(lane_addr + O_COL, ov);
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
    const float back = two_to(R - 127);  // (times 2^-kTopLog2 it may be too small for a normal number)
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      if (h >= G || !ok) break;
      const float l = red[h] + red[GP + h] + red[2 * GP + h] + red[3 * GP + h];
      const float acc = fmaf(fmaf(__uint_as_float(ov[2 * GP + h]), 0.03125f, __uint_as_float(ov[GP + h])), 0.03125f,
                             __uint_as_float(ov[h]));
      const float o = l == 0.f ? 0.f : acc / l * (1.f / (1 << kTopLog2)) * back;
      const int head = kvh * G + h;
      if (p.splits == 1) {
        p.out[static_cast<size_t>(b) * p.ldo + head * D + r] = __float2bfloat16(o);
      } else {
        const size_t slot = (static_cast<size_t>(b) * p.hq + head) * p.splits + split;
        p.o_part[slot * D + r] = o;
        if (r == 0) p.lse_part[slot] = l == 0.f ? -INFINITY : m_run[h] + log2f(l);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

template <int W>
__global__ void __launch_bounds__(MERGE_WARPS * 32) combine_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, h = blockIdx.y * (MERGE_WARPS / W) + (threadIdx.x >> 5) / W;
  if (h >= p.hq) return;
  const size_t part = (static_cast<size_t>(b) * p.hq + h) * p.splits;
  merge_shares<W>(p.o_part + part * D, p.lse_part + part, p.splits, p.out + static_cast<size_t>(b) * p.ldo + h * D);
}

using Kernel = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap, const Params);

}  // namespace dq8
}  // namespace ib200

using namespace ib200;

// q [B, ldq] bf16 (head h at columns h*128); kq / vq e4m3 [num_slots, hkv*128]
// and ksf / vsf [num_slots/16, hkv]; block_table [table_rows] rows of
// max_pages places (pitch ld_table), row bt_rows[b] (null: b); split s covers the 128-key tiles
// [s*tiles_per_split, (s+1)*tiles_per_split) of every sequence
// (splits*tiles_per_split*128 must cover the longest one); o_part / lse_part:
// fp32 [B*hq*splits*128] / [B*hq*splits], only touched when splits > 1.
extern "C" int ib_attn_decode_kv8(const void* q, int ldq, const void* kq, const void* ksf, const void* vq,
                                  const void* vsf, long long num_slots, const int* block_table, const int* bt_rows,
                                  const int* seq_lens, int table_rows, int max_pages, int ld_table, int B, int hq,
                                  int hkv, int splits, int tiles_per_split, float scale, float* o_part, float* lse_part, void* out,
                                  int ldo, int* status, cudaStream_t stream) {
  using namespace ib200::dq8;
  if (B <= 0) return 0;
  if (hkv <= 0 || hq % hkv != 0 || hq / hkv > 8 || splits < 1 || tiles_per_split < 1 || (ldq % 2) != 0 ||
      B > 65535 || splits > 65535 || num_slots < PAGE || num_slots % PAGE != 0 || max_pages < 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 3) != 0 || (ldo % 2) != 0)
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
  p.ksf = static_cast<const uint8_t*>(ksf);
  p.vsf = static_cast<const uint8_t*>(vsf);
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
  p.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  p.q_sign = scale < 0.f ? -1.f : (scale == 0.f ? 0.f : 1.f);
  p.o_part = o_part;
  p.lse_part = lse_part;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.status = status;
  const int gp = p.G <= 1 ? 1 : (p.G <= 2 ? 2 : (p.G <= 4 ? 4 : 8));
  const Kernel k = gp == 1 ? decode_kernel<1> : (gp == 2 ? decode_kernel<2> : (gp == 4 ? decode_kernel<4> : decode_kernel<8>));
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    cudaFuncSetAttribute(decode_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(1));
    cudaFuncSetAttribute(decode_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(2));
    cudaFuncSetAttribute(decode_kernel<4>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(4));
    cudaFuncSetAttribute(decode_kernel<8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(8));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  launch_pdl(k, dim3(hkv, B, splits), NUM_THREADS, smem_bytes(gp), stream, tk, tv, tk8, tv8, p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  if (splits > 1) {
    if (merge_warps(static_cast<long long>(B) * hq, splits) > 1)
      launch_pdl(combine_kernel<MERGE_WARPS>, dim3(B, hq), MERGE_WARPS * 32, 0, stream, p);
    else
      launch_pdl(combine_kernel<1>, dim3(B, (hq + MERGE_WARPS - 1) / MERGE_WARPS), MERGE_WARPS * 32, 0, stream, p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
}
