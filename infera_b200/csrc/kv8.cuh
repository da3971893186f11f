// What the kernels of the 8-bit KV cache share: e4m3 conversions, powers of
// two, the exponents of pages, and the merge of key shares. The attention
// kernels of the bf16 cache that came after them use the tcgen05 issue, the
// page checks, the reductions and scaled() too.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "sm100.cuh"

namespace ib200 {
namespace kv8 {

constexpr int D = 128;    // head dim
constexpr int PAGE = 16;  // tokens of a page
// Largest biased exponent of a page's scale, so that its inverse is a normal
// number too (bf16 rows need 247 at most).
constexpr int MAX_EXP = 253;

__device__ __forceinline__ float two_to(int e) {  // 2^e, e in [-126, 127]
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
// two values to e4m3 (nearest even, saturating, NaN stays one), and back
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t to_e5m2x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ __half2 from_e4m3x2_h(uint32_t v) {
  return __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v), __NV_E4M3));
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) { return __half22float2(from_e4m3x2_h(v)); }
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// byte offset of (row, byte k) in a block of 128-byte rows, 128-byte swizzle
__device__ __forceinline__ uint32_t sw_offset(int row, int k) {
  return static_cast<uint32_t>(row * 128 + (((k >> 4) ^ (row & 7)) << 4) + (k & 15));
}

__device__ __forceinline__ float max_over_warp(float x) {  // a NaN counts as nothing
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// w x for a weight w; what is not finite stays so where w is 0
__device__ __forceinline__ float scaled(float x, float w) { return fabsf(x) <= FLT_MAX ? x * w : x; }

// ---- tcgen05 issue by a whole warp
// The MMA warp runs its loop with all lanes and issues under the elected
// lane's predicate, not in a branch of one lane: descriptors then stay in
// uniform registers, which the instruction takes. Issued from a branch of one
// lane, each matrix instruction of the prompt kernel took 140 cycles (moves to
// uniform registers, each waited for) where the tensor core needs 32 to 64.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r));
  return r;
}
__device__ __forceinline__ void umma_e4m3_if(uint32_t on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void umma_bf16_if(uint32_t on, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
// A operand in tensor memory, kind::f16
__device__ __forceinline__ void umma_f16_ts_if(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}
// TMA loads by a whole warp in the same way
__device__ __forceinline__ void mbar_expect_tx_if(uint32_t on, uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(bytes), "r"(on)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d_if(uint32_t on, void* dst, const CUtensorMap* tm, uint64_t* bar, int c0,
                                               int c1, uint64_t cache_hint) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;\n\t}\n" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "l"(cache_hint), "r"(on)
      : "memory");
}
// a value that all lanes have, known to be uniform
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

// Row `row` of the page table, which sequence s has; null (and a status) where
// the table has no such row.
__device__ __forceinline__ const int* table_row(const int* table, int row, int table_rows, int ld_table, int s,
                                                int* status) {
  if (row >= 0 && row < table_rows) return table + static_cast<size_t>(row) * ld_table;
  if (threadIdx.x == 0) record_status_detail(status, kStatusBadIndex, 4, s, row);
  return nullptr;
}

// Page ids outside the cache become -1: rows -16 .. -1, which a tensor map
// fills with zeros. (A far id times 16 would wrap to a row that exists.)
__device__ __forceinline__ void known_pages(int (&pages)[8], int num_pages) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (static_cast<unsigned>(pages[i]) >= static_cast<unsigned>(num_pages)) pages[i] = -1;
}

// A stored exponent: 0 counts as 1, 254 and 255 as 253.
__device__ __forceinline__ int exponent_of(uint32_t sf) { return min(max(static_cast<int>(sf), 1), MAX_EXP); }

// The exponents of K and V of a page and head. A page id
// outside the cache (a bad table) loads zeros through the tensor map and takes
// the smallest exponents, as does -1 (no page).
__device__ __forceinline__ void page_exponents(const uint8_t* ksf, const uint8_t* vsf, int num_pages, int hkv,
                                               int kvh, int page, int& ke, int& ve) {
  ke = ve = 1;
  if (page < 0 || page >= num_pages) return;
  const size_t at = static_cast<size_t>(page) * hkv + kvh;
  ke = exponent_of(ksf[at]);
  ve = exponent_of(vsf[at]);
}

// out = sum_s 2^(lse_s - M) o_s / sum_s 2^(lse_s - M) over the shares of one
// row and head, by W warps of a block of MERGE_WARPS (warp w of them takes
// shares w, w + W, ...; a lane has 4 dims and makes the weight of one share in
// 32). A NaN in a share stays one, however small its weight; the output of a
// share whose lse is -inf is not written, and not used. A warp's first four
// shares are loaded before the weights are known. One warp a row is the least work; few rows with many shares wait
// for one load after another then, and take all warps of the block (1 x 120001
// keys, 37 shares: 47 us against 50).
constexpr int MERGE_WARPS = 8;
template <int W>
__device__ __forceinline__ void merge_shares(const float* o_part, const float* lse_part, int splits,
                                             __nv_bfloat16* out) {
  constexpr int AHEAD = 4;
  const int lane = threadIdx.x & 31, w0 = (threadIdx.x >> 5) % W;
  const float4* o = reinterpret_cast<const float4*>(o_part) + w0 * (D / 4) + lane;
  float4 first[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    first[i] = w0 + i * W < splits ? o[i * (W * D / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
  float mx = -INFINITY;
  for (int s = lane; s < splits; s += 32) mx = fmaxf(mx, lse_part[s]);
  mx = max_over_warp(mx);
  if (mx == -INFINITY) mx = 0.f;
  float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
  auto add = [&](float w, const float4& v) {
    if (w == 0.f) return;
    den += w;
    num[0] += v.x * w;
    num[1] += v.y * w;
    num[2] += v.z * w;
    num[3] += v.w * w;
  };
  for (int s0 = w0; s0 < splits; s0 += 32 * W, o += 32 * (W * D / 4)) {
    const int n = min(32, (splits - s0 + W - 1) / W);  // shares s0, s0 + W, ...
    float mine = 0.f;
    if (lane < n) {
      const float lse = lse_part[s0 + lane * W];
      mine = exp2f(lse - mx);
      if (mine == 0.f && lse != -INFINITY) mine = FLT_MIN;
    }
    if (s0 == w0) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) add(__shfl_sync(0xffffffffu, mine, i), first[i]);
    }
#pragma unroll 4
    for (int s = s0 == w0 ? AHEAD : 0; s < n; ++s) add(__shfl_sync(0xffffffffu, mine, s), o[s * (W * D / 4)]);
  }
  if constexpr (W > 1) {
    __shared__ float4 s_num[W][32];
    __shared__ float s_den[W];
    s_num[w0][lane] = make_float4(num[0], num[1], num[2], num[3]);
    if (lane == 0) s_den[w0] = den;
    __syncthreads();
    if (w0 != 0) return;
    for (int w = 1; w < W; ++w) {
      const float4 v = s_num[w][lane];
      den += s_den[w];
      num[0] += v.x;
      num[1] += v.y;
      num[2] += v.z;
      num[3] += v.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) num[i] = den == 0.f ? 0.f : num[i] / den;
  reinterpret_cast<uint32_t*>(out)[lane * 2] = pack_bf16(num[0], num[1]);
  reinterpret_cast<uint32_t*>(out)[lane * 2 + 1] = pack_bf16(num[2], num[3]);
}
// warps per row and head for so many of them
inline int merge_warps(long long rows, int splits) { return rows < 1024 && splits >= 8 ? MERGE_WARPS : 1; }

}  // namespace kv8
}  // namespace ib200
