// The 8-bit paged KV cache: append (with the rotation of q and k) and the
// expansion of pages to bf16 for prompt attention.
//
// One layer's channel (K or V) holds e4m3 codes [num_slots, hkv * 128]
// (slot = page * 16 + offset) and one power-of-two scale per page and head,
// sf uint8 [num_pages, hkv]: value = code * 2^(sf - 127). With a power of two
// a page whose scale grows is rewritten exactly (only codes that become
// subnormal round again), and code * scale is exact in bf16.
//
// Append: a page's scale is the smallest e with amax <= 448 * 2^(e - 127)
// over the finite values of its new rows; a page whose slot 0 is written
// starts anew with that scale, any other keeps at least the one it has and
// its rows are brought to a grown one. The scale joins all rows of a page in
// the batch, wherever they stand in it, so one warp owns a (page, head) of a
// channel: the first row of a page (its leader) looks its page's other rows
// up among all slots of the batch. Nothing depends on the order of arrival.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "sm100.cuh"

namespace ib200 {
namespace kv8 {

constexpr int D = 128;
constexpr int PAGE = 16;
constexpr int WIN = 4;        // batch rows per K/V CTA
constexpr int THREADS = 256;

__device__ __forceinline__ float two_to(int e) {  // 2^e, e in [-126, 127]
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Smallest biased exponent e (1..254) with amax <= 448 * 2^(e - 127);
// 448 = 1.75 * 2^8. amax >= 0 and finite; below 2^-126 it counts as 0.
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(1, min(254, e));
}

__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float2 from_e4m3x2(uint16_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(v, __NV_E4M3);
  return __half22float2(__half2(h));
}

struct Append {
  const __nv_bfloat16* qkv;
  int ldqkv;
  __nv_bfloat16* q_out;
  int ldq;
  const int* pos;
  const int* slots;
  const float* cos_sin;  // [max_pos, 64, 2]
  int T, hq, hkv;
  uint8_t *kq, *ksf, *vq, *vsf;
  long long num_slots;
  int max_pos;
  int* status;
  int kv_ctas;        // CTAs of the K/V part, the rest rotate q
  int head_groups;    // K/V CTAs per window of rows
  int group_heads;    // K and V heads of one such CTA
};

// (a, b) -> (a c - b s, b c + a s), each product and sum rounded on its own:
// the value does not depend on how a compiler contracts it.
__device__ __forceinline__ float rot_a(float a, float b, float c, float s) {
  return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
}
__device__ __forceinline__ float rot_b(float a, float b, float c, float s) {
  return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
}

__device__ __forceinline__ bool bad_pos(const Append& p, int t) {
  const int x = p.pos[t];
  return x < 0 || x >= p.max_pos;
}

__device__ void append_kv(const Append& p) {
  __shared__ int s_page[WIN];
  __shared__ int s_lead[WIN];
  __shared__ int s_row[WIN][PAGE];  // the last valid batch row of each slot of the page
  const int w0 = static_cast<int>(blockIdx.x) / p.head_groups * WIN;
  const int y = static_cast<int>(blockIdx.x) % p.head_groups;
  const int tid = threadIdx.x;
  int lead = 0;
  if (tid < WIN) {
    const int t = w0 + tid;
    const int slot = t < p.T ? p.slots[t] : -1;
    int page = slot < 0 ? -1 : slot / PAGE;
    if (slot >= p.num_slots) {
      page = -1;
      if (y == 0) record_status_detail(p.status, kStatusBadIndex, 2, t, slot);
    }
    // a row right behind one of the same page is not its first
    if (page >= 0 && t > 0 && p.slots[t - 1] >= 0 && p.slots[t - 1] / PAGE == page) page = -1;
    s_page[tid] = page;
    lead = page >= 0;
    s_lead[tid] = lead;
  }
  if (tid < WIN * PAGE) s_row[tid / PAGE][tid % PAGE] = -1;
  if (!__syncthreads_or(lead)) return;
  int pages[WIN];
#pragma unroll
  for (int w = 0; w < WIN; ++w) pages[w] = s_page[w];
  // eight independent loads at a time: the look through a long step's slots
  // waits for memory T / 2048 times
  for (int i0 = tid; i0 < p.T; i0 += 8 * THREADS) {
    int slot[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * THREADS;
      slot[u] = i < p.T ? __ldg(p.slots + i) : -1;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * THREADS;
      const int page = slot[u] < 0 ? -2 : slot[u] / PAGE;
#pragma unroll
      for (int w = 0; w < WIN; ++w) {
        if (page != pages[w]) continue;
        if (i < w0 + w)
          s_lead[w] = 0;  // an earlier row leads this page
        else if (!bad_pos(p, i))
          atomicMax(&s_row[w][slot[u] % PAGE], i);
      }
    }
  }
  __syncthreads();
  const int warp = tid >> 5, lane = tid & 31;
  const int h_end = min(2 * p.hkv, (y + 1) * p.group_heads);
  const int n_heads = h_end - y * p.group_heads;
  for (int task = warp; task < WIN * n_heads; task += THREADS / 32) {
    const int w = task / n_heads;
    if (!s_lead[w]) continue;
    // lane o (of 16) knows the batch row of the page's slot o
    const int my_row = s_row[w][lane % PAGE];
    const uint32_t live = __ballot_sync(0xffffffffu, my_row >= 0) & 0xffffu;
    if (live == 0) continue;  // every row of the page has a bad position
    const int hh = y * p.group_heads + task % n_heads;
    const bool is_v = hh >= p.hkv;
    const int head = is_v ? hh - p.hkv : hh;
    const long long page = pages[w];
    uint8_t* sf = (is_v ? p.vsf : p.ksf) + page * p.hkv + head;
    uint8_t* codes = (is_v ? p.vq : p.kq) + page * PAGE * p.hkv * D + head * D;
    const int e_old = *sf;
    const int my_pos = my_row >= 0 && !is_v ? p.pos[my_row] : 0;
    // this lane: dims 2 lane, 2 lane + 1 and their partners 64 further. All
    // rows are loaded before any is used, without branches: slots that the
    // batch does not write read its first row and count as zeros.
    uint32_t raw[PAGE][2];
#pragma unroll
    for (int o = 0; o < PAGE; ++o) {
      const int row = max(__shfl_sync(0xffffffffu, my_row, o), 0);
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.qkv + static_cast<size_t>(row) * p.ldqkv +
                                                              static_cast<size_t>(p.hq + hh) * D);
      if (live >> o & 1) {
        raw[o][0] = __ldg(src + lane);
        raw[o][1] = __ldg(src + lane + 32);
      } else {
        raw[o][0] = raw[o][1] = 0u;
      }
    }
    // the four values of slot o: made twice (for the maximum and for the
    // codes) rather than held, which halves the registers
    auto values = [&](int o, const float4& cs, float (&x)[4]) {
      const uint32_t a = raw[o][0], b = raw[o][1];
      if (is_v) {
        x[0] = bf16_lo(a);
        x[1] = bf16_hi(a);
        x[2] = bf16_lo(b);
        x[3] = bf16_hi(b);
      } else {
        x[0] = rot_a(bf16_lo(a), bf16_lo(b), cs.x, cs.y);
        x[1] = rot_a(bf16_hi(a), bf16_hi(b), cs.z, cs.w);
        x[2] = rot_b(bf16_lo(a), bf16_lo(b), cs.x, cs.y);
        x[3] = rot_b(bf16_hi(a), bf16_hi(b), cs.z, cs.w);
      }
    };
    auto angles = [&](int o) -> float4 {
      const int pos = __shfl_sync(0xffffffffu, my_pos, o);
      return is_v ? make_float4(0.f, 0.f, 0.f, 0.f)
                  : __ldg(reinterpret_cast<const float4*>(p.cos_sin + static_cast<size_t>(pos) * D) + lane);
    };
    float amax = 0.f;
#pragma unroll
    for (int o0 = 0; o0 < PAGE; o0 += 4) {
      if ((live >> o0 & 0xfu) == 0) continue;
      float4 cs[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) cs[u] = angles(o0 + u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float x[4];
        values(o0 + u, cs[u], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float m = fabsf(x[i]);
          if (m <= FLT_MAX) amax = fmaxf(amax, m);  // finite values set the scale
        }
      }
    }
    // non-negative floats are ordered like their bits
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    const bool anew = live & 1;
    const int e = anew ? scale_exp(amax) : max(scale_exp(amax), e_old);
    const float inv = two_to(127 - e);
    if (!anew && e > e_old) {
      // one rounding more for codes that become subnormal, none for others
      const float f = two_to(max(e_old - e, -60));
      uint32_t old[PAGE];
#pragma unroll
      for (int o = 0; o < PAGE; ++o)
        if (!(live >> o & 1)) old[o] = reinterpret_cast<uint32_t*>(codes + static_cast<size_t>(o) * p.hkv * D)[lane];
#pragma unroll
      for (int o = 0; o < PAGE; ++o) {
        if (live >> o & 1) continue;
        const float2 u = from_e4m3x2(static_cast<uint16_t>(old[o])), v = from_e4m3x2(static_cast<uint16_t>(old[o] >> 16));
        reinterpret_cast<uint32_t*>(codes + static_cast<size_t>(o) * p.hkv * D)[lane] =
            to_e4m3x2(u.x * f, u.y * f) | static_cast<uint32_t>(to_e4m3x2(v.x * f, v.y * f)) << 16;
      }
    }
#pragma unroll
    for (int o0 = 0; o0 < PAGE; o0 += 4) {
      if ((live >> o0 & 0xfu) == 0) continue;
      float4 cs[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) cs[u] = angles(o0 + u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int o = o0 + u;
        float x[4];
        values(o, cs[u], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fabsf(x[i]) <= FLT_MAX ? x[i] * inv : NAN;  // e4m3 has no infinity
        if (live >> o & 1) {
          uint16_t* c = reinterpret_cast<uint16_t*>(codes + static_cast<size_t>(o) * p.hkv * D);
          c[lane] = to_e4m3x2(x[0], x[1]);
          c[lane + 32] = to_e4m3x2(x[2], x[3]);
        }
      }
    }
    if (lane == 0) *sf = static_cast<uint8_t>(e);
  }
}

constexpr int Q_HEADS = 4;  // heads per thread: they share the loaded cos / sin

__device__ __forceinline__ void rotate8(const uint4& a, const uint4& b, const float4 (&cs)[4], uint4* na, uint4* nb) {
  const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
  uint32_t ra[4], rb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ra[i] = pack_bf16(rot_a(bf16_lo(av[i]), bf16_lo(bv[i]), cs[i].x, cs[i].y),
                      rot_a(bf16_hi(av[i]), bf16_hi(bv[i]), cs[i].z, cs[i].w));
    rb[i] = pack_bf16(rot_b(bf16_lo(av[i]), bf16_lo(bv[i]), cs[i].x, cs[i].y),
                      rot_b(bf16_hi(av[i]), bf16_hi(bv[i]), cs[i].z, cs[i].w));
  }
  *na = make_uint4(ra[0], ra[1], ra[2], ra[3]);
  *nb = make_uint4(rb[0], rb[1], rb[2], rb[3]);
}

__device__ void rotate_q(const Append& p) {
  const int ng = (p.hq + Q_HEADS - 1) / Q_HEADS;
  const long long idx = static_cast<long long>(blockIdx.x - p.kv_ctas) * THREADS + threadIdx.x;
  const int c = static_cast<int>(idx & 7);  // dims 8c .. 8c + 7 and their partners
  const long long rest = idx >> 3;
  const long long t = rest / ng;
  if (t >= p.T) return;
  const int h0 = static_cast<int>(rest % ng) * Q_HEADS;
  const int pos = p.pos[t];
  if (pos < 0 || pos >= p.max_pos) {
    if (c == 0 && h0 == 0) record_status_detail(p.status, kStatusBadIndex, 1, static_cast<int>(t), pos);
    return;
  }
  const float4* src = reinterpret_cast<const float4*>(p.cos_sin + static_cast<size_t>(pos) * D + c * 16);
  const float4 cs[4] = {__ldg(src), __ldg(src + 1), __ldg(src + 2), __ldg(src + 3)};
  const __nv_bfloat16* in = p.qkv + t * p.ldqkv + c * 8;
  __nv_bfloat16* out = p.q_out + t * p.ldq + c * 8;
  uint4 a[Q_HEADS], b[Q_HEADS];
#pragma unroll
  for (int i = 0; i < Q_HEADS; ++i)
    if (h0 + i < p.hq) {
      a[i] = *reinterpret_cast<const uint4*>(in + (h0 + i) * D);
      b[i] = *reinterpret_cast<const uint4*>(in + (h0 + i) * D + D / 2);
    }
#pragma unroll
  for (int i = 0; i < Q_HEADS; ++i)
    if (h0 + i < p.hq) {
      uint4 na, nb;
      rotate8(a[i], b[i], cs, &na, &nb);
      *reinterpret_cast<uint4*>(out + (h0 + i) * D) = na;
      *reinterpret_cast<uint4*>(out + (h0 + i) * D + D / 2) = nb;
    }
}

__global__ void __launch_bounds__(THREADS, 3) append_kernel(const Append p) {
  pdl_trigger();
  pdl_wait();
  if (static_cast<int>(blockIdx.x) < p.kv_ctas)
    append_kv(p);
  else
    rotate_q(p);
}

// ---------------------------------------------------------------- expansion

struct Expand {
  const uint8_t *kq, *ksf, *vq, *vsf;
  const int* block_table;
  const int* bt_rows;
  int ld_table;
  const int* ctx_len;
  int hkv, num_pages, most;      // most: pages of the longest sequence
  long long out_pages;           // pages that k_out / v_out hold
  __nv_bfloat16 *k_out, *v_out;  // [out_pages * 16, hkv * 128]
  int* table_out;                // [sequences, most]
  int* status;
};

__device__ __forceinline__ uint4 expand8(uint32_t lo, uint32_t hi, float f) {
  const float2 a = from_e4m3x2(static_cast<uint16_t>(lo)), b = from_e4m3x2(static_cast<uint16_t>(lo >> 16));
  const float2 c = from_e4m3x2(static_cast<uint16_t>(hi)), d = from_e4m3x2(static_cast<uint16_t>(hi >> 16));
  return make_uint4(pack_bf16(a.x * f, a.y * f), pack_bf16(b.x * f, b.y * f), pack_bf16(c.x * f, c.y * f),
                    pack_bf16(d.x * f, d.y * f));
}

// One CTA per page of a sequence: its K and V rows in bf16 at the sequence's
// consecutive pages of the output (sequence after sequence), zeros behind the
// sequence's last row, so that no stale code (a NaN) reaches the tensor core.
__global__ void __launch_bounds__(256) expand_kernel(const Expand p) {
  pdl_trigger();
  pdl_wait();
  const int pg = blockIdx.x, seq = blockIdx.y;
  const int ctx = p.ctx_len[seq];
  if (pg * PAGE >= ctx) return;
  long long base = 0;
  for (int j = 0; j < seq; ++j) base += (max(p.ctx_len[j], 0) + PAGE - 1) / PAGE;
  const long long dst = base + pg;
  if (dst >= p.out_pages) {  // lengths on the device disagree with the host's
    if (threadIdx.x == 0) {
      p.table_out[static_cast<size_t>(seq) * p.most + pg] = 0;
      record_status(p.status, kStatusBadArgs);
    }
    return;
  }
  const int row = p.bt_rows != nullptr ? p.bt_rows[seq] : seq;
  const int page = p.block_table[static_cast<size_t>(row) * p.ld_table + pg];
  const bool ok = page >= 0 && page < p.num_pages;
  if (threadIdx.x == 0) {
    p.table_out[static_cast<size_t>(seq) * p.most + pg] = static_cast<int>(dst);
    if (!ok) record_status_detail(p.status, kStatusBadIndex, 2, seq, page);
  }
  const int rows = min(PAGE, ctx - pg * PAGE);
  const int per_row = p.hkv * (D / 16);  // 16-code pieces of a row
  const int n = PAGE * per_row;
  const size_t src = static_cast<size_t>(ok ? page : 0) * n;
  const uint4* kin = reinterpret_cast<const uint4*>(p.kq) + src;
  const uint4* vin = reinterpret_cast<const uint4*>(p.vq) + src;
  uint4* kout = reinterpret_cast<uint4*>(p.k_out) + static_cast<size_t>(dst) * n * 2;
  uint4* vout = reinterpret_cast<uint4*>(p.v_out) + static_cast<size_t>(dst) * n * 2;
  const uint8_t* ksf = p.ksf + static_cast<size_t>(ok ? page : 0) * p.hkv;
  const uint8_t* vsf = p.vsf + static_cast<size_t>(ok ? page : 0) * p.hkv;
#pragma unroll 2
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const bool live = ok && i / per_row < rows;
    const int head = (i % per_row) / (D / 16);
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (live) {
      a = __ldg(kin + i);
      b = __ldg(vin + i);
    }
    const float fk = two_to(max(static_cast<int>(ksf[head]), 1) - 127);
    const float fv = two_to(max(static_cast<int>(vsf[head]), 1) - 127);
    kout[2 * i] = expand8(a.x, a.y, fk);
    kout[2 * i + 1] = expand8(a.z, a.w, fk);
    vout[2 * i] = expand8(b.x, b.y, fv);
    vout[2 * i + 1] = expand8(b.z, b.w, fv);
  }
}

}  // namespace kv8
}  // namespace ib200

using namespace ib200;

// qkv [T, ldqkv] bf16: q heads at columns [0, hq*128), k behind, then v; the
// rotated q goes to q_out [T, ldq] (which may be qkv itself), k and v to the
// slots (< 0: not stored). cos_sin [max_pos, 64, 2] fp32. Positions and slots
// out of range are recorded in the status word and their row skipped.
extern "C" int ib_kv8_append(const void* qkv, int T, int ldqkv, void* q_out, int ldq, const int* pos,
                             const int* slots, const void* cos_sin, int hq, int hkv, void* kq, void* ksf, void* vq,
                             void* vsf, long long num_slots, int max_pos, int* status, cudaStream_t stream) {
  using namespace ib200::kv8;
  if (T <= 0) return 0;
  if (hq < 1 || hkv < 1 || (ldqkv % 8) != 0 || (ldq % 8) != 0 || num_slots % PAGE != 0) return -1;
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(cos_sin)) &
       15) != 0)
    return -1;
  Append p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.ldqkv = ldqkv;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.ldq = ldq;
  p.pos = pos;
  p.slots = slots;
  p.cos_sin = static_cast<const float*>(cos_sin);
  p.T = T;
  p.hq = hq;
  p.hkv = hkv;
  p.kq = static_cast<uint8_t*>(kq);
  p.ksf = static_cast<uint8_t*>(ksf);
  p.vq = static_cast<uint8_t*>(vq);
  p.vsf = static_cast<uint8_t*>(vsf);
  p.num_slots = num_slots;
  p.max_pos = max_pos;
  p.status = status;
  // few rows: two heads per CTA, so that every (row, head) has a warp of its
  // own; many rows (prompts: one leader in 16 rows): a warp for each of 8 heads
  p.group_heads = T <= 512 ? 2 : 8;
  p.head_groups = (2 * hkv + p.group_heads - 1) / p.group_heads;
  const long long kv_ctas = static_cast<long long>((T + WIN - 1) / WIN) * p.head_groups;
  const long long q_items = static_cast<long long>(T) * ((hq + Q_HEADS - 1) / Q_HEADS) * 8;
  const long long ctas = kv_ctas + (q_items + THREADS - 1) / THREADS;
  if (ctas > 0x7fffffffLL) return -1;
  p.kv_ctas = static_cast<int>(kv_ctas);
  launch_pdl(append_kernel, dim3(static_cast<unsigned>(ctas)), THREADS, 0, stream, p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}

// The pages of n_seqs sequences (ctx_len keys each, block_table rows bt_rows
// or 0, 1, ...) in bf16: k_out / v_out [out_pages * 16, hkv * 128], sequence
// after sequence, and their page table table_out [n_seqs, most]; most: the
// pages of the longest sequence. Rows behind a sequence's last are zero.
extern "C" int ib_kv8_expand(const void* kq, const void* ksf, const void* vq, const void* vsf, int num_pages,
                             int hkv, const int* block_table, const int* bt_rows, int ld_table, const int* ctx_len,
                             int n_seqs, int most, long long out_pages, void* k_out, void* v_out, int* table_out,
                             int* status, cudaStream_t stream) {
  using namespace ib200::kv8;
  if (n_seqs <= 0 || most <= 0) return 0;
  if (hkv < 1 || n_seqs > 65535 || num_pages < 1) return -1;
  Expand p;
  p.kq = static_cast<const uint8_t*>(kq);
  p.ksf = static_cast<const uint8_t*>(ksf);
  p.vq = static_cast<const uint8_t*>(vq);
  p.vsf = static_cast<const uint8_t*>(vsf);
  p.block_table = block_table;
  p.bt_rows = bt_rows;
  p.ld_table = ld_table;
  p.ctx_len = ctx_len;
  p.hkv = hkv;
  p.num_pages = num_pages;
  p.most = most;
  p.out_pages = out_pages;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.table_out = table_out;
  p.status = status;
  launch_pdl(expand_kernel, dim3(most, n_seqs), 256, 0, stream, p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}
