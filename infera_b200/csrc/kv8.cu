// Append to the 8-bit paged KV cache, with the rotation of q and k.
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
// channel (of four heads, where the page has but one row): the first row of a
// page (its leader) looks its page's other rows up among all slots of the batch. Nothing depends on the order of arrival.
// Bound by HBM for prompts and by latency for single rows: 8192 rows of 32 + 2 x
// 8 heads take 38 us (189 MB: 5.0 TB/s, 0.76 of the copy rate), 2048 rows 12.3
// us, 256 decoding rows 5.5 us, one 3.1 us. What it took (8192 rows): a warp
// loads all 16 rows of a page before it uses any, 16 bytes a lane (100 us with
// a row at a time), and makes the rotated values twice rather than hold them
// (80 registers, 3 CTAs per SM); infinities are looked for only where the
// largest value is one (40.2 us, 41.2 with a test of each value); a page's
// angles come from shared memory (38.1). Of a page with one new row a warp
// takes four heads (256 decoding rows 5.5 us, 7.5 with a warp for each head; 128
// beside a prompt's 1500 rows 12.7 us, 23.8). Spreading the K/V CTAs among those
// that rotate q gained nothing, nor did a prefetch of a leader's next rows.
#include <float.h>

#include "kv8.cuh"

namespace ib200 {
namespace kv8 {

constexpr int WIN = 8;        // most batch rows per K/V CTA
constexpr int THREADS = 256;

// Smallest biased exponent e (1..253) with amax <= 448 * 2^(e - 127);
// 448 = 1.75 * 2^8. amax >= 0 and finite; below 2^-126 it counts as 0.
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(1, min(MAX_EXP, e));
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
  int kv_ctas;        // CTAs of the K/V part, the others rotate q
  int win;            // batch rows per K/V CTA
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

// The codes of dims 8 c .. 8 c + 7 (v.x, v.y) and their partners (v.z, v.w);
// e4m3 has no infinity, so where values may be one it becomes NaN.
__device__ __forceinline__ uint4 codes_of(float (&x)[16], float inv, bool inf) {
  if (inf)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = fabsf(x[i]) <= FLT_MAX ? x[i] : NAN;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] *= inv;
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = to_e4m3x2(x[4 * i], x[4 * i + 1]) | to_e4m3x2(x[4 * i + 2], x[4 * i + 3]) << 16;
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A lane's values of a row: a and b as they are, or rotated.
__device__ __forceinline__ void unpack16(const uint4& a, const uint4& b, float (&x)[16]) {
  const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(av[i]);
    x[2 * i + 1] = bf16_hi(av[i]);
    x[8 + 2 * i] = bf16_lo(bv[i]);
    x[8 + 2 * i + 1] = bf16_hi(bv[i]);
  }
}
__device__ __forceinline__ void rotate16(const uint4& a, const uint4& b, const float4 (&cs)[4], float (&x)[16]) {
  const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = rot_a(bf16_lo(av[i]), bf16_lo(bv[i]), cs[i].x, cs[i].y);
    x[2 * i + 1] = rot_a(bf16_hi(av[i]), bf16_hi(bv[i]), cs[i].z, cs[i].w);
    x[8 + 2 * i] = rot_b(bf16_lo(av[i]), bf16_lo(bv[i]), cs[i].x, cs[i].y);
    x[8 + 2 * i + 1] = rot_b(bf16_hi(av[i]), bf16_hi(bv[i]), cs[i].z, cs[i].w);
  }
}

// The page's codes at `at` (16 of them) under a scale that grew by 1 / f: one
// rounding more for codes that become subnormal, none for others.
__device__ __forceinline__ void shrink(uint4* at, float f) {
  const uint4 old = *at;
  uint32_t v[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u0 = from_e4m3x2(v[i] & 0xffffu), u1 = from_e4m3x2(v[i] >> 16);
    v[i] = to_e4m3x2(u0.x * f, u0.y * f) | to_e4m3x2(u1.x * f, u1.y * f) << 16;
  }
  *at = make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ bool bad_pos(const Append& p, int t) {
  const int x = p.pos[t];
  return x < 0 || x >= p.max_pos;
}

__device__ void append_kv(const Append& p, int cta) {
  __shared__ int s_page[WIN];       // pages that start in this window
  __shared__ int s_first[WIN];      // and their first rows here
  __shared__ int s_lead[WIN];       // 0: an earlier row, of another window, leads the page
  __shared__ int s_row[WIN][PAGE];  // the last valid batch row of each slot of the page
  __shared__ int s_n;
  __shared__ float4 s_cs[PAGE][D / 4];  // (cos, sin) of a page's rows, see below
  const int w0 = cta / p.head_groups * p.win;
  const int y = cta % p.head_groups;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) {
    const int t = w0 + lane;
    const int slot = lane < p.win && t < p.T ? p.slots[t] : -1;
    const int before = slot >= 0 && t > 0 ? p.slots[t - 1] : -1;
    if (slot >= p.num_slots && y == 0) record_status_detail(p.status, kStatusBadIndex, 2, t, slot);
    // a row right behind one of the same page is not its first
    const bool lead = slot >= 0 && slot < p.num_slots && (before < 0 || before / PAGE != slot / PAGE);
    const uint32_t leads = __ballot_sync(0xffffffffu, lead);
    if (lead) {
      const int n = __popc(leads & ((1u << lane) - 1u));
      s_page[n] = slot / PAGE;
      s_first[n] = t;
      s_lead[n] = 1;
    }
    if (lane == 0) s_n = __popc(leads);
  }
  if (tid < WIN * PAGE) s_row[tid / PAGE][tid % PAGE] = -1;
  __syncthreads();
  const int n_lead = s_n;
  if (n_lead == 0) return;
  auto found = [&](int w, int i, int off) {  // row i writes slot `off` of page w
    if (i < s_first[w])
      s_lead[w] = 0;  // an earlier row leads this page
    else if (!bad_pos(p, i))
      atomicMax(&s_row[w][off], i);
  };
  // all loads of 8192 slots in flight at once: a long step's slots are waited
  // for once
  const int n4 = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0 ? p.T / 4 : 0;
  for (int i0 = tid; i0 < n4; i0 += 8 * THREADS) {
    int4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * THREADS;
      v[u] = i < n4 ? __ldg(reinterpret_cast<const int4*>(p.slots) + i) : make_int4(-1, -1, -1, -1);
    }
    for (int w = 0; w < n_lead; ++w) {
      const int base = s_page[w] * PAGE;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * THREADS;
        if (i >= n4) break;
        const unsigned o0 = v[u].x - base, o1 = v[u].y - base, o2 = v[u].z - base, o3 = v[u].w - base;
        if (min(min(o0, o1), min(o2, o3)) < PAGE) {
          if (o0 < PAGE) found(w, 4 * i, o0);
          if (o1 < PAGE) found(w, 4 * i + 1, o1);
          if (o2 < PAGE) found(w, 4 * i + 2, o2);
          if (o3 < PAGE) found(w, 4 * i + 3, o3);
        }
      }
    }
  }
  for (int i = 4 * n4 + tid; i < p.T; i += THREADS) {
    const int slot = __ldg(p.slots + i);
    for (int w = 0; w < n_lead; ++w) {
      const unsigned off = slot - s_page[w] * PAGE;
      if (off < PAGE) found(w, i, off);
    }
  }
  __syncthreads();
  const int h_end = min(2 * p.hkv, (y + 1) * p.group_heads);
  const int n_heads = h_end - y * p.group_heads;
  // A CTA with one page and a head for every warp, K heads among them, loads the page's angles
  // once for all of them, in the order in which the eight lanes of a row read
  // them: lane c's float4 i at 8 i + c. (From global memory a lane's 64 bytes
  // lie beside its neighbour's, so that each load of a warp touches 16 lines.)
  const bool staged = n_lead == 1 && n_heads == THREADS / 32 && y * p.group_heads < p.hkv;
  // the slots that the batch writes of page w
  auto live_of = [&](int w) { return __ballot_sync(0xffffffffu, lane < PAGE && s_row[w][lane % PAGE] >= 0); };
  // Eight lanes have a row: dims 8 c .. 8 c + 7 and their partners 64 further.
  const int c = lane & 7, sub = lane >> 3;
  // Pages with one new row (decoding): the four groups of lanes take a head each.
  const int quads = (n_heads + 3) / 4;
  for (int task = warp; task < n_lead * quads; task += THREADS / 32) {
    const int w = task / quads;
    const uint32_t live = live_of(w);
    if (!s_lead[w] || __popc(live) != 1) continue;
    const int off = __ffs(live) - 1, row = s_row[w][off];
    const int hh = y * p.group_heads + task % quads * 4 + sub;
    const bool on = hh < h_end;
    const bool is_v = hh >= p.hkv;
    const int head = is_v ? hh - p.hkv : hh;
    uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
    float4 cs[4];
    uint8_t *sf = nullptr, *codes = nullptr;
    int e_old = 1;
    if (on) {
      const __nv_bfloat16* src =
          p.qkv + static_cast<size_t>(row) * p.ldqkv + static_cast<size_t>(p.hq + hh) * D + c * 8;
      a = __ldg(reinterpret_cast<const uint4*>(src));
      b = __ldg(reinterpret_cast<const uint4*>(src + D / 2));
      const long long page = s_page[w];
      sf = (is_v ? p.vsf : p.ksf) + page * p.hkv + head;
      codes = (is_v ? p.vq : p.kq) + page * PAGE * p.hkv * D + head * D;
      e_old = exponent_of(*sf);
    }
    const float4* from = reinterpret_cast<const float4*>(p.cos_sin + static_cast<size_t>(p.pos[row]) * D + c * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = __ldg(from + i);
    float x[16];
    if (is_v)
      unpack16(a, b, x);
    else
      rotate16(a, b, cs, x);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fabsf(x[i]) <= FLT_MAX ? fmaxf(amax, fabsf(x[i])) : amax;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!on) continue;
    const int e = off == 0 ? scale_exp(amax) : max(scale_exp(amax), e_old);
    if (off != 0 && e > e_old) {
      const float f = two_to(max(e_old - e, -60));
#pragma unroll 4
      for (int o = 0; o < PAGE; ++o)
        if (o != off) shrink(reinterpret_cast<uint4*>(codes + static_cast<size_t>(o) * p.hkv * D) + c, f);
    }
    const uint4 v = codes_of(x, two_to(127 - e), true);
    uint8_t* at = codes + static_cast<size_t>(off) * p.hkv * D + c * 8;
    *reinterpret_cast<uint2*>(at) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2*>(at + D / 2) = make_uint2(v.z, v.w);
    if (c == 0) *sf = static_cast<uint8_t>(e);
  }
  // The others: a warp has a head, four slots at a time (step s: slots 4 s ..
  // 4 s + 3). All rows are loaded before any is used.
  for (int task = warp; task < n_lead * n_heads; task += THREADS / 32) {
    const int w = task / n_heads;
    const uint32_t live = live_of(w);
    if (!s_lead[w] || __popc(live) < 2) continue;  // (none: every row of the page has a bad position)
    const int hh = y * p.group_heads + task % n_heads;
    const bool is_v = hh >= p.hkv;
    const int head = is_v ? hh - p.hkv : hh;
    const long long page = s_page[w];
    uint8_t* sf = (is_v ? p.vsf : p.ksf) + page * p.hkv + head;
    uint8_t* codes = (is_v ? p.vq : p.kq) + page * PAGE * p.hkv * D + head * D;
    const int e_old = exponent_of(*sf);
    int pos[4], at[2];
    if (staged) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = s_row[0][(tid + i * THREADS) / (D / 4)];
        at[i] = row >= 0 ? __ldg(p.pos + row) : 0;  // (a row that is not there has no bad position either)
      }
    }
    uint4 a[4], b[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int row = s_row[w][4 * s + sub];
      a[s] = b[s] = make_uint4(0u, 0u, 0u, 0u);
      pos[s] = -1;
      if (row >= 0) {
        const __nv_bfloat16* src =
            p.qkv + static_cast<size_t>(row) * p.ldqkv + static_cast<size_t>(p.hq + hh) * D + c * 8;
        a[s] = __ldg(reinterpret_cast<const uint4*>(src));
        b[s] = __ldg(reinterpret_cast<const uint4*>(src + D / 2));
        pos[s] = __ldg(p.pos + row);
      }
    }
    if (staged) {  // every warp comes here, once
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = tid + i * THREADS, j = k % (D / 4);
        s_cs[k / (D / 4)][(j & 3) * 8 + j / 4] =
            __ldg(reinterpret_cast<const float4*>(p.cos_sin + static_cast<size_t>(at[i]) * D) + j);
      }
      __syncthreads();
    }
    auto values = [&](int s, float (&x)[16]) {
      if (is_v || pos[s] < 0) {
        unpack16(a[s], b[s], x);
        return;
      }
      float4 cs[4];
      if (staged) {
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = s_cs[4 * s + sub][8 * i + c];
      } else {
        const float4* from = reinterpret_cast<const float4*>(p.cos_sin + static_cast<size_t>(pos[s]) * D + c * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = __ldg(from + i);
      }
      rotate16(a[s], b[s], cs, x);
    };
    float amax = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if ((live >> (4 * s) & 15u) == 0) continue;
      float x[16];
      values(s, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));  // (the larger of a NaN and a number is the number)
    }
    // non-negative floats are ordered like their bits
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    const bool inf = amax > FLT_MAX;
    if (inf) {  // again, of the finite values
      amax = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float x[16];
        values(s, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fabsf(x[i]) <= FLT_MAX ? fmaxf(amax, fabsf(x[i])) : amax;
      }
      amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    }
    const bool anew = live & 1;
    const int e = anew ? scale_exp(amax) : max(scale_exp(amax), e_old);
    const float inv = two_to(127 - e);
    if (!anew && e > e_old) {
      const float f = two_to(max(e_old - e, -60));
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (live >> (4 * s + sub) & 1) continue;
        shrink(reinterpret_cast<uint4*>(codes + static_cast<size_t>(4 * s + sub) * p.hkv * D) + c, f);
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if ((live >> (4 * s) & 15u) == 0) continue;
      float x[16];
      values(s, x);  // made again rather than held
      const uint4 v = codes_of(x, inv, inf);
      if (pos[s] >= 0) {
        uint8_t* at = codes + static_cast<size_t>(4 * s + sub) * p.hkv * D + c * 8;
        *reinterpret_cast<uint2*>(at) = make_uint2(v.x, v.y);
        *reinterpret_cast<uint2*>(at + D / 2) = make_uint2(v.z, v.w);
      }
    }
    if (lane == 0) *sf = static_cast<uint8_t>(e);
  }
}

constexpr int Q_HEADS = 4;  // heads per thread: they share the loaded cos / sin

__device__ __forceinline__ void rotate8(const uint4& a, const uint4& b, const float4 (&cs)[4], uint4* na, uint4* nb) {
  float x[16];
  rotate16(a, b, cs, x);
  *na = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  *nb = make_uint4(pack_bf16(x[8], x[9]), pack_bf16(x[10], x[11]), pack_bf16(x[12], x[13]), pack_bf16(x[14], x[15]));
}

__device__ void rotate_q(const Append& p, int cta) {
  const int ng = (p.hq + Q_HEADS - 1) / Q_HEADS;
  const long long idx = static_cast<long long>(cta) * THREADS + threadIdx.x;
  const int c = static_cast<int>(idx & 7);  // dims 8c .. 8c + 7 and their partners
  const long long rest = idx >> 3;
  const long long t = rest / ng;
  if (t >= p.T) return;
  const int h0 = static_cast<int>(rest % ng) * Q_HEADS;
  const __nv_bfloat16* in = p.qkv + t * p.ldqkv + c * 8;
  __nv_bfloat16* out = p.q_out + t * p.ldq + c * 8;
  uint4 a[Q_HEADS], b[Q_HEADS];
#pragma unroll
  for (int i = 0; i < Q_HEADS; ++i)
    if (h0 + i < p.hq) {  // in flight while the position is
      a[i] = *reinterpret_cast<const uint4*>(in + (h0 + i) * D);
      b[i] = *reinterpret_cast<const uint4*>(in + (h0 + i) * D + D / 2);
    }
  const int pos = p.pos[t];
  if (pos < 0 || pos >= p.max_pos) {
    if (c == 0 && h0 == 0) record_status_detail(p.status, kStatusBadIndex, 1, static_cast<int>(t), pos);
    return;
  }
  const float4* src = reinterpret_cast<const float4*>(p.cos_sin + static_cast<size_t>(pos) * D + c * 16);
  const float4 cs[4] = {__ldg(src), __ldg(src + 1), __ldg(src + 2), __ldg(src + 3)};
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
  // the K/V CTAs, which take longest, first
  const int cta = blockIdx.x;
  if (cta < p.kv_ctas)
    append_kv(p, cta);
  else
    rotate_q(p, cta - p.kv_ctas);
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
  // Few rows: 4 of them and two heads per CTA, so that they spread over the SMs
  // (64 decoding rows 4.6 us, 5.2 with eight heads); eight heads where the CTAs
  // would not all run at once, 3 per SM (a prompt of 300 rows 5.9 us, 6.4 with
  // four heads, 7.4 with two). Many rows (prompts, one leading row in 16):
  // windows of 8, fewer CTAs that lead nothing (for 512 rows and fewer a window
  // of 4 is faster: 6.4 us against 8.3).
  const bool many = T > 512;
  p.win = many ? 8 : 4;
  p.group_heads = many || static_cast<long long>((T + 3) / 4) * hkv > 3 * 148 ? 8 : 2;
  p.head_groups = (2 * hkv + p.group_heads - 1) / p.group_heads;
  const long long kv_ctas = static_cast<long long>((T + p.win - 1) / p.win) * p.head_groups;
  const long long q_items = static_cast<long long>(T) * ((hq + Q_HEADS - 1) / Q_HEADS) * 8;
  const long long ctas = kv_ctas + (q_items + THREADS - 1) / THREADS;
  if (ctas > 0x7fffffffLL) return -1;
  p.kv_ctas = static_cast<int>(kv_ctas);
  launch_pdl(append_kernel, dim3(static_cast<unsigned>(ctas)), THREADS, 0, stream, p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : static_cast<int>(e);
}
