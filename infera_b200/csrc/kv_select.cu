// Which keys of a cache stay, and moving them together.
//
// select_kernel: for each (sequence, KV head), of L keys with accumulated
// weights x: the first `sink`, the last `recent`, and of the others those with
// the largest x (equal ones: the lowest place first), `keep` in all, as places
// in ascending order. The weights are read once, into shared memory; the
// threshold is found digit by digit (11, 11 and 10 bits of the weight as an
// unsigned number of the same order) in histograms; a last pass lists each warp's
// places at or above it over the weights, and what is listed and stays is written
// behind all that lies before it. A cluster of CTAs shares a
// list: each takes a run of places and adds up the others' histograms through
// distributed shared memory.
// Bound by its chain of steps (load, three digits, list, write, a barrier or two
// after each) and, for long runs, by some 90 instructions for 32 weights: 8 lists
// of 1025 weights 8 us, 96 ragged ones up to 9000 12.5, 32 of 100001 by clusters
// of four 24 (12.8 MB of weights; 120 instructions and 27 us when one pass counted
// and another wrote). Four copies of the first histogram against equal exponents
// were slower (42 us: the others' are read through the cluster).
//
// The moves: rows src[i] -> i of a sequence's places, in place. src[i] >= i, so
// a row is never written before a row that is read later lies there: places are
// taken in ascending order, and a group's rows are all read before the first of
// them is written. A CTA owns its columns, so no other one touches them.
//   stream_kernel  long lists: groups of rows pass through a ring in shared
//                  memory (asynchronous loads run groups ahead of the stores,
//                  which is no harm: what is written lies before all that is
//                  read later), the places' slots looked up one group further
//   batch_kernel   short lists over many layers (the accepted path of a tree):
//                  the moves are listed once, and rows of several layers are
//                  held in registers at a time
// Long lists are bound by HBM: 8192 rows of 32 lists, K and V, 268 MB read and
// written, 47 us (5.7 TB/s, 0.89 of the copy rate), 2048 rows of 56 lists 22 us (4.5
// TB/s). Moved in batches of rows held in registers they took 79 and 37 us. The
// accepted rows of 48 trees in 80 layers (35 MB in pieces of 2 KB) take 14 us: 1152
// CTAs are 2.6 waves of those that the SMs hold, and each wave goes through the
// chain count, entry, page, row, with the rows of 160 layers far apart.
#include <cooperative_groups.h>

#include <algorithm>

#include "kv8.cuh"

namespace ib200 {
namespace sel {

namespace cg = cooperative_groups;
using kv8::table_row;

constexpr int BINS = 2048;
constexpr int CANDIDATES = 2048;
constexpr uint32_t STAYS = 0xffffffffu;  // (the largest weight, infinity, has 0xff800000)
constexpr int FEW = 4096;              // places of a CTA of 512 threads, at most
constexpr int MAX_CACHED = 44 * 1024;  // places that a CTA holds in shared memory, 176 KB

// places of a run when `of` ones are shared by `among`, in whole groups of a warp
__host__ __device__ constexpr int run_of(long long of, int among) {
  return static_cast<int>(((of + among - 1) / among + 127) / 128 * 128);
}

struct SelectParams {
  float* mass;            // [mass_rows, hkv, cap]
  int mass_rows, hkv;
  long long cap;
  const int* seq_lens;
  const int* bt_rows;
  int keep, sink, recent;
  int update;             // write the kept weights back, zero behind them
  int* kept;              // [n, hkv, keep]
  float* kept_mass;       // [n, hkv, keep]
  int* count;             // [n]
  int* status;
};

// An unsigned number in the order of the weights: a NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  if ((u << 1) == 0u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// CACHED: a CTA's run of places fits into its shared memory; else they are read
// in each pass.
template <bool CACHED, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) select_kernel(const SelectParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr int WARPS = THREADS / 32, MINE = BINS / THREADS;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int list = blockIdx.x / C, s = list / p.hkv, h = list % p.hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ __align__(16) uint32_t cached[];  // the run's weights as order_of gives them
  // a histogram a digit, so that none is cleared while another CTA reads it
  __shared__ __align__(16) uint32_t hist0[BINS], hist1[BINS], hist2[BINS / 2];
  __shared__ uint32_t candidates[CANDIDATES];  // those whose first digit is the threshold's
  __shared__ uint32_t n_candidates, wsum[WARPS], wgt[WARPS], weq[WARPS], s_bin, s_want, totals[2];
  auto sync_all = [&]() {  // of the CTAs that share the list
    if (C > 1)
      cluster.sync();
    else
      __syncthreads();
  };

  const int row = p.bt_rows != nullptr ? p.bt_rows[s] : s;
  long long n_keys = max(p.seq_lens[s], 0);
  for (int i = tid; i < BINS / 4; i += THREADS) {
    reinterpret_cast<uint4*>(hist0)[i] = make_uint4(0u, 0u, 0u, 0u);
    reinterpret_cast<uint4*>(hist1)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (i < BINS / 8) reinterpret_cast<uint4*>(hist2)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (tid == 0) n_candidates = 0;
  bool bad = row < 0 || row >= p.mass_rows;
  if (bad && tid == 0 && rank == 0) record_status_detail(p.status, kStatusBadIndex, 6, s, row);
  if (!bad && n_keys > p.cap) {
    if (tid == 0 && rank == 0) record_status_detail(p.status, kStatusBadIndex, 6, s, static_cast<int>(n_keys));
    n_keys = p.cap;
  }
  // a row that an earlier sequence has is that one's to change (those without keys, which pad a batch, may share one)
  if (!bad && p.update && p.bt_rows != nullptr && n_keys > 0) {
    bool twice = false;
    for (int i = tid; i < s; i += THREADS) twice = twice || p.bt_rows[i] == row;
    if (__syncthreads_or(twice)) {
      if (tid == 0 && rank == 0) record_status_detail(p.status, kStatusBadIndex, 7, s, row);
      bad = true;
    }
  }
  const int L = bad ? 0 : static_cast<int>(n_keys);
  float* x = p.mass + (static_cast<size_t>(bad ? 0 : row) * p.hkv + h) * static_cast<size_t>(p.cap);
  int* kept = p.kept + static_cast<size_t>(list) * p.keep;
  float* kept_mass = p.kept_mass + static_cast<size_t>(list) * p.keep;
  if (h == 0 && rank == 0 && tid == 0) p.count[s] = min(L, p.keep);
  const int all = C * THREADS, at = rank * THREADS + tid;
  if (L <= p.keep) {  // all stay (the whole cluster is here)
    for (int i = at; i < p.keep; i += all) {
      kept[i] = i < L ? i : -1;
      kept_mass[i] = i < L ? x[i] : 0.f;
    }
    return;
  }
  const int lo = p.sink, hi = L - p.recent;  // what lies before and behind stays
  // this CTA's run of places, in groups of four; and within it one for each warp
  const int run = run_of(L, C), first = min(L, rank * run), last = min(L, first + run);
  const int seg = run_of(run, WARPS), w0 = min(last, first + warp * seg), w1 = min(last, w0 + seg);
  const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  auto read4 = [&](int i) -> float4 {  // weights i .. i + 3, those behind the run as 0
    if (wide && i + 4 <= last) return *reinterpret_cast<const float4*>(x + i);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < last) v.x = x[i];
    if (i + 1 < last) v.y = x[i + 1];
    if (i + 2 < last) v.z = x[i + 2];
    if (i + 3 < last) v.w = x[i + 3];
    return v;
  };
  struct Keys {
    uint32_t k[4];
  };
  auto key = [&](int i, float v) { return i < lo || i >= hi ? STAYS : order_of(v); };
  // What lies before and behind the middle stays: above every weight's number.
  auto keys_of = [&](int i, const float4& v) -> Keys {
    Keys q{{order_of(v.x), order_of(v.y), order_of(v.z), order_of(v.w)}};
    if (i < lo || i + 4 > hi)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (i + c < lo || i + c >= hi) q.k[c] = STAYS;
    return q;
  };
  auto keys = [&](int i) -> Keys {
    if constexpr (CACHED) {
      const uint4 k = *reinterpret_cast<const uint4*>(cached + (i - first));
      return {{k.x, k.y, k.z, k.w}};
    } else {
      return keys_of(i, read4(i));
    }
  };
  uint32_t want = static_cast<uint32_t>(p.keep - p.sink - p.recent);  // of those that match the digits so far
  uint32_t prefix = 0, known = 0;
  __syncthreads();  // (the histograms are clear)
#pragma unroll 1
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : (digit == 1 ? 10 : 0), bits = digit == 2 ? 10 : 11;
    if (digit == 0) {
      constexpr int AHEAD = 4;  // loads, then what they are for
      for (int i0 = first + 4 * tid; i0 < last; i0 += AHEAD * 4 * THREADS) {
        float4 v[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) v[a] = read4(i0 + a * 4 * THREADS);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const int i = i0 + a * 4 * THREADS;
          if (i >= last) break;
          const Keys k = keys_of(i, v[a]);
          if constexpr (CACHED) *reinterpret_cast<uint4*>(cached + (i - first)) = make_uint4(k.k[0], k.k[1], k.k[2], k.k[3]);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (k.k[c] != STAYS) atomicAdd(&hist0[k.k[c] >> 21], 1u);
        }
      }
    } else if (digit == 1) {
      for (int i = first + 4 * tid; i < last; i += 4 * THREADS) {
        const Keys k = keys(i);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if ((k.k[c] ^ prefix) >> 21 == 0 && k.k[c] != STAYS) {
            atomicAdd(&hist1[k.k[c] >> 10 & (BINS - 1)], 1u);
            const uint32_t n = atomicAdd(&n_candidates, 1u);
            if (n < CANDIDATES) candidates[n] = k.k[c];
          }
      }
    } else if (n_candidates <= CANDIDATES) {
      for (int i = tid; i < static_cast<int>(n_candidates); i += THREADS)
        if ((candidates[i] ^ prefix) >> 10 == 0) atomicAdd(&hist2[candidates[i] & (BINS / 2 - 1)], 1u);
    } else {
      for (int i = first + 4 * tid; i < last; i += 4 * THREADS) {
        const Keys k = keys(i);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if ((k.k[c] ^ prefix) >> 10 == 0 && k.k[c] != STAYS) atomicAdd(&hist2[k.k[c] & (BINS / 2 - 1)], 1u);
      }
    }
    sync_all();
    // the bin in which the want-th largest lies: thread t has MINE bins, from MINE t on from the top
    uint32_t c[MINE] = {};
    const int top = (1 << bits) - MINE - MINE * tid;
    uint32_t* hist = digit == 0 ? hist0 : (digit == 1 ? hist1 : hist2);
    for (int r = 0; r < C && top >= 0; ++r) {
      const uint32_t* other = (C > 1 ? cluster.map_shared_rank(hist, r) : hist) + top;
#pragma unroll
      for (int i = 0; i < MINE; i += 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(other + i);
        c[MINE - 1 - i] += v.x;
        c[MINE - 2 - i] += v.y;
      }
    }
    uint32_t own = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) own += c[i];
    uint32_t sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) wsum[warp] = sum;
    __syncthreads();
    uint32_t before = sum - own + __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane] : 0u);
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      if (before < want && before + c[i] >= want) {
        s_bin = static_cast<uint32_t>(top + MINE - 1 - i);
        s_want = want - before;
      }
      before += c[i];
    }
    __syncthreads();  // s_bin
    if (want == 0) break;  // (of the middle nothing stays)
    want = s_want;
    prefix |= s_bin << shift;
    known |= ((1u << bits) - 1) << shift;
  }
  if (known == 0) prefix = STAYS - 1;  // above the number of every weight
  // A warp's places above the threshold, and at it, of which the list's first `want` stay: counted, and listed over
  // the weights that have been looked at.
  uint32_t gt = 0, eq = 0;
  uint32_t* listed = CACHED ? cached + (w0 - first) : nullptr;
  const uint32_t below = (1u << lane) - 1;
  uint32_t on = 0;
  constexpr int GROUPS = 4;  // of 32 places whose loads are under way together
  for (int i0 = w0; i0 < w1; i0 += 32 * GROUPS) {
    uint32_t k[GROUPS];
#pragma unroll
    for (int a = 0; a < GROUPS; ++a) {
      const int i = i0 + 32 * a + lane;
      k[a] = 0;
      if (i < w1) {
        if constexpr (CACHED)
          k[a] = cached[i - first];
        else
          k[a] = key(i, x[i]);
      }
    }
#pragma unroll
    for (int a = 0; a < GROUPS; ++a) {
      const int i = i0 + 32 * a + lane;
      const bool is = k[a] >= prefix && i < w1;
      const uint32_t all_on = __ballot_sync(0xffffffffu, is);
      if constexpr (CACHED)
        if (is) listed[on + __popc(all_on & below)] = static_cast<uint32_t>(i);
      on += __popc(all_on);
      eq += is && k[a] == prefix;
    }
  }
  eq = __reduce_add_sync(0xffffffffu, eq);
  gt = on - eq;
  const int n_listed = CACHED ? static_cast<int>(on) : w1 - w0;
  if (lane == 0) {
    wgt[warp] = gt;
    weq[warp] = eq;
  }
  __syncthreads();
  gt = __reduce_add_sync(0xffffffffu, lane < warp ? wgt[lane] : 0u);
  eq = __reduce_add_sync(0xffffffffu, lane < warp ? weq[lane] : 0u);
  if (C > 1) {
    if (warp == WARPS - 1 && lane == 0) {
      totals[0] = gt + wgt[WARPS - 1];
      totals[1] = eq + weq[WARPS - 1];
    }
    cluster.sync();
    uint32_t a = 0, b = 0;
    if (lane < rank) {
      const uint32_t* other = cluster.map_shared_rank(totals, lane);
      a = other[0];
      b = other[1];
    }
    gt += __reduce_add_sync(0xffffffffu, a);
    eq += __reduce_add_sync(0xffffffffu, b);
  }
  // a place goes behind all that stay before it
  for (int j0 = 0; j0 < n_listed; j0 += 32 * GROUPS) {
    int place[GROUPS];
    float v[GROUPS];
#pragma unroll
    for (int a = 0; a < GROUPS; ++a) {
      const int j = j0 + 32 * a + lane;
      place[a] = j >= n_listed ? -1 : (CACHED ? static_cast<int>(listed[j]) : w0 + j);
      v[a] = place[a] >= 0 ? x[place[a]] : 0.f;
    }
#pragma unroll
    for (int a = 0; a < GROUPS; ++a) {
      if (j0 + 32 * a >= n_listed) break;
      const uint32_t k = key(place[a], v[a]);
      const uint32_t above = __ballot_sync(0xffffffffu, place[a] >= 0 && k > prefix);
      const uint32_t same = __ballot_sync(0xffffffffu, place[a] >= 0 && k == prefix);
      const uint32_t e = eq + __popc(same & below), to = gt + __popc(above & below) + min(e, want);
      if ((above >> lane & 1) != 0 || ((same >> lane & 1) != 0 && e < want)) {
        kept[to] = place[a];
        kept_mass[to] = v[a];
      }
      gt += __popc(above);
      eq += __popc(same);
    }
  }
  if (C > 1 || p.update) sync_all();  // (no CTA leaves while another reads its totals)
  if (p.update) {
    for (int i = at; i < L; i += all) x[i] = i < p.keep ? __ldcg(kept_mass + i) : 0.f;
  }
}

struct MoveParams {
  uint8_t* k;
  uint8_t* v;
  int layers, group;         // layers of a CTA
  long long layer_bytes;
  int pitch;                 // bytes of a slot
  int width, lanes;          // bytes of a list's columns, 16-byte pieces of a CTA's
  int parts;
  int num_pages;
  const int* block_table;
  const int* bt_rows;
  int table_rows, max_pages, ld_table;
  const int* src;            // [n, heads, m], or [n, m] where `shared`
  int heads, m;
  bool shared;               // all heads' columns move by the sequence's list
  const int* count;          // [n]
  const int* start;          // [n] or null
  int* status;
};

// What the CTAs of a sequence know; count 0: nothing moves.
struct MoveSeq {
  const int* bt;
  int count;
  long long start;
};
__device__ __forceinline__ MoveSeq move_seq(const MoveParams& p, int s) {
  const int row = p.bt_rows != nullptr ? p.bt_rows[s] : s;
  MoveSeq q{table_row(p.block_table, row, p.table_rows, p.ld_table, s, p.status), min(max(p.count[s], 0), p.m),
            p.start != nullptr ? p.start[s] : 0};
  if (q.bt == nullptr) q.count = 0;
  if (q.start < 0) {
    if (threadIdx.x == 0) record_status_detail(p.status, kStatusBadIndex, 1, s, static_cast<int>(q.start));
    q.count = 0;
  }
  // a sequence whose places an earlier one has too stays as that one leaves it (those without moves may share a row)
  if (p.bt_rows != nullptr && q.count > 0) {
    bool twice = false;
    for (int i = threadIdx.x; i < s; i += blockDim.x) twice = twice || p.bt_rows[i] == row;
    if (__syncthreads_or(twice)) {
      if (threadIdx.x == 0) record_status_detail(p.status, kStatusBadIndex, 7, s, row);
      q.count = 0;
    }
  }
  return q;
}
// Whether entry e of value v moves: what does not and should goes to the status word.
__device__ __forceinline__ bool moves_at(const MoveParams& p, const MoveSeq& q, int s, int e, int v) {
  if (v == e || v == -1) return false;
  if (v > e && q.start + v < static_cast<long long>(p.max_pages) * kv8::PAGE) return true;
  record_status_detail(p.status, kStatusBadIndex, 8, s, v);
  return false;
}
// The slots of a move between pages ga and gb; false (and a status) where there is no such page.
__device__ __forceinline__ bool known(const MoveParams& p, int s, int ga, int gb) {
  const bool a = static_cast<unsigned>(ga) < static_cast<unsigned>(p.num_pages);
  const bool b = static_cast<unsigned>(gb) < static_cast<unsigned>(p.num_pages);
  if (!a || !b) record_status_detail(p.status, kStatusBadIndex, 2, s, a ? gb : ga);
  return a && b;
}

constexpr int STREAM_WARPS = 8;
constexpr int STAGE = 4096;  // bytes of a warp and stage
constexpr int STAGES = 3;

template <int RB>  // bytes of a row that a CTA moves
__global__ void __launch_bounds__(STREAM_WARPS * 32, 2) stream_kernel(const MoveParams p) {
  constexpr int RW = STAGE / RB;                  // rows of a warp and stage
  constexpr int RL = (RW + 31) / 32;              // rows that a lane looks up
  constexpr int LANES = RB / 16;                  // lanes of a row
  constexpr int PIECES = STAGE / 16 / 32;
  extern __shared__ __align__(16) uint8_t ring[];  // [STAGES][STREAM_WARPS][STAGE]
  __shared__ int2 slots[STAGES][STREAM_WARPS][RW];
  pdl_trigger();
  pdl_wait();
  const int s = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const MoveSeq q = move_seq(p, s);
  if (q.count == 0) return;
  const int* src = p.src + static_cast<size_t>(p.shared ? s : blockIdx.x) * p.m;
  uint8_t* cache = (static_cast<int>(blockIdx.y) < p.parts ? p.k : p.v) + blockIdx.z * p.layer_bytes +
                   static_cast<size_t>(h) * p.width + static_cast<size_t>(blockIdx.y % p.parts) * RB;
  const int n = (q.count + STREAM_WARPS * RW - 1) / (STREAM_WARPS * RW);
  auto entry = [&](int k, int i) { return (k * STREAM_WARPS + warp) * RW + lane + 32 * i; };
  int v[RL], at[RL], ga[RL], gb[RL];  // entries of the stage after next to load; of the next one: entries (or -1), pages
  auto load_src = [&](int k) {
#pragma unroll
    for (int i = 0; i < RL; ++i) {
      const int e = entry(k, i);
      v[i] = e < q.count && lane + 32 * i < RW ? src[e] : -1;
    }
  };
  auto load_pages = [&](int k) {
#pragma unroll
    for (int i = 0; i < RL; ++i) {
      const int e = entry(k, i);
      at[i] = moves_at(p, q, s, e, v[i]) ? v[i] : -1;
      ga[i] = gb[i] = 0;
      if (at[i] >= 0) {
        ga[i] = q.bt[(q.start + at[i]) / kv8::PAGE];
        gb[i] = q.bt[(q.start + e) / kv8::PAGE];
      }
    }
  };
  auto load_rows = [&](int k) {
    if (k < n) {
      int2* list = slots[k % STAGES][warp];
#pragma unroll
      for (int i = 0; i < RL; ++i) {
        if (lane + 32 * i >= RW) break;
        const bool on = at[i] >= 0 && known(p, s, ga[i], gb[i]);
        list[lane + 32 * i] = on ? make_int2(ga[i] * kv8::PAGE + static_cast<int>((q.start + at[i]) % kv8::PAGE),
                                             gb[i] * kv8::PAGE + static_cast<int>((q.start + entry(k, i)) % kv8::PAGE))
                                 : make_int2(-1, -1);
      }
      __syncwarp();
      const uint32_t dst = smem_u32(ring) + ((k % STAGES) * STREAM_WARPS + warp) * STAGE + lane * 16;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int from = list[i * (32 / LANES) + lane / LANES].x;
        if (from >= 0)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * 512),
                       "l"(cache + static_cast<size_t>(from) * p.pitch + (lane % LANES) * 16)
                       : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  load_src(0);
  load_pages(0);
  load_src(1);
  for (int k = 0; k < STAGES - 1; ++k) {
    load_rows(k);
    load_pages(k + 1);
    load_src(k + 2);
  }
  for (int k = 0; k < n; ++k) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();  // the stage's rows are read, of all warps
    const int2* list = slots[k % STAGES][warp];
    const uint8_t* from = ring + ((k % STAGES) * STREAM_WARPS + warp) * STAGE + lane * 16;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int to = list[i * (32 / LANES) + lane / LANES].y;
      if (to >= 0)
        *reinterpret_cast<uint4*>(cache + static_cast<size_t>(to) * p.pitch + (lane % LANES) * 16) =
            *reinterpret_cast<const uint4*>(from + i * 512);
    }
    __syncwarp();  // the list of stage k + STAGES - 1 is not that of stage k, but k + STAGES' is
    load_rows(k + STAGES - 1);
    load_pages(k + STAGES);
    load_src(k + STAGES + 1);
  }
}

constexpr int MOVE_THREADS = 256;
constexpr int ENTRIES = 2 * MOVE_THREADS;  // places resolved at a time
constexpr int UNITS = 8;                   // 16-byte pieces that a thread holds

__global__ void __launch_bounds__(MOVE_THREADS) batch_kernel(const MoveParams p) {
  pdl_trigger();
  pdl_wait();
  const int s = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int from[ENTRIES], to[ENTRIES];
  __shared__ int wsum[MOVE_THREADS / 32];
  const MoveSeq q = move_seq(p, s);
  if (q.count == 0) return;
  const int* src = p.src + (static_cast<size_t>(s) * p.heads + h) * p.m;
  const int l0 = blockIdx.z * p.group, layers = min(p.group, p.layers - l0);
  // this thread's 16 bytes of a row, and its first row in a round of `rows`
  const int part = blockIdx.y % p.parts, lanes = min(p.lanes, p.width / 16 - part * p.lanes);
  const int rows = MOVE_THREADS / lanes, mine_row = tid / lanes;
  uint8_t* cache = (static_cast<int>(blockIdx.y) < p.parts ? p.k : p.v) + l0 * p.layer_bytes + static_cast<size_t>(h) * p.width +
                   static_cast<size_t>(part * p.lanes + tid % lanes) * 16;
  for (int e0 = 0; e0 < q.count; e0 += ENTRIES) {
    // slots of the next places that move, in order
    int a[2], b[2];
    bool moves[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = e0 + 2 * tid + i;
      const int v = e < q.count ? src[e] : -1;
      moves[i] = moves_at(p, q, s, e, v);
      a[i] = b[i] = 0;
      if (moves[i]) {
        const int ga = q.bt[(q.start + v) / kv8::PAGE], gb = q.bt[(q.start + e) / kv8::PAGE];
        moves[i] = known(p, s, ga, gb);
        a[i] = ga * kv8::PAGE + static_cast<int>((q.start + v) % kv8::PAGE);
        b[i] = gb * kv8::PAGE + static_cast<int>((q.start + e) % kv8::PAGE);
      }
    }
    const int mine = moves[0] + moves[1];
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) wsum[warp] = sum;
    __syncthreads();
    int total = 0, at = sum - mine;
#pragma unroll
    for (int w = 0; w < MOVE_THREADS / 32; ++w) {
      at += w < warp ? wsum[w] : 0;
      total += wsum[w];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (moves[i]) {
        from[at] = a[i];
        to[at++] = b[i];
      }
    __syncthreads();
    // rounds of rows, layer by layer: UNITS rounds are read before the first is written
    int l = 0, e = mine_row;  // this thread's row of the next round: its layer and move
    const int more = total > 0 && mine_row < rows ? layers : 0;
    for (int done = 0; done < layers * total; done += rows * UNITS) {
      uint4 v[UNITS];
      int ll = l, ee = e;
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        while (ee >= total && ll < more) ee -= total, ++ll;
        if (ll < more) v[i] = __ldcg(reinterpret_cast<const uint4*>(cache + ll * p.layer_bytes + static_cast<size_t>(from[ee]) * p.pitch));
        ee += rows;
      }
      __syncthreads();  // all are read
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        while (e >= total && l < more) e -= total, ++l;
        if (l < more) *reinterpret_cast<uint4*>(cache + l * p.layer_bytes + static_cast<size_t>(to[e]) * p.pitch) = v[i];
        e += rows;
      }
    }
    __syncthreads();  // the list is used
  }
}

}  // namespace sel
}  // namespace ib200

using namespace ib200;

// mass fp32 [mass_rows, hkv, cap], row bt_rows[s] (null: s); kept / kept_mass
// [n, hkv, keep], count [n]. sink + recent <= keep. cluster: CTAs of a list, 1 to 8.
extern "C" int ib_kv_select(float* mass, int mass_rows, int hkv, long long cap, const int* seq_lens,
                            const int* bt_rows, int n, int keep, int sink, int recent, int update, int cluster,
                            int* kept, float* kept_mass, int* count, int* status, cudaStream_t stream) {
  using namespace ib200::sel;
  if (n <= 0) return 0;
  if (hkv <= 0 || keep < 1 || sink < 0 || recent < 0 || sink > keep - recent || cap < 0 || cap > INT32_MAX / 2 ||
      (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8) ||
      static_cast<long long>(n) * hkv * cluster > INT32_MAX)
    return -1;
  SelectParams p{mass, mass_rows, hkv, cap, seq_lens, bt_rows, keep, sink, recent, update, kept, kept_mass, count, status};
  const int run = run_of(cap, cluster);  // the longest of a CTA
  const bool cached = run <= MAX_CACHED;
  // few weights a thread: the barriers of half as many warps are quicker (1025 keys 8.2 us against 9.2)
  const int threads = run <= FEW ? 512 : 1024;
  const auto kernel = threads == 512 ? select_kernel<true, 512> : (cached ? select_kernel<true, 1024> : select_kernel<false, 1024>);
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(select_kernel<true, 1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_CACHED * 4);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(n) * hkv * cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = cached ? static_cast<size_t>(run) * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
}

// Caches [layers, num_slots, row_bytes] (v null: one channel). src [n, heads, m]:
// list (s, h) moves the columns h * row_bytes / heads .. of places start[s] +
// src[s, h, i] to start[s] + i, i < count[s].
extern "C" int ib_kv_compact(void* k, void* v, int layers, long long num_slots, int row_bytes, const int* block_table,
                             const int* bt_rows, int table_rows, int max_pages, int ld_table, const int* src, int n,
                             int heads, int m, const int* count, const int* start, int num_sms, int* status,
                             cudaStream_t stream) {
  using namespace ib200::sel;
  if (n <= 0 || m <= 0 || layers <= 0) return 0;
  if (heads <= 0 || row_bytes <= 0 || row_bytes % heads != 0 || (row_bytes / heads) % 16 != 0 || num_slots < kv8::PAGE ||
      num_slots % kv8::PAGE != 0 || num_slots > INT32_MAX || max_pages < 0 || k == nullptr || num_sms <= 0 ||
      static_cast<long long>(n) * heads > INT32_MAX ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0)
    return -1;
  MoveParams p;
  p.k = static_cast<uint8_t*>(k);
  p.v = static_cast<uint8_t*>(v);
  p.layers = layers;
  p.layer_bytes = num_slots * row_bytes;
  p.pitch = row_bytes;
  p.width = row_bytes / heads;
  p.num_pages = static_cast<int>(num_slots / kv8::PAGE);
  p.block_table = block_table;
  p.bt_rows = bt_rows;
  p.table_rows = table_rows;
  p.max_pages = max_pages;
  p.ld_table = ld_table;
  p.src = src;
  p.m = m;
  p.count = count;
  p.start = start;
  p.status = status;
  const int channels = v != nullptr ? 2 : 1;
  // long lists, and those of single heads, in columns of up to 256 bytes; whole rows of other widths in batches
  if (layers <= 65535 && (heads > 1 ? p.width == 256 : m > 64 && row_bytes % 256 == 0)) {
    p.shared = heads == 1;
    p.width = 256;
    p.heads = row_bytes / 256;
    if (static_cast<long long>(n) * p.heads > INT32_MAX) return -1;
    const long long lists = static_cast<long long>(n) * p.heads * channels * layers;
    // a CTA moves some 50 GB/s: where the lists are few, two or four share their columns
    p.parts = lists >= 2 * num_sms ? 1 : (2 * lists >= 2 * num_sms ? 2 : 4);
    const auto kernel = p.parts == 1 ? stream_kernel<256> : (p.parts == 2 ? stream_kernel<128> : stream_kernel<64>);
    constexpr int smem = STAGES * STREAM_WARPS * STAGE;
    static bool attr_set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
      for (auto k : {stream_kernel<256>, stream_kernel<128>, stream_kernel<64>}) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return static_cast<int>(e);
      }
      if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    return static_cast<int>(launch_pdl(kernel, dim3(static_cast<unsigned>(n) * p.heads, channels * p.parts, layers),
                                       STREAM_WARPS * 32, smem, stream, p));
  }
  p.shared = false;
  p.heads = heads;
  const long long lists = static_cast<long long>(n) * heads * channels;
  // rows of more than 4 KB in parts; layers in as many groups as give each SM eight CTAs, three of which it holds at a
  // time (75 registers)
  const int pieces = p.width / 16;
  p.parts = (pieces + MOVE_THREADS - 1) / MOVE_THREADS;
  p.lanes = (pieces + p.parts - 1) / p.parts;
  const long long groups = std::min<long long>(layers, std::max<long long>(1, 8LL * num_sms / (lists * p.parts)));
  p.group = static_cast<int>((layers + groups - 1) / groups);
  if (static_cast<long long>(p.group) * ENTRIES > INT32_MAX) return -1;
  const dim3 grid(static_cast<unsigned>(n) * heads, channels * p.parts, (layers + p.group - 1) / p.group);
  if (grid.z > 65535) return -1;
  return static_cast<int>(launch_pdl(batch_kernel, grid, MOVE_THREADS, 0, stream, p));
}
