// Attention of drafted tokens that form a tree (speculative decoding) over the
// bf16 paged KV cache, on tcgen05. A sequence's last q_len keys are its nodes;
// node i sees the keys before them and node j where bit j of its mask is set.
//
//   S = Q K^T, O += W V,  w = 2^(c s - m - 32) in bf16 (rounded, by up to 2^-8 of
//   itself, as in the prompt kernel), the sum of the softmax over the fp32 weights
//
// One bf16 digit of W is a choice: outputs are off by 0.0020 to 0.0023 in the
// 2-norm, where rounding the output alone gives 0.0017. A second digit in the
// other half of S's columns, as the decode kernel with weights has, gives 0.0017
// and takes 12.6 -> 14.2 us (8 nodes over 508 keys), 90 -> 95 (40 ragged trees),
// 287 -> 357 (16 x 64 nodes) and 121 -> 148 (61 over 100001): too much for an error
// that the prompt kernel's rows, which the cache comes from, have too. The sum over
// the rounded weights gives 0.0033 instead of 0.0048 as the largest error of the 16
// sequences, and takes 287 -> 315 us.
//
// The query heads of a KV head are packed: rows are (node, head) pairs. A CTA
// takes 128 rows and walks its keys in tiles of 64 (4 pages), 16 KB of K and 16
// KB of V in a ring of five slots that both take in turn:
//   warp 0      TMA producer
//   warp 1      MMA issuer: S(j), then W V of tile j - 1
//   warps 2..5  softmax, a thread per row; they also stage Q
// S is double-buffered in TMEM, so the scores of a tile are made while the
// softmax of the one before runs; a tile's weights lie over its scores. Two
// CTAs to an SM (half of TMEM and of shared memory each) hide each other's
// starts, ends and waits. More than 128 rows of a tree are items of their own
// that read the same keys, from L2 but for the first.
//
// Masks are looked at only in the tiles that hold nodes (the last ones). There
// the values' infinities and NaN are multiplied as zeros (a weight of zero does
// not cancel them) and written at the end to the rows that see them, and V rows
// behind the sequence, which a recycled page may have left as NaN, are zeroed.
//
// The tiles of all items, laid end to end, are cut into equal runs, one for each
// CTA of a single wave: batches of any raggedness are balanced, and the loads of
// a run's next item are under way while the one before ends. An item that a cut
// falls in is merged from its pieces by a second kernel; a run has at most two
// such pieces, the end of an item and the beginning of one, so the workspace does
// not depend on the batch.
//
// Up to 128 rows are bound by HBM: captured calls of 40 ragged trees of up to 26 nodes
// (32 heads over 8) over up to 5000 keys on scattered pages take 91 us, where the
// bytes need 67: the CTAs read at 7.5 TB/s once they run, 7 us after the launch; the
// last one ends 12 us after the mean, and then two or three pieces of each item are
// merged. With more rows two CTAs take 1640 cycles for a tile each. Their products or
// their exponentials alone need 1024, but shared memory 1536: a tile's scores read 48
// KB of it (8 steps of 4 KB of Q and 2 KB of K), W V 16 KB, and TMA writes 32 KB, at
// 128 bytes a cycle. A softmax takes 1170 cycles (290 to the
// maximum, 820 for the weights, with the other CTA's on the same units), and its next
// scores queue 470 behind the other CTA's products. 64 nodes of 64 heads (four items)
// over 8192 keys, 16 sequences, take 284 to 330 us (0.51 to 0.6 of the library's bf16
// rate), 61 nodes over 100001 keys 117 to 142, at 1.5 GHz and 990 W: the power limit's
// clock, so that fewer cycles do not show in full. 8 nodes over 508 keys take 12 us:
// 4 to the first scores, 0.6 a tile, the merge's launch or eight tiles.
// Tried and no faster (the 16 sequences): two query tiles a CTA that share the ring,
// with one MMA warp or two (297 us); 128-key tiles, one CTA to an SM (321) or two
// (337); eight softmax warps a tile with a common maximum (375); all of Q (352) or
// half of it (298, 1810 cycles) in tensor memory, with one S buffer.
#include <algorithm>

#include "kv8.cuh"
#include "tma_host.h"
#include "tree_pieces.h"

namespace ib200 {
namespace atree {

using kv8::elect_one;
using kv8::mbar_expect_tx_if;
using kv8::scaled;
using kv8::tma_load_2d_if;
using kv8::umma_bf16_if;
using kv8::umma_commit_if;
using kv8::umma_f16_ts_if;
using kv8::uniform;

constexpr int D = 128;
constexpr int PAGE = 16;
constexpr int BQ = 128;               // rows of an item
constexpr int BKV = 64;
constexpr int TILE_PAGES = BKV / PAGE;
constexpr int QBLK = 128 * 128;       // bytes of 128 rows x 64 bf16
constexpr int BLK = BKV * 128;        // bytes of 64 rows x 64 bf16
constexpr int TILE = 2 * BLK;         // K or V of 64 keys
constexpr int SLOTS = 5;
constexpr int NUM_THREADS = 192;
constexpr int SMEM_BYTES = 1024 + 2 * QBLK + SLOTS * TILE;  // barriers in the first 1024; two CTAs fill an SM
constexpr uint32_t TMEM_COLS = 256;   // S0 [0,64) S1 [64,128), W over them; O [128,256)
constexpr uint32_t O_COL = 128;
constexpr float kLagLog2 = 8.0f;      // the running maximum may lag by this much
// Weights carry a factor of 2^-32, and a merge's one of 2^-16: 2^24 of the lagging ones, and 2^16 pieces, times bf16's
// largest value are numbers of 32 bits. The sums carry it too, so it divides out (bf16 has the exponents for it).
constexpr float kDownLog2 = 32.0f, kUp = 4294967296.0f, kMergeDownLog2 = 16.0f;
constexpr int kStart = 3;             // what an item's start and end cost, in key tiles

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
  int n_seqs;
  int hq, hkv, G, nodes;   // nodes: of an item, 128 / G
  int blocks;              // items of the longest tree and KV head
  bool cut;                // items may be cut; else one goes to the run in which it begins
  int runs;                // CTAs of the first kernel
  float c;                 // |scale| * log2(e)
  uint32_t q_flip, q_keep;
  float* o_part;           // [2 * runs, 128 rows, 128]: of run w the piece that an item begins with in 2 w + 1, another in 2 w
  float* lse_part;         // [2 * runs, 128]
  int2* pieces;            // [n_seqs, hkv, blocks] first run and number of runs of an item
  __nv_bfloat16* out;
  int ldo;
  int* status;
};

// A sequence: its rows, its keys and how many of them come before the nodes,
// and its items (each KV head's `blocks`, of `tiles` tiles; one where there are no keys).
struct Seq {
  int start, n, ctx, base, blocks, tiles;
  const int* bt;
};
__device__ __forceinline__ Seq sequence(const Params& p, int s, int* status) {
  Seq q;
  const int want = max(p.q_len[s], 0), row = p.bt_rows != nullptr ? p.bt_rows[s] : s;
  q.start = p.q_start[s];
  q.ctx = max(p.ctx_len[s], 0);
  q.n = min(want, min(p.blocks * p.nodes, 32 * p.words));
  q.n = q.start < 0 || q.start > p.T ? 0 : min(q.n, p.T - q.start);
  q.base = q.ctx - want;  // (may be negative: nodes without a key)
  if (q.n < want) record_status_detail(status, kStatusBadIndex, 9, s, want);
  if (q.ctx > p.max_pages * PAGE) record_status_detail(status, kStatusBadIndex, 1, s, q.ctx);
  q.ctx = min(q.ctx, p.max_pages * PAGE);
  q.bt = p.block_table + static_cast<size_t>(row) * p.ld_table;
  if (row < 0 || row >= p.table_rows) {
    record_status_detail(status, kStatusBadIndex, 4, s, row);
    q.ctx = 0;
    q.bt = p.block_table;
  }
  q.blocks = (q.n + p.nodes - 1) / p.nodes;
  q.tiles = max(1, (q.ctx + BKV - 1) / BKV);
  return q;
}

__device__ __forceinline__ long long divide(long long a, long long b) {  // a, b >= 0; in 32 bits where that does
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// A CTA's run, segment by segment. All items lie end to end on a line, an item
// of `tiles` tiles taking kStart + tiles units (its start costs as much as some
// tiles); first each sequence's first 128 rows, then the second ones of those
// that have more, and so on, so that with equal trees the runs that read the
// same keys read them at the same time. Run w of C goes from total * w / C to
// total * (w + 1) / C. Called by whole warps, which all walk alike.
struct Walk {
  long long at, end, first, total;  // this segment's first unit, the run's end, the item's first unit
  int ctas;
  int s, kvh, block;
  Seq sq;

  // units of a sequence's items of one block
  __device__ __forceinline__ static long long units(const Params& p, const Seq& q, int block) {
    return q.blocks > block ? static_cast<long long>(p.hkv) * (kStart + q.tiles) : 0;
  }
  __device__ __forceinline__ Walk(const Params& p, int* status) {
    const int lane = threadIdx.x & 31;
    total = 0;
    Seq mine0{};  // the lane's first sequence
    for (int i = lane; i < p.n_seqs; i += 32) {
      const Seq q = sequence(p, i, status);
      if (i == lane) mine0 = q;
      total += units(p, q, 0) * q.blocks;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    ctas = static_cast<int>(max(1ll, min(static_cast<long long>(gridDim.x), total)));  // every run has a unit
    at = end = 0;
    if (static_cast<int>(blockIdx.x) >= ctas) return;
    at = divide(total * blockIdx.x, ctas);
    end = divide(total * (blockIdx.x + 1), ctas);
    if (at >= end) return;
    long long before = 0;
    for (block = 0; block < p.blocks; ++block) {
      for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
        const int i = s0 + lane;
        const long long mine = i < p.n_seqs ? units(p, s0 == 0 ? mine0 : sequence(p, i, nullptr), block) : 0;
        long long sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long v = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += v;
        }
        const uint32_t has = __ballot_sync(0xffffffffu, at < before + sum);
        if (has != 0) {
          const int l = __ffs(has) - 1;
          s = s0 + l;
          first = before + __shfl_sync(0xffffffffu, sum - mine, l);
          sq = sequence(p, s, nullptr);
          kvh = static_cast<int>(divide(at - first, kStart + sq.tiles));
          first += static_cast<long long>(kvh) * (kStart + sq.tiles);
          if (!p.cut && at > first) {  // the item is the run's in which it begins
            at = first + kStart + sq.tiles;
            enter(p);
          }
          return;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    end = at;  // (the lengths changed under the kernel)
  }
  __device__ __forceinline__ bool more() const { return at < end; }
  __device__ __forceinline__ long long last(const Params& p) const {  // one past the segment
    const long long stop = first + kStart + sq.tiles;
    return p.cut ? min(stop, end) : stop;
  }
  // the segment's key tiles: first one and count
  __device__ __forceinline__ int tile() const { return static_cast<int>(max(0ll, at - first - kStart)); }
  __device__ __forceinline__ int count(const Params& p) const {
    return sq.ctx > 0 ? max(0, static_cast<int>(last(p) - first) - kStart - tile()) : 0;
  }
  // the run that unit u lies in
  __device__ __forceinline__ int run_of(long long u) const { return static_cast<int>(divide((u + 1) * ctas - 1, total)); }
  __device__ __forceinline__ void advance(const Params& p) {
    at = last(p);
    enter(p);
  }
  // to the item that begins at `at`, if the one before ended there
  __device__ __forceinline__ void enter(const Params& p) {
    if (at < first + kStart + sq.tiles) return;
    first = at;
    if (at >= end || ++kvh < p.hkv) return;
    kvh = 0;
    do {  // (units are left, so there is such a sequence)
      if (++s == p.n_seqs) {
        s = 0;
        if (++block >= p.blocks) {  // (the lengths changed under the kernel)
          end = at;
          return;
        }
      }
      sq = sequence(p, s, nullptr);
    } while (sq.blocks <= block);
  }
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

// Writes what is not finite among the values of a segment's nodes to the row's
// output (dst) where the row sees it. Rare, so nothing here is tuned.
template <typename T>
__device__ __noinline__ void write_not_finite(const Params& p, const int* bt, const int* mask, int kvh, int base, int k_lo,
                                              int k_hi, T* dst) {
  for (int d = 0; d < D; d += 2) {
    float lo = 0.f, hi = 0.f;  // an infinity, a NaN, or 0
    for (int k = max(k_lo, max(base, 0)); k < k_hi; ++k) {
      const int j = k - base, page = bt[k / PAGE];
      if (j >= 32 * p.words || (mask[j >> 5] >> (j & 31) & 1) == 0) continue;
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_pages)) continue;
      const uint32_t u = *reinterpret_cast<const uint32_t*>(
          p.v + ((static_cast<size_t>(page) * PAGE + k % PAGE) * p.hkv + kvh) * D + d);
      if ((u & 0x7f80u) == 0x7f80u) lo += bf16_lo(u);
      if ((u & 0x7f800000u) == 0x7f800000u) hi += bf16_hi(u);
    }
    if (lo != 0.f) dst[d] = static_cast<T>(lo);
    if (hi != 0.f) dst[d + 1] = static_cast<T>(hi);
  }
}

__global__ void __launch_bounds__(NUM_THREADS, 2)
    tree_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ CUtensorMap tmK4, const __grid_constant__ CUtensorMap tmV4,
                const __grid_constant__ Params p) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {  // (the 128-byte swizzle counts from multiples of 1024)
    if (threadIdx.x == 0) record_status(p.status, kStatusBadArgs);
    return;
  }
  uint8_t* sQ = smem + 1024;             // dims 0..63, dims 64..127
  uint8_t* sKV = sQ + 2 * QBLK;          // load i in slot i % SLOTS
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint64_t* q_ready = bars;
  uint64_t* full = bars + 1;             // [SLOTS]
  uint64_t* empty = full + SLOTS;        // [SLOTS]
  uint64_t* s_full = empty + SLOTS;      // [2]
  uint64_t* p_full = s_full + 2;         // [2]
  uint64_t* pv_done = p_full + 2;        // [2] W V of tile j commits to pv_done[j & 1]
  uint64_t* drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* not_finite = abort_flag + 1;

  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_ready, 128);
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 128);
      mbar_init(&pv_done[s], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *not_finite = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmK4);
    tma_prefetch_desc(&tmV4);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  Walk walk(p, blockIdx.x == 0 && threadIdx.x < 32 ? p.status : nullptr);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);

  if (warp == 0) {
    // The whole warp runs along and the elected lane issues, so that the operands stay in uniform registers: a lane
    // of its own took some 80 cycles a box, 16 of them a tile of scattered pages.
    const uint32_t on = elect_one();
    // another item of the sequence reads these keys too, or none
    const uint64_t pol = p.blocks > 1 ? policy_evict_last() : policy_evict_first();
    int issued = 0, st = 0, ph = 1;
    bool ok = true;
    for (; walk.more() && ok; walk.advance(p)) {
      const Seq& sq = walk.sq;
      const int kvh = walk.kvh, j_lo = walk.tile(), nk = walk.count(p);
      if (nk == 0) continue;
      const int n_pages = (sq.ctx + PAGE - 1) / PAGE;
      int next[TILE_PAGES], pages[TILE_PAGES], before[TILE_PAGES];  // of K's next tile, K's, V's
      auto load_pages = [&](int j) {
#pragma unroll
        for (int i = 0; i < TILE_PAGES; ++i) {
          const int lp = (j_lo + j) * TILE_PAGES + i;
          next[i] = sq.bt[lp < n_pages ? lp : 0];
        }
      };
      auto load_tile = [&](int j, const int (&at)[TILE_PAGES], const CUtensorMap* tm1, const CUtensorMap* tm4) {
        ok = mbar_wait_warp(&empty[st], static_cast<uint32_t>(ph), abort_flag, p.status, kStatusTimeoutEmpty);
        if (!ok) return;
        // consecutive pages are one box per half (the swizzle repeats every 8 rows)
        bool run = true;
#pragma unroll
        for (int pg = 1; pg < TILE_PAGES; ++pg) run = run && at[pg] == at[0] + pg;
        const int n = min(TILE_PAGES, n_pages - (j_lo + j) * TILE_PAGES);  // pages that the sequence has here
        uint8_t* dst = sKV + st * TILE;
        mbar_expect_tx_if(on, &full[st], 2 * n * PAGE * 128);
        if (run && n == TILE_PAGES) {
          tma_load_2d_if(on, dst, tm4, &full[st], kvh * D, at[0] * PAGE, pol);
          tma_load_2d_if(on, dst + BLK, tm4, &full[st], kvh * D + 64, at[0] * PAGE, pol);
        } else {
#pragma unroll
          for (int pg = 0; pg < TILE_PAGES; ++pg)
            if (pg < n) {
              tma_load_2d_if(on, dst + pg * PAGE * 128, tm1, &full[st], kvh * D, at[pg] * PAGE, pol);
              tma_load_2d_if(on, dst + BLK + pg * PAGE * 128, tm1, &full[st], kvh * D + 64, at[pg] * PAGE, pol);
            }
        }
        ++issued;
        if (++st == SLOTS) {
          st = 0;
          ph ^= 1;
        }
      };
      load_pages(0);
      // in the order in which the MMA warp takes them: K(j), then V(j - 1)
      for (int j = 0; j <= nk && ok; ++j) {
#pragma unroll
        for (int i = 0; i < TILE_PAGES; ++i) {
          before[i] = pages[i];
          const int pg = static_cast<int>(uniform(next[i]));  // (page ids outside the cache load zeros)
          pages[i] = static_cast<unsigned>(pg) < static_cast<unsigned>(p.num_pages) ? pg : -1;
        }
        if (j + 1 < nk) load_pages(j + 1);  // in flight while we wait
        if (j < nk) load_tile(j, pages, &tmK, &tmK4);
        if (j > 0 && ok) load_tile(j - 1, before, &tmV, &tmV4);
      }
    }
    for (int i = max(0, issued - SLOTS); i < issued; ++i)
      mbar_wait_warp(&full[i % SLOTS], static_cast<uint32_t>((i / SLOTS) & 1), nullptr, nullptr, 0, kWaitLimitNs / 4);
  } else if (warp == 1) {
    const uint32_t on = elect_one();
    const uint32_t idesc_s = make_idesc_bf16(128, BKV);
    const uint32_t idesc_o = make_idesc_bf16(128, D, true);  // B = V with adjacent dims (MN-major)
    const uint64_t q_desc = make_sw128_desc(smem_u32(sQ), 16, 1024);
    const uint64_t k_desc = make_sw128_desc(smem_u32(sKV), 16, 1024);
    const uint64_t v_desc = make_sw128_desc(smem_u32(sKV), BLK, 1024);
    bool ok = true;
    int done = 0;        // tiles of the segments before
    int load = 0;        // loads taken
    uint32_t seg = 0;
    // (descriptor addresses are in units of 16 bytes)
    for (; walk.more() && ok; walk.advance(p)) {
    const int nk = walk.count(p);
    if (nk == 0) continue;
    ok = mbar_wait_warp(q_ready, seg++ & 1, abort_flag, p.status, kStatusTimeoutFull);
    for (int j = done; j <= done + nk && ok; ++j) {
      if (j < done + nk) {
        const int i = load++, st = i % SLOTS;
        ok = mbar_wait_warp(&full[st], static_cast<uint32_t>((i / SLOTS) & 1), abort_flag, p.status, kStatusTimeoutFull);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < 8; ++s)
          umma_bf16_if(on, tmem + (j & 1) * BKV, q_desc + ((s >> 2) * QBLK + (s & 3) * 32) / 16,
                       k_desc + (st * TILE + (s >> 2) * BLK + (s & 3) * 32) / 16, idesc_s, s > 0 ? 1u : 0u);
        umma_commit_if(on, &s_full[j & 1]);
        umma_commit_if(on, &empty[st]);
      }
      if (j > done) {
        const int jj = j - 1, i = load++, st = i % SLOTS;
        ok = mbar_wait_warp(&p_full[jj & 1], static_cast<uint32_t>((jj >> 1) & 1), abort_flag, p.status,
                            kStatusTimeoutTmemEmpty) &&
             mbar_wait_warp(&full[st], static_cast<uint32_t>((i / SLOTS) & 1), abort_flag, p.status, kStatusTimeoutFull);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < BKV / 16; ++s)
          // W packs keys 16s .. 16s + 15 of the tile into columns 8s .. 8s + 7 of its S
          umma_f16_ts_if(on, tmem + O_COL, tmem + (jj & 1) * BKV + s * 8, v_desc + (st * TILE + s * 2048) / 16, idesc_o,
                         (jj > done || s > 0) ? 1u : 0u);
        umma_commit_if(on, &pv_done[jj & 1]);
        umma_commit_if(on, &empty[st]);
      }
    }
    done += nk;
    }
    umma_commit_if(on, drain);
    mbar_wait_warp(drain, 0, nullptr, p.status, kStatusTimeoutFull);
  } else {
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    bool ok = true;
    int done = 0;        // tiles of the segments before
    // the W V of tile jj has completed: its commit is completion (jj >> 1) + 1
    // of pv_done[jj & 1], and no later one on that barrier can have been issued
    auto wait_pv = [&](int jj) {
      if (ok) ok = mbar_wait_warp(&pv_done[jj & 1], static_cast<uint32_t>((jj >> 1) & 1), abort_flag, p.status,
                                  kStatusTimeoutTmemFull);
      tc_fence_after();
    };
    for (; walk.more() && ok; walk.advance(p)) {
    const Seq& sq = walk.sq;
    const int G = p.G, kvh = walk.kvh, block = walk.block;
    const int j_lo = walk.tile(), nk = walk.count(p);
    const int first = block * p.nodes;                  // the item's first node
    const int n_rows = min(p.nodes, sq.n - first) * G;
    const bool live = r < n_rows;
    const int node = first + (live ? r / G : 0), head = kvh * G + (live ? r % G : 0);
    const int row = sq.start + node;
    // the item's pieces are those of the runs that it lies in
    const int run = walk.run_of(walk.first);
    const int pieces = p.cut ? walk.run_of(walk.first + kStart + sq.tiles - 1) - run + 1 : 1;
    const bool begins = walk.at == walk.first;
    const size_t part = (2 * static_cast<size_t>(blockIdx.x) + begins) * BQ + r;
    if (p.cut && begins && threadIdx.x == 64) p.pieces[(walk.s * p.hkv + kvh) * p.blocks + block] = make_int2(run, pieces);
    if (nk == 0) {  // no key tile in this piece, or none at all
      if (live) {
        if (pieces > 1)
          p.lse_part[part] = -INFINITY;
        else
          for (int i = 0; i < D / 8; ++i)
            reinterpret_cast<uint4*>(p.out + static_cast<size_t>(row) * p.ldo + head * D)[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      continue;
    }
    {  // stage this row (rows that do not exist are zero); the scores of the segment before are made
      const uint4* src = reinterpret_cast<const uint4*>(p.q + static_cast<size_t>(row) * p.ldq + head * D);
      uint4 v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = live ? src[i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] = make_uint4((v[i].x ^ p.q_flip) & p.q_keep, (v[i].y ^ p.q_flip) & p.q_keep, (v[i].z ^ p.q_flip) & p.q_keep,
                          (v[i].w ^ p.q_flip) & p.q_keep);
        *reinterpret_cast<uint4*>(sQ + (i >> 3) * QBLK + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = v[i];
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(q_ready);
    }
    const int* mask = p.mask + static_cast<size_t>(row) * p.words;
    const bool awake = __any_sync(0xffffffffu, live);    // a warp without rows only keeps step
    float m_run = -INFINITY;
    float l_run = 0.f;
    for (int j = done; j < done + nk && ok; ++j) {
      const int k0 = (j_lo + j - done) * BKV;
      // the tile has nodes, or ends behind the sequence (whose nodes lie behind its keys where the table cuts it)
      const bool edge = k0 + BKV > min(sq.base, sq.ctx);
      if (!mbar_wait_warp(&s_full[j & 1], static_cast<uint32_t>((j >> 1) & 1), abort_flag, p.status,
                          kStatusTimeoutTmemFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (edge) {
        // V rows of the tile, half a row a thread: zeroed behind the sequence, and where a node's is not finite. (S of
        // this tile was issued after the product that freed the slot: the barrier is in this load's phase or past it.)
        const int at = j - done, i = 2 * done + (at + 1 < nk ? 2 * at + 2 : 2 * nk - 1);  // loads: K0, K1, V0, K2, V1, ..
        const int st = i % SLOTS, vr = r & (BKV - 1), key = k0 + vr;
        if (!mbar_wait_warp(&full[st], static_cast<uint32_t>((i / SLOTS) & 1), abort_flag, p.status, kStatusTimeoutFull)) {
          ok = false;
          break;
        }
        uint8_t* src = sKV + st * TILE + (r >> 6) * BLK + vr * 128;
        if (key >= sq.ctx) {
#pragma unroll
          for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(src + c * 16) = make_uint4(0u, 0u, 0u, 0u);
        } else if (key >= sq.base) {
#pragma unroll 4
          for (int c = 0; c < 8; ++c) {
            uint4* at = reinterpret_cast<uint4*>(src + ((c ^ (vr & 7)) << 4));
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
      if (awake) {
        const uint32_t s_addr = lane_addr + (j & 1) * BKV;
        uint32_t v[BKV];
        tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        tmem_ld_wait();
        if (edge) {
          const uint64_t seen = seen_of(mask, p.words, k0, sq.base, sq.ctx);
          const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
#pragma unroll
          for (int i = 0; i < BKV; ++i)
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
          if (j > done) {
            // O *= alpha once the W V of the tile before has landed; none is issued until this tile's W is published
            wait_pv(j - 1);
            if (!ok) break;
#pragma unroll 1
            for (int c0 = 0; c0 < 128; c0 += 32) {
              uint32_t o[32];
              tmem_ld32(lane_addr + O_COL + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(lane_addr + O_COL + c0, o);
            }
          }
          m_run = m_use;
        }
        const float m_ref = m_run == -INFINITY ? 0.f : m_run;
        // w = 2^(c s - m - 32) as bf16 pairs over the S columns just read
        const uint64_t c2 = f2pack(p.c, p.c), b2 = f2pack(-m_ref - kDownLog2, -m_ref - kDownLog2);
        uint64_t l2[2] = {f2pack(0.f, 0.f), f2pack(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < BKV; i += 2) {
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
      mbar_arrive(&p_full[j & 1]);
    }
    ok = __all_sync(0xffffffffu, ok);
    done += nk;
    wait_pv(done - 1);
    if (ok) {
      const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;   // a NaN stays one
      const bool merge = pieces > 1;
      if (merge && live) p.lse_part[part] = l_run == 0.f ? -INFINITY : m_run + log2f(l_run * kUp);
#pragma unroll 1
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(lane_addr + O_COL + c0, o);
        tmem_ld_wait();
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = l_run == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
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
      if (*not_finite != 0 && live) {
        const int k_lo = j_lo * BKV, k_hi = min(sq.ctx, (j_lo + nk) * BKV);
        if (merge)
          write_not_finite(p, sq.bt, mask, kvh, sq.base, k_lo, k_hi, p.o_part + part * D);
        else
          write_not_finite(p, sq.bt, mask, kvh, sq.base, k_lo, k_hi, p.out + static_cast<size_t>(row) * p.ldo + head * D);
      }
      __syncwarp();
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

// Merge the pieces of cut items,
//   o = sum_k 2^(lse_k - M) o_k / sum_k 2^(lse_k - M)
// LANES lanes a row, which have 4 dims of each 4 LANES, and W warps that share a row's pieces. With two pieces a
// row most instructions are the row's, not the pieces', so 8 lanes take a row, and a warp four (65536 rows of 16
// sequences, 64 nodes, 64 heads: 12 us from cold caches; a warp a row 22).
template <int LANES, int W>
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ Params p) {
  constexpr int V = 32 / LANES;              // float4s a lane
  constexpr int ROWS = 8 / W * V;            // of a block
  constexpr int AHEAD = W > 1 ? 4 : 2;       // pieces under way
  static_assert(W == 1 || (W == 8 && V == 1), "the barrier below is the row's");
  pdl_trigger();
  pdl_wait();
  const int item = blockIdx.x, s = item / (p.hkv * p.blocks), kvh = item / p.blocks % p.hkv, block = item % p.blocks;
  const int2 pc = p.pieces[item];  // (of an item that there is)
  const Seq sq = sequence(p, s, nullptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LANES - 1);
  const int w0 = warp % W, r = blockIdx.y * ROWS + warp / W * V + (threadIdx.x & 31) / LANES;
  const int at = r / p.G, node = block * p.nodes + at;
  if (at >= p.nodes || node >= sq.n || pc.y <= 1 || !pieces_exist(pc.x, pc.y, p.runs)) return;  // (the same for a row's warps)
  auto part = [&](int k) { return static_cast<size_t>(piece_at(pc.x, k)) * BQ + r; };
  float num[V][4] = {}, den = 0.f, top = -INFINITY;
  for (int k0 = w0; k0 < pc.y; k0 += AHEAD * W) {
    float lse[AHEAD];
    float4 o[AHEAD][V];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int k = k0 + i * W;
      lse[i] = -INFINITY;
      if (k < pc.y) {
        lse[i] = p.lse_part[part(k)];
        const float4* src = reinterpret_cast<const float4*>(p.o_part + part(k) * D) + lane;
#pragma unroll
        for (int v = 0; v < V; ++v) o[i][v] = src[v * LANES];
      }
    }
    float mx = top;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) mx = fmaxf(mx, lse[i]);
    const float f = top == -INFINITY ? 0.f : exp2f(top - mx);
    den *= f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int d = 0; d < 4; ++d) num[v][d] = scaled(num[v][d], f);
    top = mx;
    const float ref = mx == -INFINITY ? 0.f : mx + kMergeDownLog2;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (lse[i] == -INFINITY) continue;  // (a piece without keys wrote no more)
      const float w = exp2f(lse[i] - ref);
      den += w;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        num[v][0] += scaled(o[i][v].x, w);
        num[v][1] += scaled(o[i][v].y, w);
        num[v][2] += scaled(o[i][v].z, w);
        num[v][3] += scaled(o[i][v].w, w);
      }
    }
  }
  if constexpr (W > 1) {
    __shared__ float4 s_num[W][32];
    __shared__ float2 s_den[W];
    s_num[w0][lane] = make_float4(num[0][0], num[0][1], num[0][2], num[0][3]);
    if (lane == 0) s_den[w0] = make_float2(top, den);
    __syncthreads();
    if (w0 != 0) return;
    float mx = -INFINITY;
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_den[w].x);
    den = num[0][0] = num[0][1] = num[0][2] = num[0][3] = 0.f;
    for (int w = 0; w < W; ++w) {
      const float2 td = s_den[w];
      if (td.x == -INFINITY && td.y == 0.f) continue;
      const float f = exp2f(td.x - mx);
      const float4 v = s_num[w][lane];
      den += td.y * f;
      num[0][0] += scaled(v.x, f);
      num[0][1] += scaled(v.y, f);
      num[0][2] += scaled(v.z, f);
      num[0][3] += scaled(v.w, f);
    }
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  uint2* dst = reinterpret_cast<uint2*>(p.out + static_cast<size_t>(sq.start + node) * p.ldo + (kvh * p.G + r - at * p.G) * D) + lane;
#pragma unroll
  for (int v = 0; v < V; ++v)
    dst[v * LANES] = make_uint2(pack_bf16(num[v][0] * inv, num[v][1] * inv), pack_bf16(num[v][2] * inv, num[v][3] * inv));
}

}  // namespace atree
}  // namespace ib200

using namespace ib200;

// q [T, ldq] bf16 (head h at columns h*128); caches bf16 [num_slots, hkv*128];
// q_start / q_len / ctx_len [n_seqs], ctx_len with the nodes; mask int32 [T,
// words]; max_nodes: the most nodes of a sequence. ctas: equal runs that all
// items' units are cut into; o_part null: an item goes to the run in which it
// begins. o_part / lse_part: fp32 [2*ctas*128*128] / [2*ctas*128], pieces
// [2 * n_seqs * hkv * ceil(max_nodes / (128 / G))].
extern "C" int ib_attn_tree(const void* q, int T, int ldq, const void* k_cache, const void* v_cache, long long num_slots,
                            const int* q_start, const int* q_len, const int* ctx_len, const int* mask, int words,
                            int n_seqs, int max_nodes, const int* block_table, const int* bt_rows, int table_rows,
                            int max_pages, int ld_table, int hq, int hkv, float scale, int ctas,
                            float* o_part, float* lse_part, int* pieces, void* out, int ldo, int* status, cudaStream_t stream) {
  using namespace ib200::atree;
  if (T <= 0 || n_seqs <= 0 || max_nodes <= 0) return 0;
  if (hkv <= 0 || hq % hkv != 0 || hq / hkv > 16 || ctas < 1 || words < 1 || words > 8 ||
      max_nodes > 32 * words || n_seqs > 65535 || (ldq % 8) != 0 || (ldo % 8) != 0 || num_slots < PAGE ||
      num_slots % PAGE != 0 || max_pages < 0 || max_pages > (1 << 26) ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
    return -1;
  if (o_part != nullptr && (lse_part == nullptr || pieces == nullptr || (reinterpret_cast<uintptr_t>(o_part) & 15) != 0 ||
                            (reinterpret_cast<uintptr_t>(pieces) & 7) != 0))
    return -1;
  try {
    const int kvw = hkv * D;
    CUtensorMap tk, tv, tk4, tv4;
    const auto bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (!cached_tmap_2d(&tk, k_cache, bf, 2, num_slots, kvw, kvw, 16, 64) ||
        !cached_tmap_2d(&tv, v_cache, bf, 2, num_slots, kvw, kvw, 16, 64) ||
        !cached_tmap_2d(&tk4, k_cache, bf, 2, num_slots, kvw, kvw, BKV, 64) ||
        !cached_tmap_2d(&tv4, v_cache, bf, 2, num_slots, kvw, kvw, BKV, 64))
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
    p.nodes = BQ / p.G;
    p.blocks = (max_nodes + p.nodes - 1) / p.nodes;
    p.n_seqs = n_seqs;
    p.cut = o_part != nullptr;
    p.runs = ctas;
    p.pieces = reinterpret_cast<int2*>(pieces);
    p.c = fmaxf(fabsf(scale) * 1.4426950408889634f, 1.2e-38f);  // positive: masked scores are -inf times it
    p.q_flip = scale < 0.f ? 0x80008000u : 0u;
    p.q_keep = scale == 0.f ? 0u : ~0u;
    p.o_part = o_part;
    p.lse_part = lse_part;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.ldo = ldo;
    p.status = status;
    static bool attr_set[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t e;
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
      e = cudaFuncSetAttribute(tree_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
      if (e != cudaSuccess) return static_cast<int>(e);
      if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    e = launch_pdl(tree_kernel, dim3(ctas), NUM_THREADS, SMEM_BYTES, stream, tk, tv, tk4, tv4, p);
    if (e != cudaSuccess) return static_cast<int>(e);
    const unsigned items = static_cast<unsigned>(n_seqs) * hkv * p.blocks;
    // few items have many pieces: a block a row then (61 nodes of 32 heads over 100001 keys, 20 pieces)
    if (p.cut && 4 * items <= static_cast<unsigned>(ctas))
      e = launch_pdl(merge_kernel<32, 8>, dim3(items, BQ), 256, 0, stream, p);
    else if (p.cut)
      e = launch_pdl(merge_kernel<8, 1>, dim3(items, BQ / 32), 256, 0, stream, p);
    return static_cast<int>(e);
  } catch (...) {  // (no memory for a tensor map's entry)
    return -3;
  }
}
