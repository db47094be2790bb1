// paged_attention.cu — attention of one new token per sequence over a paged key-value cache.
//
//   out[b, h, :] = sum_j w_j V[j] / sum_j w_j,   w_j = exp(scale * q[b, h] . K[j]),   lse[b, h] = log(sum_j w_j)
//
// over the keys j that the newest token sees: all of the sequence's lens[b], or, with a window, the last `window` of them and
// the first `sinks`.  Key j lies in slot j % page_size of page block_table[b, j / page_size]; query head h reads key head
// h / (heads / kv_heads).  16-bit elements, fp32 sums, head dimension 64, 128 or 256.  No counterpart in the reference.
//
// Every key and value is read once (once for every 16 query heads that share it) and used for 2 * group products: HBM bounds it,
// and the work goes into an even share of the bytes for every SM, enough of them in flight, and few instructions per byte.
//   * The keys that are seen are counted through in blocks of 16 (first keys, then the window), so a mask costs nothing but at
//     the blocks' edges: a position in that count gives the key, the key its page.
//   * One warp loads: it looks the pages of 32 blocks up at a time, a batch ahead, and has the TMA unit copy the blocks (a 4-D
//     tensor map over component, head, slot and page, so any order of them in memory) into a ring of tiles.  (With the copies
//     in the warps that compute, cp.async a lane, a step was 460 instructions and 1300 cycles.  Keys and values copied as one,
//     through a fifth dimension: no gain, 173.8 us for 174.0 with heads of 64, 95.1 for 94.5 with heads of 128.)
//   * The other warps are workers of their own: each takes its blocks of every tile and keeps its own running maximum, sum and
//     output in registers (one pass).  They meet when a sequence's tiles end.
//   * Products go through mma.sync m16n8k16 with the keys (for the scores) and the components (for the output) as the 16 rows
//     and the query heads that share a key head as the 8 columns: half as many instructions as with the heads as rows, for up
//     to 8 heads.  (A tcgen05 tile is 128 rows; the rate asked for here is 1 % of what those do.)
//   * A step that raises no running maximum, which a vote finds out, needs no reduction over lanes.
//   * The weights enter the second product as two 16-bit numbers, the rounded value and what it lost, so that the output has
//     one rounding to 16 bits, its own.  fp16 has no numbers below 2^-24, so there the largest weight is 2^14 instead of 1:
//     what is lost of a weight is at most 2^-39 of the largest.
// Two ways to share out the keys:
//   cluster  the CTAs of a cluster take equal parts of one sequence and key head and add up through distributed shared
//            memory: one launch, no workspace.  For sequences of few tiles.
//   stream   every CTA takes an equal part of all tiles of all sequences in a row, wherever that part begins and ends; parts
//            of a sequence that spans CTAs go to a workspace and a second kernel, started early, adds them up in their order.
//            Neighbouring heads, whose rows are neighbours in memory where the slot comes before the head, belong to CTAs that
//            run side by side through the same keys (`lanes`), which DRAM rewards: 256 sequences of up to 2000 keys, 32 heads of
//            64, 437 us with the heads one behind the other, 356 side by side.
// Both give the same bits in every run: no atomics, and parts are added in a fixed order.
//
// Every wait on an mbarrier is bounded by timeout_ns: on expiry the CTA records a status, the loads stop, and the other warps run
// their loops to the end without computing, so that they meet at all their barriers.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <atomic>
#include <mutex>

#include "iris/iris.cuh"
#include "iris/overlap.cuh"
#include "iris/ptx_sm100.cuh"

namespace iris {
namespace paged {

using namespace iris::ptx;

constexpr int kRows = 16;                        // query heads of a segment, at most
constexpr int kBlock = 16;                       // keys of a product
constexpr int kHalfBlock = kBlock * 128;         // bytes of a block's keys (or values) in a panel
constexpr int kJoinThreads = 512;
constexpr int64_t kMostKeys = 0x7fffffff - 1023;   // of a sequence: positions are looked at up to a batch of blocks behind the last
// What the exponents of the weights are counted from, for a maximum m.  fp16: weights are made 2^14 times as large.  (At 1, 20000
// keys that weigh 2^-26 of the largest each, 3e-4 of the sum, were left out of the output; 14 and not 15, as a score's rounding may
// put a weight above the maximum's.)  Not where m is so large that its own rounding would take a weight out of what fp16 holds.
template <bool F16>
__device__ __forceinline__ float origin(float m) { return F16 && fabsf(m) < 4194304.f ? m - 14.f : m; }
constexpr uint32_t kSitePage = 95, kSiteLoad = 98, kSiteTile = 99;

template <int D, int COLS = 8>
struct Shape {
  static constexpr int kWarps = D == 256 ? 2 : 4;              // that compute; one more loads
  static constexpr int kThreads = (kWarps + 1) * 32;
  static constexpr int kBlocks = D == 64 ? 2 : 1;              // blocks of a warp in a tile
  static constexpr int kTileBlocks = kWarps * kBlocks;
  static constexpr int kTile = kTileBlocks * kBlock;           // keys of a tile
  static constexpr int kStages = D == 256 ? 2 : 3;             // ring of tiles
  static constexpr int kQBufs = kStages;                       // queries of the segments that the ring reaches
  static constexpr int kPanels = D / 64;                       // a tile lies in panels of 64 components,
  static constexpr int kBlockBytes = 2 * kHalfBlock;           // a block of a panel: rows of 128 bytes, keys and values
  static constexpr int kPanel = kTileBlocks * kBlockBytes;
  static constexpr int kStageBytes = kPanels * kPanel;         // 32 KB
  static constexpr int kQPitch = D * 2 + 16;                   // (rows 16 bytes apart in the banks)
  static constexpr int kQBytes = COLS * kQPitch;
  static constexpr int kStats = 2 * kWarps * kRows * 4;        // maxima and sums of the warps
  static constexpr int kBars = 2 * kStages * 8;
  static constexpr int kWords = (kStages * kTileBlocks + 8) * 4;   // which keys of a block count, and a few others
  static constexpr int kUsed = kStages * kStageBytes + kQBufs * kQBytes + kStats + kBars + kWords;
  static constexpr int kSmem = kUsed + 1024;                   // (the ring begins on 1024 bytes)
  static constexpr int kPerSm = 2;
  static_assert(kStageBytes >= kWarps * COLS * D * 4, "ring");
  static_assert(kPerSm * (kSmem + 1024) <= 228 * 1024, "shared-memory budget");
};

struct Params {
  CUtensorMap k, v;          // [pages, slots, key heads, components], box: 64 components of one head, a block or a page of fewer rows
  const uint8_t* q;          // strides in bytes
  const int* table;
  const int* lens;
  uint8_t* out;
  float* lse;                // may be null
  StatusBlock* status;       // may be null
  float* parts;              // stream: [ctas][2][rows][D], then maxima and sums [ctas][2][rows][2]
  int4* jobs;                // stream: what the second kernel adds up
  uint64_t timeout_ns;
  int64_t q_batch, q_head, table_pitch, out_batch, out_head, lse_batch;
  int batch, group, row_tiles, segments_per_seq, pages, page_shift, wide, window, sinks;
  int lanes, turns;          // segments of a sequence (key head and row tile) = turns * lanes: number turn * lanes + lane
  int groups, rows;          // stream: CTA g * lanes + lane of the first kernel takes the g-th part of the lane's tiles; rows of a part
  float scale_log2;
};

__device__ __forceinline__ float exp2_fast(float x) {   // ex2.approx: 2 ulp, 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The 8 x 8 matrix of 16-bit elements whose row g lane 4 g + t holds columns 2 t and 2 t + 1 of, transposed.
__device__ __forceinline__ uint32_t transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if (F16) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&b);
}
template <bool F16>
__device__ __forceinline__ float2 unpack(uint32_t v) {
  return F16 ? __half22float2(*reinterpret_cast<__half2*>(&v)) : __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}

// The keys that a sequence's newest token sees, counted through in whole blocks: positions 0 .. head - 1 are the keys of that
// number, of which those below `sinks` count, the others key position + skip, of which those from `start` to `len` do.
struct Seen {
  int n, head, sinks, skip, start, len;
};
__device__ __forceinline__ Seen seen_of(const Params& p, int len) {
  const int64_t cap = (int64_t)p.wide << p.page_shift;
  len = len < 0 ? 0 : (int64_t)len > cap ? (int)cap : len;
  Seen s;
  s.len = len;
  s.start = p.window > 0 && len > p.window ? len - p.window : 0;
  s.sinks = min(p.sinks, s.start);
  s.head = (s.sinks + kBlock - 1) & ~(kBlock - 1);
  s.skip = (s.start & ~(kBlock - 1)) - s.head;
  s.n = len - s.skip;
  return s;
}
// The block's keys that count, a bit each, and the first of them all.
__device__ __forceinline__ uint32_t block_mask(const Seen& s, int at, int& key) {
  const bool first = at < s.head;
  key = first ? at : at + s.skip;
  const int from = first ? 0 : s.start - key, to = (first ? s.sinks : s.len) - key;
  if (to <= 0) return 0;
  return (to >= kBlock ? 0xffffu : (1u << to) - 1) & (from > 0 ? 0xffffu << from : 0xffffu);
}
template <int D>
__device__ __forceinline__ int tiles_of(const Seen& s) {   // a sequence without keys has one tile too: its output is zeros
  constexpr int kTile = Shape<D>::kTile;
  const int t = s.n / kTile + (s.n % kTile != 0);
  return t ? t : 1;
}

// Where a worker is: tile `tile` of `tiles` of the segment that is its lane's in turn `seg` of sequence b.
struct Cursor {
  Seen s;
  int b, seg, tile, tiles, next_len;
};
template <int D>
__device__ __forceinline__ void enter(const Params& p, Cursor& c, int len) {
  c.s = seen_of(p, len);
  c.tiles = tiles_of<D>(c.s);
  c.next_len = c.b + 1 < p.batch ? p.lens[c.b + 1] : 0;
}
// Whether a new segment begins.
template <int D>
__device__ __forceinline__ bool advance(const Params& p, Cursor& c) {
  if (++c.tile < c.tiles) return false;
  c.tile = 0;
  if (++c.seg == p.turns) {
    c.seg = 0;
    if (++c.b < p.batch) enter<D>(p, c, c.next_len);
  }
  return true;
}

// Joins a part with maximum m2 and sum l2 (not 0) to (m, l); f and f2: what the outputs of the two are multiplied by.
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2, float& f, float& f2) {
  const float top = fmaxf(m, m2);
  f = m == top ? 1.f : exp2_fast(m - top);
  f2 = m2 == top ? 1.f : exp2_fast(m2 - top);
  l = l * f + l2 * f2;
  m = top;
}
__device__ __forceinline__ void add(float4& a, float f, const float4& x, float f2) {
  a.x = a.x * f + x.x * f2, a.y = a.y * f + x.y * f2, a.z = a.z * f + x.z * f2, a.w = a.w * f + x.w * f2;
}
__device__ __forceinline__ float log_sum(float m, float l) {   // m in powers of two
  return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}
// One output row of 4 columns: rounded to 16 bits.
template <bool F16>
__device__ __forceinline__ void store4(uint8_t* dst, float4 a, float f) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack<F16>(a.x * f, a.y * f), pack<F16>(a.z * f, a.w * f));
}

// COLS: columns of heads, 8 or 16.
template <int D, bool F16, bool CLUSTER, int COLS>
__global__ void __launch_bounds__(Shape<D, COLS>::kThreads, Shape<D, COLS>::kPerSm)
    paged_attention_kernel(const __grid_constant__ Params p) {
  using S = Shape<D, COLS>;
  constexpr int kWarps = S::kWarps, kB = S::kBlocks, kTile = S::kTile, kTB = S::kTileBlocks;
  constexpr int kN = COLS / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_mem = smem + S::kStages * S::kStageBytes;
  float* stat_m = reinterpret_cast<float*>(q_mem + S::kQBufs * S::kQBytes);
  float* stat_l = stat_m + kWarps * kRows;
  const uint32_t bars = smem_u32(stat_l + kWarps * kRows);
  volatile uint32_t* masks = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(stat_l + kWarps * kRows) + S::kBars);
  volatile int* words = reinterpret_cast<int*>(const_cast<uint32_t*>(masks) + S::kStages * kTB);
  volatile uint32_t* abort_flag = const_cast<volatile uint32_t*>(masks) + S::kStages * kTB + 4;
  volatile uint32_t* never = abort_flag + 1;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (S::kStages + s); };
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;     // scores: keys g and g + 8 of a block, heads 2 t and 2 t + 1
  const uint32_t ring = smem_u32(smem), q_s = smem_u32(q_mem);

  if (threadIdx.x == 0) {
    prefetch_tensormap(&p.k);
    prefetch_tensormap(&p.v);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), kWarps);
    }
    *abort_flag = *never = 0;
    mbar_fence_init();
  }
  // columns of no head are zeros
  for (int i = threadIdx.x; i < S::kQBufs * S::kQBytes / 16; i += S::kThreads) reinterpret_cast<uint4*>(q_mem)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_launch();

  // ---- this CTA's tiles: from cursor c on, `count` of them ----
  Cursor c;
  int64_t first = 0, total = 0;              // stream: its first tile among all
  int count, groups = 1;
  const int lane_of = CLUSTER ? blockIdx.y : blockIdx.x % p.lanes, my_group = CLUSTER ? 0 : blockIdx.x / p.lanes;
  auto segment_of = [&](const Cursor& at) { return at.seg * p.lanes + lane_of; };
  if (CLUSTER) {
    c.b = blockIdx.z;
    c.seg = 0;
    enter<D>(p, c, p.lens[c.b]);
    const int parts = gridDim.x, r = blockIdx.x;
    c.tile = (int)((int64_t)c.tiles * r / parts);
    count = (int)((int64_t)c.tiles * (r + 1) / parts) - c.tile;
  } else {
    // tiles of the sequences before each thread's share of them
    const int per = (p.batch + S::kThreads - 1) / S::kThreads;
    const int b0 = min(p.batch, (int)threadIdx.x * per), b1 = min(p.batch, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of<D>(seen_of(p, p.lens[b]));
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    int64_t* sums = reinterpret_cast<int64_t*>(stat_m);
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t before = upto - mine;
#pragma unroll
    for (int w = 0; w <= kWarps; ++w) {
      if (w < warp) before += sums[w];
      total += sums[w];
    }
    total *= p.turns;
    before *= p.turns;
    mine *= p.turns;
    groups = (int)min((int64_t)p.groups, total);   // with a tile each at least: a part from every CTA that a segment spans
    if (my_group >= groups) return;                // (then the jobs are listed by segment)
    first = total * my_group / groups;
    count = (int)(total * (my_group + 1) / groups - first);
    if (mine > 0 && before <= first && first < before + mine) {
      int64_t left = first - before;
      int b = b0, n, len;
      for (;; ++b) {
        len = p.lens[b];
        n = tiles_of<D>(seen_of(p, len));
        if (left < (int64_t)n * p.turns) break;
        left -= (int64_t)n * p.turns;
      }
      const int turn = p.turns == 1 ? 0 : (int)(left / n);
      words[0] = b;
      words[1] = turn;
      words[2] = (int)(left - (int64_t)turn * n);
      words[3] = len;
    }
    __syncthreads();
    c.b = words[0];
    c.seg = words[1];
    enter<D>(p, c, words[3]);
    c.tile = words[2];
  }

  if (warp == kWarps) {
    // ---- loads ----
    // A batch: 32 blocks of one segment, a lane each: which of its keys count, its page (pages of 8: its two) and its first slot.
    constexpr int kBatch = 32 / kTB;          // tiles
    struct Batch {
      uint32_t mask;
      int page, page2, slot, key;
    };
    const bool whole_blocks = p.page_shift >= 4, two_pages = p.page_shift == 3;
    auto look_up = [&](const Cursor& at, int left) {
      Batch b;
      b.key = 0;
      b.mask = left > 0 ? block_mask(at.s, at.tile * kTile + lane * kBlock, b.key) : 0;
      b.page = b.page2 = 0;
      b.slot = b.key & ((1 << p.page_shift) - 1);
      const int* row = p.table + at.b * p.table_pitch + (b.key >> p.page_shift);
      if (whole_blocks ? b.mask : two_pages ? b.mask & 0xff : 0) b.page = row[0];
      if (two_pages && b.mask >> 8) b.page2 = row[1];
      return b;
    };
    // the cursor of the batch behind the one at c, of `left` tiles yet to come: what the latter leaves of them
    auto next_batch = [&](Cursor& at, int& left) {
      const int n = min(kBatch, at.tiles - at.tile);
      left -= n;
      if (left <= 0) return;
      at.tile += n - 1;
      advance<D>(p, at);
    };
    Cursor l = c, ahead = c;
    int ahead_left = count, in_batch = 0, stage = 0, q_buf = 0;
    bool fresh = true;                        // the next tile is its segment's first here
    Batch now = look_up(l, count);
    next_batch(ahead, ahead_left);
    Batch next = look_up(ahead, ahead_left);
    int issued = 0;
    for (; issued < count; ++issued) {
      const int use = issued / S::kStages;
      if (use > 0 && !mbar_wait_warp(empty(stage), (use - 1) & 1, p.timeout_ns, abort_flag)) {
        if (lane == 0) record_status(p.status, kTimeout, kSiteLoad, blockIdx.x, issued, 0);
        *abort_flag = 1;
        break;
      }
      const int first_lane = in_batch * kTB;
      const bool mine = lane >= first_lane && lane < first_lane + kTB;
      uint32_t mask = now.mask;
      if (whole_blocks && mask && (uint32_t)now.page >= (uint32_t)p.pages) {
        if (mine) record_status(p.status, kBadPointer, kSitePage, l.b, now.key, (uint64_t)(int64_t)now.page);
        mask = 0;
      }
      if (two_pages) {
        uint32_t bad = (uint32_t)now.page >= (uint32_t)p.pages ? 0xffu : 0;
        if ((uint32_t)now.page2 >= (uint32_t)p.pages) bad |= 0xff00u;
        if (mine && bad & mask)
          record_status(p.status, kBadPointer, kSitePage, l.b, now.key, (uint64_t)(int64_t)(bad & mask & 0xff ? now.page : now.page2));
        mask &= ~bad;
      }
      const int seg = segment_of(l), kv = p.row_tiles == 1 ? seg : seg / p.row_tiles, r0 = (seg - kv * p.row_tiles) * kRows;
      const int rows = fresh ? min(COLS, p.group - r0) : 0;
      const uint32_t tile = ring + stage * S::kStageBytes;
      if (whole_blocks || two_pages) {
        const uint32_t blocks = __ballot_sync(0xffffffffu, mine && mask) >> first_lane;
        if (mine) masks[stage * kTB + lane - first_lane] = mask;
        __syncwarp();
        const bool one = elect_one();
        if (one) mbar_expect_tx(full(stage), __popc(blocks) * (S::kPanels * S::kBlockBytes) + rows * D * 2);
        if (whole_blocks) {
#pragma unroll
          for (int b = 0; b < kTB; ++b) {
            const int page = __shfl_sync(0xffffffffu, now.page, first_lane + b), slot = __shfl_sync(0xffffffffu, now.slot, first_lane + b);
            if (one && (blocks >> b & 1)) {
              const uint32_t at = tile + b * S::kBlockBytes;
#pragma unroll
              for (int h = 0; h < S::kPanels; ++h) tma_load_4d(at + h * S::kPanel, &p.k, h * 64, kv, slot, page, full(stage));
#pragma unroll
              for (int h = 0; h < S::kPanels; ++h)
                tma_load_4d(at + h * S::kPanel + kHalfBlock, &p.v, h * 64, kv, slot, page, full(stage));
            }
          }
        } else {
          // pages of 8 (half of a block of which no key is seen is copied all the same, from page 0)
#pragma unroll
          for (int i = 0; i < 2 * kTB; ++i) {
            const int page = __shfl_sync(0xffffffffu, i & 1 ? now.page2 : now.page, first_lane + i / 2);
            if (one && (blocks >> i / 2 & 1)) {
              const uint32_t at = tile + i / 2 * S::kBlockBytes + (i & 1) * 1024;
#pragma unroll
              for (int h = 0; h < S::kPanels; ++h) {
                tma_load_4d(at + h * S::kPanel, &p.k, h * 64, kv, 0, page, full(stage));
                tma_load_4d(at + h * S::kPanel + kHalfBlock, &p.v, h * 64, kv, 0, page, full(stage));
              }
            }
          }
        }
        if (one && rows > 0) {
          const uint8_t* src = p.q + l.b * p.q_batch + (int64_t)(kv * p.group + r0) * p.q_head;
          const uint32_t dst = q_s + q_buf * S::kQBytes;
          for (int r = 0; r < rows; ++r) bulk_load(dst + r * S::kQPitch, src + r * p.q_head, D * 2, full(stage));
        }
      } else {
        // pages of fewer than 8 keys: looked up a key a lane, all blocks at once, and copied a page at a time
        const int size = 1 << p.page_shift;
        int page[kTB];
        uint32_t got[kTB], bytes = 0;
#pragma unroll
        for (int b = 0; b < kTB; ++b) {
          const uint32_t m = __shfl_sync(0xffffffffu, now.mask, first_lane + b);
          const int key = __shfl_sync(0xffffffffu, now.key, first_lane + b) + (lane & 15);
          got[b] = m >> (lane & 15) & 1;
          page[b] = got[b] ? p.table[l.b * p.table_pitch + (key >> p.page_shift)] : -1;
        }
#pragma unroll
        for (int b = 0; b < kTB; ++b) {
          const bool good = got[b] && (uint32_t)page[b] < (uint32_t)p.pages;
          const int key = __shfl_sync(0xffffffffu, now.key, first_lane + b) + (lane & 15);
          if (got[b] && !good) record_status(p.status, kBadPointer, kSitePage, l.b, key, (uint64_t)(int64_t)page[b]);
          got[b] = __ballot_sync(0xffffffffu, good) & 0xffffu;
          if (lane == 0) masks[stage * kTB + b] = got[b];
          for (int j = 0; j < kBlock; j += size)
            if (got[b] >> j & ((1u << size) - 1)) bytes += size * 128 * 2 * S::kPanels;
        }
        __syncwarp();
        if (lane == 0) mbar_expect_tx(full(stage), bytes + rows * D * 2);
#pragma unroll
        for (int b = 0; b < kTB; ++b) {
          for (int j = 0; j < kBlock; j += size) {
            const uint32_t part = got[b] >> j & ((1u << size) - 1);
            const int from = __shfl_sync(0xffffffffu, page[b], part ? j + __ffs(part) - 1 : 0);
            if (part && lane == 0) {
              const uint32_t at = tile + b * S::kBlockBytes + j * 128;
#pragma unroll
              for (int h = 0; h < S::kPanels; ++h) {
                tma_load_4d(at + h * S::kPanel, &p.k, h * 64, kv, 0, from, full(stage));
                tma_load_4d(at + h * S::kPanel + kHalfBlock, &p.v, h * 64, kv, 0, from, full(stage));
              }
            }
          }
        }
        if (lane == 0) {
          const uint8_t* src = p.q + l.b * p.q_batch + (int64_t)(kv * p.group + r0) * p.q_head;
          const uint32_t dst = q_s + q_buf * S::kQBytes;
          for (int r = 0; r < rows; ++r) bulk_load(dst + r * S::kQPitch, src + r * p.q_head, D * 2, full(stage));
        }
      }
      __syncwarp();
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
      fresh = advance<D>(p, l);
      if (fresh) q_buf = q_buf + 1 == S::kQBufs ? 0 : q_buf + 1;
      if (++in_batch == kBatch || fresh) {
        in_batch = 0;
        now = next;
        next_batch(ahead, ahead_left);
        next = look_up(ahead, ahead_left);
      }
    }
    // loads in flight write into this CTA's shared memory, whether the other warps still wait for them or not: wait for each, bounded
    for (int s = 0; s < S::kStages; ++s) {
      const int n = (issued + S::kStages - 1 - s) / S::kStages;
      if (n > 0) mbar_wait(full(s), (n - 1) & 1, 200000, never);
    }
    __syncwarp();
    if (CLUSTER && gridDim.x > 1) {
      cluster_sync_all();
      cluster_sync_all();
    }
    return;
  }

  // ---- products ----
  float o[D / 16][kN][4], m[kN][2], sum[kN][2];   // output: components g and g + 8 of 16, heads 2 t and 2 t + 1
  uint32_t q[D / 16][kN][2];
  auto clear = [&]() {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      sum[n][0] = sum[n][1] = 0.f;
    }
  };
  clear();
  const int mat = lane >> 3, mrow = lane & 7;   // ldmatrix: which of the four 8 x 8 pieces this lane addresses, and its row
  int stage = 0, q_buf = 0;
  uint32_t parity = 0;
  bool fresh = true, whole = c.tile == 0, ok = true;   // whole: the segment began in this CTA
  int64_t seg_first = first - c.tile;           // stream: its first tile among all
  // where a warp leaves its results: its own rows of the tile it has just used up, 1024 floats in each block of a panel
  auto result_of = [&](int w, int row, int col) {
    constexpr int kPer = 1024 / D;              // rows of a block
    const int piece = row / kPer, block = w * kB + piece % kB, panel = piece / kB;
    return reinterpret_cast<float*>(smem + stage * S::kStageBytes + panel * S::kPanel + block * S::kBlockBytes) + (row % kPer) * D + col;
  };
  auto meet = [&]() { named_barrier_sync(1, kWarps * 32); };

  // The warps' results of a segment (whose last stage here is `stage`): sum over them of this thread's four columns of a row.
  auto merged = [&](int item, float& mx, float& l) {
    const int row = item / (D / 4), col = item % (D / 4);
    mx = stat_m[row];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, stat_m[w * kRows + row]);
    l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = stat_m[w * kRows + row], lw = stat_l[w * kRows + row];
      const float f = mw == mx ? 1.f : exp2_fast(mw - mx);
      const float4 x =
          *reinterpret_cast<const float4*>(result_of(w, row, (((col >> 1) ^ (row >> 1 & 3)) << 3) | ((col & 1) << 2)));
      if (lw != 0.f) {    // (a warp without keys, or with keys of minus infinity only, adds nothing; one with a NaN adds that)
        l += lw * f;
        a.x += x.x * f, a.y += x.y * f, a.z += x.z * f, a.w += x.w * f;
      }
    }
    return a;
  };
  // A row's finished values: output, and the logarithm of the sum
  auto finish = [&](int b, int head, int col, float4 a, float mx, float l) {
    store4<F16>(p.out + b * p.out_batch + head * p.out_head + col * 8, a, l == 0.f ? 0.f : 1.f / l);
    if (p.lse && col == 0) p.lse[b * p.lse_batch + head] = log_sum(mx, l);
  };
  // this warp's results; groups of 8 columns in an order that keeps the banks apart
  auto deposit = [&]() {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = sum[n][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int row = 8 * n + 2 * t + e;
        if (g == 0) {
          stat_m[warp * kRows + row] = origin<F16>(m[n][e]);
          stat_l[warp * kRows + row] = x;
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          *result_of(warp, row, (((2 * i) ^ (row >> 1 & 3)) << 3) + g) = o[i][n][e];
          *result_of(warp, row, (((2 * i + 1) ^ (row >> 1 & 3)) << 3) + g) = o[i][n][2 + e];
        }
      }
  };

#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    if (ok && !mbar_wait_warp(full(stage), parity, p.timeout_ns, abort_flag)) {
      if (lane == 0) record_status(p.status, kTimeout, kSiteTile, blockIdx.x, i, 0);
      *abort_flag = 1;
      ok = false;
    }
    if (fresh && ok) {
      const uint32_t qs = q_s + q_buf * S::kQBytes;
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int kk = 0; kk < D / 16; kk += 2) {
          uint32_t r[4];
          ldsm4(r, qs + (8 * n + mrow) * S::kQPitch + ((kk * 2 + mat) << 4));
          q[kk][n][0] = r[0], q[kk][n][1] = r[1], q[kk + 1][n][0] = r[2], q[kk + 1][n][1] = r[3];
        }
    }
    fresh = false;
    const uint32_t ks = ring + stage * S::kStageBytes + warp * kB * S::kBlockBytes, vs = ks + kHalfBlock;
    uint32_t word = 0;
    if (ok) {
#pragma unroll
      for (int j = 0; j < kB; ++j) word |= masks[stage * kTB + warp * kB + j] << 16 * j;
    }
    bool cleared = false;
    if (word) {
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        const uint32_t mask = word >> 16 * j & 0xffffu;
        if (mask && mask != 0xffffu) {   // values of keys that do not count: zeros, since zero times them has to be zero
          for (int x = lane; x < S::kPanels * kBlock * 8; x += 32)
            if (!(mask >> (x / 8 % kBlock) & 1))
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs + (x / (8 * kBlock)) * S::kPanel + j * S::kBlockBytes +
                                                                           x % (8 * kBlock) * 16), "r"(0) : "memory");
          cleared = true;
        }
      }
      if (cleared) __syncwarp();
      constexpr int kChains = kB * kN == 1 ? 2 : 1;   // of additions to a score, so that products overlap
      float s[kB][kN][4];
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        float sc[kChains][kN][4];
#pragma unroll
        for (int x = 0; x < kChains; ++x)
#pragma unroll
          for (int n = 0; n < kN; ++n) sc[x][n][0] = sc[x][n][1] = sc[x][n][2] = sc[x][n][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t a[4];
          ldsm4(a, ks + (kk >> 2) * S::kPanel + j * S::kBlockBytes + ((mat & 1) * 8 + mrow) * 128 + ((((kk & 3) * 2 + (mat >> 1)) ^ mrow) << 4));
#pragma unroll
          for (int n = 0; n < kN; ++n) mma<F16>(sc[kk % kChains][n], a, q[kk][n][0], q[kk][n][1]);
        }
        const uint32_t mask = word >> 16 * j & 0xffffu;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][n][e] = sc[0][n][e] + (kChains == 2 ? sc[kChains - 1][n][e] : 0.f);
        if (mask != 0xffffu) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(mask >> (g + 8 * (e >> 1)) & 1))
#pragma unroll
              for (int n = 0; n < kN; ++n) s[j][n][e] = -INFINITY;
        }
      }
      float mx[kN][2];
      bool grows = false;
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[0][n][e], s[0][n][2 + e]);
#pragma unroll
          for (int j = 1; j < kB; ++j) x = fmaxf(x, fmaxf(s[j][n][e], s[j][n][2 + e]));
          mx[n][e] = x * p.scale_log2;
          grows |= mx[n][e] > m[n][e];
        }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = mx[n][e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float m_new = fmaxf(m[n][e], x);
            const float f = m_new == m[n][e] ? 1.f : exp2_fast(origin<F16>(m[n][e]) - origin<F16>(m_new));
            m[n][e] = m_new;
            sum[n][e] *= f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) o[d][n][e] *= f, o[d][n][2 + e] *= f;
          }
      }
      uint32_t hi[kB][kN][2], lo[kB][kN][2];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const float s0 = m[n][0] == -INFINITY ? 0.f : -origin<F16>(m[n][0]), s1 = m[n][1] == -INFINITY ? 0.f : -origin<F16>(m[n][1]);
#pragma unroll
        for (int j = 0; j < kB; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {     // keys g, g + 8
            const float w0 = exp2_fast(fmaf(s[j][n][2 * h], p.scale_log2, s0));
            const float w1 = exp2_fast(fmaf(s[j][n][2 * h + 1], p.scale_log2, s1));
            sum[n][0] += w0;
            sum[n][1] += w1;
            const uint32_t r = pack<F16>(w0, w1);
            const float2 back = unpack<F16>(r);
            hi[j][n][h] = transpose(r);
            lo[j][n][h] = transpose(pack<F16>(w0 - back.x, w1 - back.y));
          }
      }
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        if (kB > 1 && !(word >> 16 * j & 0xffffu)) continue;   // (nothing was loaded there)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t a[4];
          ldsm4_t(a, vs + (d >> 2) * S::kPanel + j * S::kBlockBytes + ((mat >> 1) * 8 + mrow) * 128 + ((((d & 3) * 2 + (mat & 1)) ^ mrow) << 4));
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            mma<F16>(o[d][n], a, hi[j][n][0], hi[j][n][1]);
            mma<F16>(o[d][n], a, lo[j][n][0], lo[j][n][1]);
          }
        }
      }
    }
    __syncwarp();        // every lane has read the tile

    const bool ends = c.tile + 1 == c.tiles, last_one = i + 1 == count;
    if (CLUSTER && last_one) break;
    if (!CLUSTER && (ends || last_one)) {
      deposit();
      meet();
      const int seg = segment_of(c), kv = p.row_tiles == 1 ? seg : seg / p.row_tiles, r0 = (seg - kv * p.row_tiles) * kRows;
      const int rows = min(kRows, p.group - r0);
      const bool direct = whole && ends;
      float* part = p.parts + ((int64_t)blockIdx.x * 2 + (whole ? 1 : 0)) * p.rows * D;
      float* ml = p.parts + (int64_t)gridDim.x * 2 * p.rows * D + ((int64_t)blockIdx.x * 2 + (whole ? 1 : 0)) * p.rows * 2;
#pragma unroll 1
      for (int item = threadIdx.x; item < rows * (D / 4); item += kWarps * 32) {
        float mx, l;
        const float4 a = merged(item, mx, l);
        const int row = item / (D / 4), col = item % (D / 4);
        if (direct) {
          finish(c.b, kv * p.group + r0 + row, col, a, mx, l);
        } else {
          *reinterpret_cast<float4*>(part + row * D + col * 4) = a;
          if (col == 0) *reinterpret_cast<float2*>(ml + row * 2) = make_float2(mx, l);
        }
      }
      if (threadIdx.x == 0 && whole) {
        // what the second kernel adds up: a segment's parts from this CTA to that of its last tile; listed by segment
        // where there are fewer of them than CTAs, else by the CTA in which it begins
        const int64_t segments = (int64_t)p.batch * p.segments_per_seq, id = (int64_t)c.b * p.segments_per_seq + seg;
        const int last = ends ? my_group : (int)(((seg_first + c.tiles) * groups - 1) / total);
        const int4 job = make_int4(my_group, last, ends ? -1 : c.b, seg);
        if (segments <= gridDim.x) p.jobs[id] = job;
        else if (!ends || last_one) p.jobs[blockIdx.x] = job;
      }
      if (threadIdx.x == 0 && !whole && last_one && p.batch * (int64_t)p.segments_per_seq > gridDim.x)
        p.jobs[blockIdx.x] = make_int4(0, 0, -1, 0);
      meet();            // the tile and the statistics are free again
      cleared = true;
      clear();
      fresh = whole = true;
      seg_first += c.tiles;
      q_buf = q_buf + 1 == S::kQBufs ? 0 : q_buf + 1;
    }
    if (cleared) {       // (written to like ordinary memory, before the next copy into it)
      fence_proxy_async_smem();
      __syncwarp();
    }
    if (lane == 0 && ok) mbar_arrive(empty(stage));   // (a warp that gave up frees none, so nothing is copied over a copy on its way)
    advance<D>(p, c);
    if (++stage == S::kStages) {
      stage = 0;
      parity ^= 1;
    }
  }

  if (CLUSTER) {
    deposit();
    meet();
    const int kv = p.row_tiles == 1 ? (int)blockIdx.y : (int)blockIdx.y / p.row_tiles, r0 = ((int)blockIdx.y - kv * p.row_tiles) * kRows;
    const int rows = min(kRows, p.group - r0);
    const int parts = gridDim.x;
    if (parts == 1) {
      for (int item = threadIdx.x; item < rows * (D / 4); item += kWarps * 32) {
        float mx, l;
        const float4 a = merged(item, mx, l);
        finish(blockIdx.z, kv * p.group + r0 + item / (D / 4), item % (D / 4), a, mx, l);
      }
      return;
    }
    // where the queries were: this CTA's part, for the others to read
    float* part = reinterpret_cast<float*>(q_mem);
    float2* ml = reinterpret_cast<float2*>(part + COLS * D);
    static_assert(COLS * D * 4 + COLS * 8 <= S::kQBufs * S::kQBytes, "the part fits");
    for (int item = threadIdx.x; item < rows * (D / 4); item += kWarps * 32) {
      float mx, l;
      const float4 a = merged(item, mx, l);
      *reinterpret_cast<float4*>(part + item * 4) = a;
      if (item % (D / 4) == 0) ml[item / (D / 4)] = make_float2(mx, l);
    }
    cluster_sync_all();
    const uint32_t part_s = smem_u32(part), ml_s = smem_u32(ml);
    for (int item = blockIdx.x * kWarps * 32 + threadIdx.x; item < rows * (D / 4); item += parts * kWarps * 32) {
      const int row = item / (D / 4);
      float mx = -INFINITY, l = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int r = 0; r < parts; ++r) {
        float mr, lr;
        float4 x;
        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(mr), "=f"(lr) : "r"(mapa_shared(ml_s + row * 8, r)) : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                     : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(mapa_shared(part_s + item * 16, r)) : "memory");
        if (lr == 0.f) continue;
        float fo, fr;
        join(mx, l, mr, lr, fo, fr);
        add(a, fo, x, fr);
      }
      finish(blockIdx.z, kv * p.group + r0 + row, item % (D / 4), a, mx, l);
    }
    cluster_sync_all();   // no CTA leaves before the others have read its part
  }
}

// Second kernel of the stream form where few segments span many CTAs each: a block adds up 32 columns of a row, 8 lanes to a
// part, so that all parts of the row are on their way at once.  (2 x 8 rows of 148 parts, a block of 16 warps to a row and a warp
// to every 16th part: 28.7 us for the whole call instead of 26.7.)
template <int D, bool F16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_long_kernel(const __grid_constant__ Params p) {
  constexpr int kTeams = kJoinThreads / 8, U = 4;
  __shared__ float4 acc[kJoinThreads / 32][8];
  __shared__ float2 stats[kJoinThreads / 32];
  grid_dependency_wait();
  grid_dependency_launch();
  const int4 job = p.jobs[blockIdx.x];
  if (job.z < 0) return;
  const int kv = job.w / p.row_tiles, r0 = (job.w - kv * p.row_tiles) * kRows, row = blockIdx.y;
  if (row >= min(kRows, p.group - r0)) return;
  const int team = threadIdx.x / 8, c = threadIdx.x % 8, col = blockIdx.z * 32 + c * 4, lane_of = job.w % p.lanes;
  const float* ml = p.parts + (int64_t)p.groups * p.lanes * 2 * p.rows * D;
  const int n = job.y - job.x + 1;
  float mx = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i0 = team; i0 < n; i0 += kTeams * U) {
    float2 s[U];
    float4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kTeams;
      s[u] = make_float2(-INFINITY, 0.f);
      if (i < n) {
        const int64_t slot = ((int64_t)((job.x + i) * p.lanes + lane_of) * 2 + (i == 0 ? 1 : 0)) * p.rows + row;
        s[u] = *reinterpret_cast<const float2*>(ml + slot * 2);
        x[u] = *reinterpret_cast<const float4*>(p.parts + slot * D + col);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s[u].y == 0.f) continue;
      float fo, fr;
      join(mx, l, s[u].x, s[u].y, fo, fr);
      add(a, fo, x[u], fr);
    }
  }
  // the four teams of a warp, then the warps, four at a time
  auto over_teams = [&]() {
#pragma unroll
    for (int o = 8; o < 32; o *= 2) {
      const float m2 = __shfl_xor_sync(0xffffffffu, mx, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
      const float4 x = make_float4(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o),
                                   __shfl_xor_sync(0xffffffffu, a.z, o), __shfl_xor_sync(0xffffffffu, a.w, o));
      if (l2 != 0.f) {
        float fo, fr;
        join(mx, l, m2, l2, fo, fr);
        add(a, fo, x, fr);
      }
    }
  };
  over_teams();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane < 8) acc[warp][lane] = a;
  if (lane == 0) stats[warp] = make_float2(mx, l);
  __syncthreads();
  if (warp != 0) return;
  mx = -INFINITY, l = 0.f;
  a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = lane / 8; w < kJoinThreads / 32; w += 4) {
    const float2 s = stats[w];
    if (s.y == 0.f) continue;
    float fo, fr;
    join(mx, l, s.x, s.y, fo, fr);
    add(a, fo, acc[w][c], fr);
  }
  over_teams();
  if (lane >= 8) return;
  const int head = kv * p.group + r0 + row;
  store4<F16>(p.out + job.z * p.out_batch + head * p.out_head + col * 2, a, l == 0.f ? 0.f : 1.f / l);
  if (p.lse && col == 0) p.lse[job.z * p.lse_batch + head] = log_sum(mx, l);
}

// The same for more segments, of fewer parts each: the parts of a segment that spans CTAs, in their order.  A warp takes 128 columns of a
// row (`rows_per` rows a block); the block's warps share out the parts of a row where there are fewer rows than warps.
template <int D, bool F16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ Params p, int rows_per) {
  constexpr int kW = kJoinThreads / 32;
  constexpr int kV = D / 128 ? D / 128 : 1;          // 16-byte pieces of a row per lane
  __shared__ float4 acc[kW][D / 4];
  __shared__ float2 stats[kW];
  grid_dependency_wait();
  grid_dependency_launch();
  const int4 job = p.jobs[blockIdx.x];
  if (job.z < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = kW / rows_per;                   // warps of a row
  const int row = blockIdx.y * rows_per + warp / share, w = warp % share;
  const int kv = job.w / p.row_tiles, r0 = (job.w - kv * p.row_tiles) * kRows;
  const bool live = row < min(kRows, p.group - r0);
  const int lane_of = job.w % p.lanes;
  const float* ml = p.parts + (int64_t)p.groups * p.lanes * 2 * p.rows * D;
  float mx = -INFINITY, l = 0.f;
  float4 a[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int n = job.y - job.x + 1;
  if (live) {
    constexpr int U = 8;
#pragma unroll 1
    for (int i0 = w; i0 < n; i0 += share * U) {
      float2 s[U];
      float4 x[U][kV];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * share;
        s[u] = make_float2(-INFINITY, 0.f);
        if (i < n) {
          const int64_t slot = ((int64_t)((job.x + i) * p.lanes + lane_of) * 2 + (i == 0 ? 1 : 0)) * p.rows + row;
          s[u] = *reinterpret_cast<const float2*>(ml + slot * 2);
#pragma unroll
          for (int v = 0; v < kV; ++v)
            if (lane + v * 32 < D / 4) x[u][v] = *reinterpret_cast<const float4*>(p.parts + slot * D + (lane + v * 32) * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s[u].y == 0.f) continue;
        float fo, fr;
        join(mx, l, s[u].x, s[u].y, fo, fr);
#pragma unroll
        for (int v = 0; v < kV; ++v) add(a[v], fo, x[u][v], fr);
      }
    }
  }
  if (share > 1) {
#pragma unroll
    for (int v = 0; v < kV; ++v)
      if (lane + v * 32 < D / 4) acc[warp][lane + v * 32] = a[v];
    if (lane == 0) stats[warp] = make_float2(mx, l);
    __syncthreads();
    if (w != 0) return;
    for (int r = 1; r < share; ++r) {
      const float2 s = stats[warp + r];
      if (s.y == 0.f) continue;
      float fo, fr;
      join(mx, l, s.x, s.y, fo, fr);
#pragma unroll
      for (int v = 0; v < kV; ++v)
        if (lane + v * 32 < D / 4) add(a[v], fo, acc[warp + r][lane + v * 32], fr);
    }
  }
  if (!live) return;
  const int head = kv * p.group + r0 + row;
  const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int v = 0; v < kV; ++v)
    if (lane + v * 32 < D / 4) store4<F16>(p.out + job.z * p.out_batch + head * p.out_head + (lane + v * 32) * 8, a[v], f);
  if (p.lse && lane == 0) p.lse[job.z * p.lse_batch + head] = log_sum(mx, l);
}

}  // namespace paged
}  // namespace iris

// ================================================================================================
// Host side
// ================================================================================================
namespace {

using namespace iris::paged;
thread_local char g_paged_err[256] = "";

int refuse(const char* what) {
  snprintf(g_paged_err, sizeof(g_paged_err), "paged attention: %s", what);
  return -1;
}

int sms_of(int device) {
  static std::atomic<int> known[64];
  if (device >= 0 && device < 64 && known[device].load(std::memory_order_relaxed)) return known[device].load(std::memory_order_relaxed);
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  if (device >= 0 && device < 64) known[device].store(sms, std::memory_order_relaxed);
  return sms;
}

// The limit of dynamic shared memory is a property of the kernel on one device.
template <class K>
cudaError_t allow_smem(K kernel, int bytes, int device, std::atomic<uint64_t>& done) {
  if (device < 64 && (done.load(std::memory_order_acquire) >> device & 1)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device < 64) done.fetch_or(1ull << device, std::memory_order_release);
  return e;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, []() {
    void* q = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) == cudaSuccess &&
        r == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(q);
    else
      (void)cudaGetLastError();
  });
  return fn;
}

// CTAs of a cluster, or 0 for the stream form, for so many segments of at most so many tiles on a GPU that holds `resident` CTAs.
// A tile takes a CTA alone 0.7 us.  The stream form shares any lengths out evenly, but begins with sums over all lengths and
// ends with a second kernel.  us, clusters of 1 / 2 / 4 / 8 and stream, 4 query heads of 128 to a key head, pages of 16:
//      8 segments   64 keys 3.7 / 4.6 / 5.0 / 5.6, 6.1    512 keys 8.6 / 6.9 / 6.1 / 6.6, 7.8    4096 keys 50 / 28 / 16 / 11.5, 9.3
//    128 segments   256 keys 6.0 / 6.2 / 11 / 24, 14      1024 keys 15.5 / 11.3 / 15.9 / 30, 18.5   4096 keys 53 / 32 / 33 / 43, 33
//    512 segments   256 keys 14.5 / 25 / 46 / 101, 18     1024 keys 33 / 39 / 61 / 119, 35          4096 keys 112 / 99 / 111 / 173, 95
//   2048 segments   64 keys 30 / 74 / 156 / 364, 20       512 keys 60 / 100 / 190 / 421, 58         1024 keys 101 / 135 / .., 103
// Over 68 such cases (heads of 64, 128 and 256, 1 to 256 sequences of up to 64 to 4096 keys) the rule is 0.6 % off the best on
// average, 9 % at worst.
int choose_cluster(int64_t segments, int64_t tiles, int resident) {
  if (segments > 4 * resident) return 0;                       // many short ones: a CTA for each costs more than it works
  if (segments > resident) return tiles <= 20 ? 1 : 0;         // more than one round of CTAs, the last of them not full
  int cluster = 1;
  while (cluster < 8 && cluster * 4 <= tiles && segments * cluster * 2 <= resident) cluster *= 2;   // two tiles each, at least
  // the chain of a CTA's tiles against the stream form's, which is longer by 4.8 tiles' time for its beginning and end; uneven
  // lengths speak for the latter, the more the longer they are
  return tiles <= 100 && (double)tiles / cluster <= 4.8 + (double)segments * tiles / resident ? cluster : 0;
}

template <int D, bool F16>
int launch_paged(Params& p, int cluster, int device, cudaStream_t stream) {
  static std::atomic<uint64_t> done[4];
  const int wide = p.group > 8;
  const auto kern = cluster ? wide ? paged_attention_kernel<D, F16, true, 16> : paged_attention_kernel<D, F16, true, 8>
                            : wide ? paged_attention_kernel<D, F16, false, 16> : paged_attention_kernel<D, F16, false, 8>;
  const int smem = wide ? Shape<D, 16>::kSmem : Shape<D, 8>::kSmem;
  cudaError_t e = allow_smem(kern, smem, device, done[wide * 2 + (cluster ? 1 : 0)]);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster ? cluster : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  const int ctas = p.groups * p.lanes;
  cfg.gridDim = cluster ? dim3(cluster, p.segments_per_seq, p.batch) : dim3(ctas);
  cfg.blockDim = dim3(Shape<D>::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kern, (const Params)p);
  if (e == cudaSuccess && !cluster) {
    const int64_t segments = (int64_t)p.batch * p.segments_per_seq;
    const int jobs = (int)(segments < ctas ? segments : ctas);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    if (jobs * 16 <= ctas) {
      cfg.gridDim = dim3(jobs, p.rows, D / 32);
      e = cudaLaunchKernelEx(&cfg, paged_join_long_kernel<D, F16>, (const Params)p);
    } else {
      // a block for every row while there are few, else several rows a block
      int per = kJoinThreads / 32;
      while (per > 1 && jobs * ((p.rows + per - 1) / per) < ctas) per /= 2;
      cfg.gridDim = dim3(jobs, (p.rows + per - 1) / per);
      e = cudaLaunchKernelEx(&cfg, paged_join_kernel<D, F16>, (const Params)p, per);
    }
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();   // reported here: it must not turn up at someone else's launch
    snprintf(g_paged_err, sizeof(g_paged_err), "paged attention: launch: %s", cudaGetErrorString(e));
    return -3;
  }
  return 0;
}

}  // namespace

extern "C" {

const char* iris_paged_attention_last_error() { return g_paged_err; }

// The arguments of a call, packed: one pointer instead of 35 arguments to convert (2 us of the host's time less).
// q [batch, heads, dim], k and v [pages, page_size, kv_heads, dim], out like q: pitches in elements, 16-byte aligned rows.
// table [batch, wide] and lens [batch]: int32.  lse [batch, heads] fp32 or null.  longest: what the lengths are expected not to
// exceed (0: the table's width); it chooses the form and nothing else.  cluster: CTAs of a cluster, 0 the stream form, -1 by rule.
struct IrisPagedAttentionArgs {
  const void *q, *k, *v, *table, *lens;
  void *out, *lse, *work, *status, *stream;
  int64_t q_batch, q_head, page_pitch, slot_pitch, head_pitch, table_pitch, out_batch, out_head, lse_batch;
  int64_t batch, heads, dim, pages, page_size, kv_heads, wide, dtype, window, sinks, longest, cluster, work_bytes, device, timeout_ns;
  double scale;
};

// Returns 0, a positive number of bytes if the form needs a workspace of that size (16-byte aligned) and got a smaller one, or
// a negative code with a message in iris_paged_attention_last_error().  The device must be the current one.
int iris_k_paged_attention(const IrisPagedAttentionArgs* args) {
  g_paged_err[0] = 0;
  const auto [q, k, v, table, lens, out, lse, work, status, stream, q_batch0, q_head0, page_pitch0, slot_pitch0, head_pitch0,
              table_pitch0, out_batch0, out_head0, lse_batch0, batch, heads, dim, pages, page_size, kv_heads, wide, dtype, window,
              sinks, longest, cluster0, work_bytes, device, timeout_ns, scale] = *args;
  int64_t q_batch = q_batch0, q_head = q_head0, page_pitch = page_pitch0, slot_pitch = slot_pitch0, head_pitch = head_pitch0;
  int64_t table_pitch = table_pitch0, out_batch = out_batch0, out_head = out_head0, lse_batch = lse_batch0, cluster = cluster0;
  if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || heads > (1 << 20)) return refuse("query heads must be a multiple of key heads");
  if (dim != 64 && dim != 128 && dim != 256) return refuse("head dimension 64, 128 or 256");
  if (dtype != 0 && dtype != 1) return refuse("dtype must be 0 (bf16) or 1 (fp16)");
  if (page_size < 1 || (page_size & (page_size - 1))) return refuse("page size must be a power of two");
  if (pages < 1 || wide < 1 || pages > 0x7fffffff || wide > 0x7fffffff || batch > 0x7fffffff || page_size > (1 << 30)) return refuse("no pages, or too many");
  if (wide * page_size > kMostKeys) return refuse("the block table is for more than 2^31 - 1024 keys of a sequence");
  const float scale_log2 = (float)(scale * 1.4426950408889634);
  if (window < 0 || sinks < 0 || !(scale_log2 > 0.f) || isinf(scale_log2)) return refuse("window and sinks must not be negative, scale above 0");
  // a pitch along one element says nothing
  if (batch == 1) q_batch = out_batch = table_pitch = lse_batch = 0;
  if (heads == 1) q_head = out_head = 0;
  if (pages == 1) page_pitch = 0;
  if (page_size == 1) slot_pitch = 0;
  if (kv_heads == 1) head_pitch = 0;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) % 16 || (q_batch | q_head | page_pitch | slot_pitch | head_pitch | out_batch | out_head) % 8)
    return refuse("rows of q, k, v and out must start on 16 bytes");
  if ((pages > 1 && page_pitch < dim) || (page_size > 1 && slot_pitch < dim) || (kv_heads > 1 && head_pitch < dim))
    return refuse("rows of the cache must not overlap");
  const uint8_t *q8 = static_cast<const uint8_t*>(q), *out8 = static_cast<const uint8_t*>(out);
  const auto past = [](int64_t a, int64_t pa, int64_t b, int64_t pb, int64_t c, int64_t pc, int64_t n) {   // bytes of a view
    return ((a - 1) * pa + (b - 1) * pb + (c - 1) * pc + n) * 2;
  };
  const int64_t q_bytes = past(batch, q_batch, heads, q_head, 1, 0, dim), out_bytes = past(batch, out_batch, heads, out_head, 1, 0, dim);
  const int64_t cache_bytes = past(pages, page_pitch, page_size, slot_pitch, kv_heads, head_pitch, dim);
  for (const void* c : {k, v})
    if (out8 < static_cast<const uint8_t*>(c) + cache_bytes && static_cast<const uint8_t*>(c) < out8 + out_bytes)
      return refuse("out must not lie in the cache");
  // out is q itself, or none of its heads meets one of q's
  if (out8 < q8 + q_bytes && q8 < out8 + out_bytes && !(out8 == q8 && out_batch == q_batch && out_head == q_head)) {
    bool apart = out_batch == q_batch && out_head == q_head;
    for (int64_t j = 1 - heads; apart && j < heads; ++j) {
      const int64_t off = (out8 - q8) / 2 + j * q_head, last = q_batch ? off / q_batch : 0;
      for (int64_t i = last - 1; i <= last + 1; ++i)
        if (i > -batch && i < batch && off - i * q_batch > -dim && off - i * q_batch < dim) apart = false;
    }
    if (!apart) return refuse("out must be q itself, or share no memory with it");
  }
  using namespace iris::overlap;
  const Rows to(out, dim * 2, {batch, out_batch * 2}, {heads, out_head * 2}), sums(lse, heads * 4, {batch, lse_batch * 4});
  const Rows from(q, dim * 2, {batch, q_batch * 2}, {heads, q_head * 2});
  const Rows keys(k, dim * 2, {pages, page_pitch * 2}, {page_size, slot_pitch * 2}, {kv_heads, head_pitch * 2});
  const Rows values(v, dim * 2, {pages, page_pitch * 2}, {page_size, slot_pitch * 2}, {kv_heads, head_pitch * 2});
  if (!apart(to) || !apart(sums)) return refuse("rows of out, or of lse, must not overlap");
  if (meet(sums, to) || meet(sums, from) || meet(sums, keys) || meet(sums, values))
    return refuse("lse must share no memory with q, out or the cache");
  const int sms = sms_of((int)device);
  if (sms < 1) return refuse("no device");
  const Rows pages_of(table, wide * 4, {batch, table_pitch * 4}), lengths(lens, batch * 4);
  if (meet(to, pages_of) || meet(to, lengths) || meet(sums, pages_of) || meet(sums, lengths))
    return refuse("out and lse must share no memory with the block table or the lengths");
  Params p;
  memset(&p, 0, sizeof(p));
  p.batch = (int)batch;
  p.group = (int)(heads / kv_heads);
  p.row_tiles = (p.group + kRows - 1) / kRows;
  p.segments_per_seq = (int)kv_heads * p.row_tiles;
  p.rows = p.group < kRows ? p.group : kRows;
  // lanes: as many of a sequence's segments side by side as leave no more than one CTA in 32 without work
  const int resident = sms * 2;
  p.lanes = 1;
  for (int n = 2; n <= p.segments_per_seq && n <= resident; ++n)
    if (p.segments_per_seq % n == 0 && resident / n * n * 32 >= resident * 31) p.lanes = n;
  p.turns = p.segments_per_seq / p.lanes;
  p.groups = resident / p.lanes;
  const int64_t segments = batch * p.segments_per_seq;
  if (cluster < 0) {
    int64_t most = wide * (int64_t)page_size;
    if (longest > 0 && longest < most) most = longest;
    if (window > 0 && window < most && sinks < most - window) most = window + sinks;
    const int64_t tile = dim == 64 ? Shape<64>::kTile : dim == 128 ? Shape<128>::kTile : Shape<256>::kTile;
    const int64_t tiles = (most + tile - 1) / tile;
    cluster = choose_cluster(segments, tiles, resident);
  }
  if (batch > 65535 || p.segments_per_seq > 65535) cluster = 0;
  if (cluster == 0) {
    const int64_t ctas = (int64_t)p.groups * p.lanes, need = ctas * (16 + 2 * p.rows * (dim + 2) * 4);
    if (!work || work_bytes < need) return (int)need;
    p.jobs = static_cast<int4*>(work);
    p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(work) + ctas * 16);
  } else {
    p.lanes = p.turns = 1;   // (a CTA's lane is its block's y)
  }
  if (cluster != 0 && cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8) {
    return refuse("a cluster has 1, 2, 4 or 8 CTAs");
  }
  p.q = static_cast<const uint8_t*>(q);
  p.table = static_cast<const int*>(table);
  p.lens = static_cast<const int*>(lens);
  p.out = static_cast<uint8_t*>(out);
  p.lse = static_cast<float*>(lse);
  p.status = static_cast<iris::StatusBlock*>(status);
  p.q_batch = q_batch * 2, p.q_head = q_head * 2;
  const EncodeTiledFn encode = encode_fn();
  if (!encode) return refuse("cuTensorMapEncodeTiled is not available");
  {
    // (a pitch along one element has to be a legal one all the same)
    const auto pitch = [row = dim * 2](int64_t x) { return (cuuint64_t)(x ? x * 2 : row); };
    const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)kv_heads, (cuuint64_t)page_size, (cuuint64_t)pages};
    const cuuint64_t strides[3] = {pitch(head_pitch), pitch(slot_pitch), pitch(page_pitch)};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)(page_size < kBlock ? page_size : kBlock), 1}, ones[4] = {1, 1, 1, 1};
    const auto type = dtype ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = 0; i < 2; ++i) {
      const CUresult r = encode(i ? &p.v : &p.k, type, 4, const_cast<void*>(i ? v : k), dims, strides, box, ones,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                dim == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
      if (r != CUDA_SUCCESS) {
        snprintf(g_paged_err, sizeof(g_paged_err), "paged attention: cuTensorMapEncodeTiled failed with %d", (int)r);
        return -2;
      }
    }
  }
  p.timeout_ns = timeout_ns > 0 ? (uint64_t)timeout_ns : 2000000000ull;
  p.table_pitch = table_pitch;
  p.out_batch = out_batch * 2, p.out_head = out_head * 2;
  p.lse_batch = lse_batch;
  p.pages = (int)pages;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.wide = (int)wide;
  p.window = window < 0x7fffffff ? (int)window : 0x7fffffff;
  p.sinks = sinks < 0x7fffffff ? (int)sinks : 0x7fffffff;
  p.scale_log2 = scale_log2;
  const auto st = static_cast<cudaStream_t>(stream);
  if (dim == 64) return dtype ? launch_paged<64, true>(p, (int)cluster, (int)device, st) : launch_paged<64, false>(p, (int)cluster, (int)device, st);
  if (dim == 128) return dtype ? launch_paged<128, true>(p, (int)cluster, (int)device, st) : launch_paged<128, false>(p, (int)cluster, (int)device, st);
  return dtype ? launch_paged<256, true>(p, (int)cluster, (int)device, st) : launch_paged<256, false>(p, (int)cluster, (int)device, st);
}

}  // extern "C"
