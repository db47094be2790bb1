// paged_cache.cu — pages of a paged key-value cache handed out and taken back on the GPU, from the requests' lengths.
//
// reserve: request b holds lens[b] tokens in ceil(lens[b] / page_size) pages and gets new_lens[b] more.  In the requests' order
// each takes the pages it lacks from the end of the list of free pages,
//
//   need_b = ceil((lens[b] + new_lens[b]) / page_size) - ceil(lens[b] / page_size),   first_b = need_0 + .. + need_{b-1}
//   block_table[b, held_b + i] = free[count - 1 - (first_b + i)],   0 <= i < need_b
//
// as long as they last: a request with first_b + need_b > count, too long for its row of the table or for the caller's limit, with
// more tokens than rows were left for them, or that holds tokens although only empty ones are asked for, gets nothing.  Every new
// token gets its position and its slot, page * page_size + position % page_size.  release: pages of chosen requests go back to the
// end of the list, in their order; negative entries of a row are passed over.  No counterpart in the reference.
//
// A call's time is its launch and a few passes through memory in a row (lengths, prefix sums, free list or table, output), so
// it is one launch: every CTA of one cluster makes the prefix sums for itself, in chunks of a few requests per thread, and the
// tokens and pages of a chunk are shared out over the cluster's threads, whatever their lengths, by a search in the chunk's sums.
// What may be updated in place (lengths, count) is written after a barrier of the cluster, when every CTA has read it.
// All sums are whole numbers in 64 bits.
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>

#include "iris/overlap.cuh"
#include "iris/ptx_sm100.cuh"

namespace iris {
namespace pages {

using namespace iris::ptx;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

struct Params {
  const int* lens;
  const int* more;           // reserve: new tokens per request; release: not 0 for the requests to end
  int* table;
  int* free;
  const int* count;
  int* slots;
  int* positions;
  int* lens_out;
  int* count_out;
  int64_t table_pitch, tokens, row_stride;
  int64_t most;              // tokens of a request
  int batch, wide, page_shift, capacity;
  int most_held;             // that a request may hold already
};

// A chunk of requests, PER a thread, and the sums over them, for every thread to search.  One a thread up to 512 requests, else
// four (1574 requests of up to 41 tokens: 26.7 us with one, 12.1 with four; 512 of one token: 4.1 and 5.4).
template <int PER>
struct Chunk {
  static constexpr int kChunk = kThreads * PER;
  int64_t pages_upto[kChunk];      // of pages, this request's included
  int64_t tokens_upto[kChunk];
  int len[kChunk];                 // ~ length: no pages for it
  int64_t warp_sum[2][kWarps];
};

// The same for requests that end.
template <int PER>
struct Leaving {
  static constexpr int kChunk = kThreads * PER;
  int64_t entries_upto[kChunk];    // of their rows
  int64_t pages_upto[kChunk];      // of these, the pages
  int found[kChunk];               // pages in this CTA's share of the entries
  bool leaves[kChunk];
  int in_warp[2][kWarps];
  int64_t warp_sum[2][kWarps];
};
template <int PER>
__device__ __forceinline__ int found_by(const Leaving<PER>& c, int i, int cta) {
  int n;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(n) : "r"(mapa_shared(smem_u32(&c.found[i]), cta)) : "memory");
  return n;
}

// Sums of the threads before this one and this one's own.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t* warp_sum, int64_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sum[warp] = x;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) x += warp_sum[w];
    all += warp_sum[w];
  }
  return x;
}

// The first request of the chunk with more than `at` before or in it.
template <int N>
__device__ __forceinline__ int search(const int64_t* upto, int64_t at) {
  int lo = 0;
#pragma unroll
  for (int step = N / 2; step > 0; step >>= 1)
    if (upto[lo + step - 1] <= at) lo += step;
  return lo;
}

// Gives the pages of the requests that are asked for back to the list.  Negative entries of their rows are no pages (a program may
// take pages out of a row itself, those that a window has left behind for instance): they are passed over.  So each CTA of the cluster
// first counts the pages in its share of a chunk's entries, the CTAs put their counts together, and then each moves the entries of
// its share, their places counted on from there.
// (Cold caches, without the count and with it: 8 requests of 256 pages 8 and 11 us, 512 of 32 11 and 12, 512 of 256 32 and 41.)
template <int PER>
__device__ __forceinline__ void release(const Params& p, Leaving<PER>& c) {
  constexpr int kPer = PER, kChunk = Leaving<PER>::kChunk, U = 4;   // U: loads under way at once
  const int mask = (1 << p.page_shift) - 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x, ctas = gridDim.x;
  const int count = min(max(*p.count, 0), p.capacity);
  int64_t pages = 0;               // of the chunks before, also of requests that the list had no room for
  int64_t used = 0;                // taken back so far
  const auto entry_of = [&](int base, int r, int64_t k) {
    return p.table + (base + r) * p.table_pitch + (k - (r ? c.entries_upto[r - 1] : 0));
  };
  for (int base = 0; base < p.batch; base += kChunk) {
    int64_t need[kPer], sum = 0, entries, all;
    bool asked[kPer];
    __syncthreads();               // the chunk before has been used
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = threadIdx.x * kPer + u, b = base + i;
      asked[u] = b < p.batch && p.more[b] != 0;
      need[u] = asked[u] ? min((max((int64_t)p.lens[b], (int64_t)0) + mask) >> p.page_shift, (int64_t)p.wide) : 0;
      sum += need[u];
      c.found[i] = 0;
    }
    int64_t upto = scan(sum, c.warp_sum[0], entries) - sum;
#pragma unroll
    for (int u = 0; u < kPer; ++u) c.entries_upto[threadIdx.x * kPer + u] = upto += need[u];
    __syncthreads();
    const int64_t from = entries * rank / ctas, to = entries * (rank + 1) / ctas;
    // U tiles of entries at once, from k0 on: their requests, places and contents
    int request[U], page[U];
    int* entry[U];
    auto look = [&](int64_t k0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t k = k0 + u * kThreads + threadIdx.x;
        request[u] = search<kChunk>(c.entries_upto, min(k, to - 1));
        entry[u] = k < to ? entry_of(base, request[u], k) : nullptr;
        page[u] = entry[u] ? *entry[u] : -1;
      }
    };
    for (int64_t k0 = from; k0 < to; k0 += kThreads * U) {
      look(k0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t there = __ballot_sync(0xffffffffu, page[u] >= 0);
        const int r = __shfl_sync(0xffffffffu, request[u], 0);
        if (__all_sync(0xffffffffu, request[u] == r)) {
          if (lane == 0 && there) atomicAdd(&c.found[r], __popc(there));
        } else if (page[u] >= 0) {
          atomicAdd(&c.found[request[u]], 1);
        }
      }
    }
    __syncthreads();
    cluster_sync_all();            // every CTA has counted its share, and read the lengths
    sum = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      need[u] = 0;
      for (int x = 0; x < ctas; ++x) need[u] += found_by(c, threadIdx.x * kPer + u, x);
      sum += need[u];
    }
    upto = scan(sum, c.warp_sum[1], all) - sum;
    const int64_t room = p.capacity - count - pages;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = threadIdx.x * kPer + u;
      c.pages_upto[i] = upto += need[u];
      asked[u] = asked[u] && (need[u] == 0 || upto <= room);
      c.leaves[i] = asked[u];
    }
    __syncthreads();
    // requests whose pages go back come before those that found no room, so pages before a request have all gone back
    if (all == entries) {          // all entries are pages, each has its place
      for (int64_t k0 = from; k0 < to; k0 += kThreads * U) {
        if (to - from > kThreads * U) look(k0);                     // (else they are still there)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (entry[u] && c.leaves[request[u]]) p.free[count + pages + k0 + u * kThreads + threadIdx.x] = page[u], *entry[u] = -1;
      }
    } else if (from < to) {
      const int r0 = search<kChunk>(c.entries_upto, from);
      int64_t at = count + pages + (r0 ? c.pages_upto[r0 - 1] : 0);
      for (int x = 0; x < rank; ++x) at += found_by(c, r0, x);
      int turn = 0;
      for (int64_t k0 = from; k0 < to; k0 += kThreads, turn ^= 1) {
        const int64_t k = k0 + threadIdx.x;
        const int r = search<kChunk>(c.entries_upto, min(k, to - 1));
        const bool leaves = k < to && c.leaves[r];
        int* at_entry = leaves ? entry_of(base, r, k) : nullptr;
        const int got = leaves ? *at_entry : -1;
        const uint32_t there = __ballot_sync(0xffffffffu, got >= 0);
        if (lane == 0) c.in_warp[turn][warp] = __popc(there);
        __syncthreads();
        int before = __popc(there & ((1u << lane) - 1)), tile = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) before += c.in_warp[turn][w];
          tile += c.in_warp[turn][w];
        }
        if (got >= 0) p.free[at + before] = got;
        if (leaves) *at_entry = -1;
        at += tile;
      }
    }
    if (room > 0) {
      const int i = all <= room ? kChunk : search<kChunk>(c.pages_upto, room);   // the first that found no room
      used += i ? c.pages_upto[i - 1] : 0;
    }
    pages += all;
    __syncthreads();
    cluster_sync_all();            // every CTA has read the others' counts
#pragma unroll
    for (int u = 0; u < kPer; ++u)
      if (rank == 0 && asked[u]) p.lens_out[base + threadIdx.x * kPer + u] = 0;
  }
  if (rank == 0 && threadIdx.x == 0) *p.count_out = (int)(count + used);
}

// Pages, slots and positions for new tokens (at the top of the file).
template <int PER>
__device__ __forceinline__ void reserve(const Params& p, Chunk<PER>& c) {
  constexpr int kPer = PER, kChunk = Chunk<PER>::kChunk;
  const int mask = (1 << p.page_shift) - 1;
  const int rank = blockIdx.x, ctas = gridDim.x;
  const int64_t at0 = (int64_t)rank * kThreads + threadIdx.x, step = (int64_t)ctas * kThreads;
  const int count = min(max(*p.count, 0), p.capacity);
  int64_t pages = 0, tokens = 0;   // of the chunks before
  int64_t used = 0;                // pages handed out so far

  // This thread's requests of a chunk, base + threadIdx.x * kPer on: granted or not, and the chunk's sums in shared memory.
  int len[kPer], more[kPer];
  bool granted[kPer];
  auto held_of = [&](int n) { return (int)(((int64_t)n + mask) >> p.page_shift); };
  auto take_in = [&](int base, int64_t& all_pages, int64_t& all_tokens) {
    int64_t need[kPer], t_upto[kPer], sum = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int b = base + threadIdx.x * kPer + u;
      len[u] = more[u] = 0;
      if (b < p.batch) {
        len[u] = max(p.lens[b], 0);
        more[u] = max(p.more[b], 0);
      }
    }
    __syncthreads();               // the chunk before has been used
#pragma unroll
    for (int u = 0; u < kPer; ++u) t_upto[u] = sum += more[u];
    const int64_t before = scan(sum, c.warp_sum[1], all_tokens) - sum;
#pragma unroll
    for (int u = 0; u < kPer; ++u) t_upto[u] += before;
    sum = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int b = base + threadIdx.x * kPer + u;
      need[u] = 0;
      granted[u] = b < p.batch;
      const int64_t end = (int64_t)len[u] + more[u];
      granted[u] = granted[u] && end <= p.most && (len[u] <= p.most_held || more[u] == 0) &&
                   (p.row_stride ? more[u] <= p.row_stride : tokens + t_upto[u] <= p.tokens);
      if (granted[u]) need[u] = ((end + mask) >> p.page_shift) - held_of(len[u]);
      sum += need[u];
    }
    int64_t upto = scan(sum, c.warp_sum[0], all_pages) - sum;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int i = threadIdx.x * kPer + u;
      upto += need[u];
      granted[u] = granted[u] && (need[u] == 0 || pages + upto <= count);
      c.pages_upto[i] = upto;
      c.tokens_upto[i] = t_upto[u];
      c.len[i] = granted[u] ? len[u] : ~len[u];
    }
    // requests that got pages come before those that did not, so the last of them has the sum
    __syncthreads();
  };
  auto last_granted = [&](int64_t all) {   // pages of the chunk that were handed out
    if (all == 0) return (int64_t)0;
    const int64_t room = count - pages;
    if (all <= room) return all;
    // the largest sum within the room
    if (room <= 0) return (int64_t)0;
    const int i = search<kChunk>(c.pages_upto, room);
    return i > 0 ? c.pages_upto[i - 1] : (int64_t)0;
  };

  for (int base = 0; base < p.batch; base += kChunk) {
    int64_t all_pages = 0, all_tokens = 0;
    take_in(base, all_pages, all_tokens);
    const int64_t got = last_granted(all_pages);
    used += got;
    for (int64_t k = at0; k < got; k += step) {
      const int r = search<kChunk>(c.pages_upto, k);
      const int64_t i = k - (r ? c.pages_upto[r - 1] : 0);
      p.table[(base + r) * p.table_pitch + held_of(c.len[r]) + i] = p.free[count - 1 - (pages + k)];
    }
    // token rows of this chunk's requests: packed one request behind the other, or row_stride rows to a request
    const int n = min(kChunk, p.batch - base);
    const int64_t row0 = p.row_stride ? base * p.row_stride : tokens;
    const int64_t row1 = min(p.tokens, p.row_stride ? (base + n) * p.row_stride : tokens + all_tokens);
    // Many rows: four in a row to a thread, one search, and a page looked up once for the rows that lie in it (32 prompts,
    // 65536 rows: 9.3 -> 7.8 us).  Few: one to a thread (512 requests of one token: 4.1 us, 5.5 with four).
    const int width = row1 - row0 > 2 * step ? 4 : 1;
    for (int64_t at = row0 + width * at0; at < row1; at += width * step) {
      int r;
      int64_t j;
      if (p.row_stride) {
        r = (int)((at - row0) / p.row_stride);
        j = at - row0 - r * p.row_stride;
      } else {
        r = search<kChunk>(c.tokens_upto, at - row0);
        j = at - row0 - (r ? c.tokens_upto[r - 1] : 0);
      }
      int slot[4], position[4], known = -1, page = -1;
      int64_t more_here = c.tokens_upto[r] - (r ? c.tokens_upto[r - 1] : 0);
      const int n4 = (int)min((int64_t)width, row1 - at);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        slot[u] = position[u] = -1;
        if (u >= n4) break;
        while (p.row_stride ? j >= p.row_stride : j >= more_here) {   // on to the next request (that has a token)
          ++r;
          j = 0;
          known = -1;
          more_here = c.tokens_upto[r] - c.tokens_upto[r - 1];
        }
        if (c.len[r] >= 0 && j < more_here) {
          const int pos = (int)(c.len[r] + j), i = pos >> p.page_shift, fresh = i - held_of(c.len[r]);
          if (i != known) {
            known = i;
            page = fresh < 0 ? p.table[(base + r) * p.table_pitch + i]
                             : p.free[count - 1 - (pages + (r ? c.pages_upto[r - 1] : 0) + fresh)];
          }
          const int64_t s = ((int64_t)page << p.page_shift) + (pos & mask);
          position[u] = pos;
          slot[u] = page < 0 || s > 0x7fffffff ? -1 : (int)s;   // an entry that is no page: as a token that is not kept
        }
        ++j;
      }
      if (n4 == 4 && !((reinterpret_cast<uintptr_t>(p.slots + at) | reinterpret_cast<uintptr_t>(p.positions + at)) & 15)) {
        *reinterpret_cast<int4*>(p.slots + at) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        *reinterpret_cast<int4*>(p.positions + at) = make_int4(position[0], position[1], position[2], position[3]);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (u < n4) p.slots[at + u] = slot[u], p.positions[at + u] = position[u];
      }
    }
    pages += all_pages;
    tokens += all_tokens;
  }
  const int64_t end = p.row_stride ? p.batch * p.row_stride : tokens;
  for (int64_t row = end + at0; row < p.tokens; row += step) p.slots[row] = p.positions[row] = -1;
  cluster_sync_all();   // every CTA has read the lengths and the count
  if (rank != 0) return;
  for (int base = 0; base < p.batch; base += kChunk) {
    if (p.batch > kChunk) {   // (the only chunk is still there)
      if (base == 0) pages = tokens = 0;
      int64_t all_pages = 0, all_tokens = 0;
      take_in(base, all_pages, all_tokens);
      pages += all_pages;
      tokens += all_tokens;
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int b = base + threadIdx.x * kPer + u;
      if (b < p.batch) p.lens_out[b] = !granted[u] ? p.lens[b] : len[u] + more[u];
    }
  }
  if (threadIdx.x == 0) *p.count_out = (int)(count - used);
}

template <bool RELEASE, int PER>
__global__ void __launch_bounds__(kThreads) pages_kernel(const __grid_constant__ Params p) {
  __shared__ std::conditional_t<RELEASE, Leaving<PER>, Chunk<PER>> c;
  grid_dependency_wait();
  grid_dependency_launch();
  if constexpr (RELEASE) release<PER>(p, c);
  else reserve<PER>(p, c);
}

thread_local char g_err[256] = "";

int refuse(const char* what) {
  snprintf(g_err, sizeof(g_err), "%s", what);
  return -1;
}

// An array of a call; in_place: where else it may lie.
struct Array {
  iris::overlap::Rows rows;
  bool written;
  uintptr_t in_place[2];
};
Array ints(const void* at, int64_t n, bool written = false, const void* in_place = nullptr, const void* or_in_place = nullptr) {
  return {{at, n * 4}, written, {reinterpret_cast<uintptr_t>(in_place), reinterpret_cast<uintptr_t>(or_in_place)}};
}
Array rows_of(const void* table, int64_t batch, int64_t wide, int64_t pitch) {
  return {{table, wide * 4, {batch, pitch * 4}}, true, {0, 0}};
}
// Whether what is written shares memory with anything else, but for what may be updated in place.
template <int N>
bool share_memory(const Array (&arrays)[N]) {
  for (int i = 0; i < N; ++i)
    for (int j = 0; j < i; ++j) {
      const Array &a = arrays[i], &b = arrays[j];
      if (!a.written && !b.written) continue;
      if (meet(a.rows, b.rows) && !(a.rows.at == b.rows.at && a.rows.end == b.rows.end &&
                                    (a.in_place[0] == b.rows.at || a.in_place[1] == b.rows.at)))
        return true;
    }
  return false;
}

template <bool RELEASE>
int launch(const Params& p, int64_t items, void* stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  // as many CTAs as have something to write, up to a cluster of eight
  int ctas = 1;
  while (ctas < 8 && items > (int64_t)ctas * kThreads) ctas *= 2;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = p.batch <= kThreads ? cudaLaunchKernelEx(&cfg, pages_kernel<RELEASE, 1>, p)
                                            : cudaLaunchKernelEx(&cfg, pages_kernel<RELEASE, 4>, p);
  if (e == cudaSuccess) return 0;
  (void)cudaGetLastError();   // reported here: it must not turn up at someone else's launch
  snprintf(g_err, sizeof(g_err), "launch: %s", cudaGetErrorString(e));
  return -3;
}

}  // namespace pages
}  // namespace iris

extern "C" {

const char* iris_pages_last_error() { return iris::pages::g_err; }

// The arguments of a call, packed (see paged_attention.cu).  All arrays int32 on the current device.  table [batch, wide] with
// rows table_pitch apart; free [capacity], count [1].  slots, positions [tokens]: row_stride rows to a request, or, with
// row_stride 0, packed; rows of no token get -1.  lens_out and count_out may be lens and count.
struct IrisReserveArgs {
  const void *lens, *new_lens;
  void *table, *free;
  const void *count;
  void *slots, *positions, *lens_out, *count_out, *stream;
  int64_t table_pitch, wide, capacity, page_size, batch, tokens, row_stride;
};

static int reserve(const IrisReserveArgs* args, int64_t max_len, bool fresh) {
  using namespace iris::pages;
  g_err[0] = 0;
  const auto [lens, new_lens, table, free, count, slots, positions, lens_out, count_out, stream, table_pitch, wide, capacity,
              page_size, batch, tokens, row_stride] = *args;
  if (page_size < 1 || (page_size & (page_size - 1)) || page_size > (1 << 30)) return refuse("page size must be a power of two");
  if (batch < 1 || batch > 0x7fffffff - 4 * kThreads || wide < 1 || wide > 0x7fffffff || capacity < 0 || capacity > 0x7fffffff || tokens < 0 || row_stride < 0)
    return refuse("sizes out of range");
  const Array arrays[] = {ints(lens, batch), ints(new_lens, batch), ints(free, capacity), ints(count, 1), rows_of(table, batch, wide, table_pitch),
                          ints(slots, tokens, true), ints(positions, tokens, true), ints(lens_out, batch, true, lens, new_lens),
                          ints(count_out, 1, true, count)};
  if (share_memory(arrays)) return refuse("arrays that are written must not share memory with others");
  Params p;
  memset(&p, 0, sizeof(p));
  p.lens = static_cast<const int*>(lens);
  p.more = static_cast<const int*>(new_lens);
  p.table = static_cast<int*>(table);
  p.free = static_cast<int*>(free);
  p.count = static_cast<const int*>(count);
  p.slots = static_cast<int*>(slots);
  p.positions = static_cast<int*>(positions);
  p.lens_out = static_cast<int*>(lens_out);
  p.count_out = static_cast<int*>(count_out);
  p.table_pitch = table_pitch, p.tokens = tokens, p.row_stride = row_stride;
  p.batch = (int)batch, p.wide = (int)wide, p.capacity = (int)capacity;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.most = wide << p.page_shift < 0x7fffffff ? wide << p.page_shift : 0x7fffffff;
  if (max_len < p.most) p.most = max_len;
  p.most_held = fresh ? 0 : 0x7fffffff;
  return launch<false>(p, tokens, stream);
}

int iris_k_reserve_slots(const IrisReserveArgs* args) { return reserve(args, INT64_MAX, false); }

// The same with a limit to the tokens of a request, below what its row of the table has room for; fresh: not 0 for requests that
// hold nothing alone.
struct IrisReserveWithinArgs {
  IrisReserveArgs all;
  int64_t max_len, fresh;
};
int iris_k_reserve_slots_within(const IrisReserveWithinArgs* args) { return reserve(&args->all, args->max_len, args->fresh != 0); }

// which [batch]: not 0 for the requests whose pages go back; their length becomes 0 and their entries of the table -1.
int iris_k_release_slots(void* lens, const void* which, void* table, int64_t table_pitch, int64_t wide, void* free,
                         int64_t capacity, void* count, int page_size, int64_t batch, void* stream) {
  using namespace iris::pages;
  g_err[0] = 0;
  if (page_size < 1 || (page_size & (page_size - 1))) return refuse("page size must be a power of two");
  if (batch < 1 || batch > 0x7fffffff - 4 * kThreads || wide < 1 || wide > 0x7fffffff || capacity < 0 || capacity > 0x7fffffff)
    return refuse("sizes out of range");
  const Array arrays[] = {ints(which, batch), ints(lens, batch, true, which), ints(free, capacity, true), ints(count, 1, true),
                          rows_of(table, batch, wide, table_pitch)};
  if (share_memory(arrays)) return refuse("arrays that are written must not share memory with others");
  Params p;
  memset(&p, 0, sizeof(p));
  p.lens = static_cast<const int*>(lens);
  p.more = static_cast<const int*>(which);
  p.table = static_cast<int*>(table);
  p.free = static_cast<int*>(free);
  p.count = static_cast<const int*>(count);
  p.lens_out = static_cast<int*>(lens);
  p.count_out = static_cast<int*>(count);
  p.table_pitch = table_pitch;
  p.batch = (int)batch, p.wide = (int)wide, p.capacity = (int)capacity;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  return launch<true>(p, batch * wide, stream);
}

}  // extern "C"
