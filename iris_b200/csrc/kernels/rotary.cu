// rotary.cu — what lies between the projection of queries, keys and values and the attention, in one pass over its output:
// a norm of every query and key head, the rotation by the token's position, and the keys' and values' way into a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                      (per head of q and k, w per component; or y = x)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)    for each pair (a, b) of the first `rotary` components, with the
//                                                           angle of the token's position and the pair
//   cache[slot] = rotated k, v
//
// Pairs are (i, i + rotary / 2) or, interleaved, (2 i, 2 i + 1).  cos and sin come from a table in fp32 (a row per position:
// rotary / 2 cosines, then the sines), so that far positions lose nothing; arithmetic is fp32 with one rounding at the end.
// No counterpart in the reference.
//
// HBM bounds it: every element is read once and written once (keys and values twice, with a cache).  A lane takes 16 components
// of a head, the two 8-component pieces whose components are each other's partners, so that neither rotation nor norm needs more
// than the registers and a few shuffles; the lanes of a token keep their cosines and sines and take several of its heads, whose
// loads are all under way before the first is used.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "iris/iris.cuh"
#include "iris/overlap.cuh"
#include "iris/ptx_sm100.cuh"

namespace iris {
namespace rotary {

using namespace iris::ptx;

constexpr int kThreads = 256;
constexpr uint32_t kSitePosition = 96, kSiteSlot = 97;

struct Params {
  const uint8_t* qkv;        // pitches in bytes
  uint8_t* out;
  const int* positions;
  const float* table;
  const uint8_t* q_weight;   // null: no norm
  const uint8_t* k_weight;
  uint8_t* k_cache;          // null: no cache
  uint8_t* v_cache;
  const int* slots;
  StatusBlock* status;
  int64_t tokens, ld_in, ld_out, ld_table, page_pitch, slot_pitch, head_pitch, cache_slots;
  int positions_in_table, heads, kv_heads, dim, half, page_shift;
  int token_shift;           // log2 of the tokens of a block
  int out_heads;             // heads written to out: all, those of q and k (in place), or those of q
  float eps;
};

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
template <bool F16>
__device__ __forceinline__ float2 unpack(uint32_t v) {
  return F16 ? __half22float2(*reinterpret_cast<const __half2*>(&v)) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack(float2 f) {
  if (F16) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (a, b) turned by the angles whose cosines and sines are c and s.
__device__ __forceinline__ void turn(float2& a, float2& b, float2 c, float2 s) {
  const float2 x = fma2(mul2(b, s), make_float2(-1.f, -1.f), mul2(a, c));
  b = fma2(a, s, mul2(b, c));
  a = x;
}

// LANES: lanes of a head, the power of two from dim / 16 on.  HEADS: heads of a lane.  A block has `spread` groups of lanes to a
// token; block (x, y): tokens x * (groups / spread) on, heads y * spread * HEADS on.  (64 registers, four blocks to an SM, although
// that spills a little: 16384 tokens of 96 heads of 128, 181 us with 78 registers, 173 with 64; two heads to a lane 195.  fp32
// arithmetic two operations to an instruction: 177 -> 172 us there, 89 -> 86 with 48 heads.)
template <int LANES, bool F16, bool INTERLEAVED, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS == 1 ? 5 : 4) qk_norm_rope_kernel(const __grid_constant__ Params p) {
  constexpr int kGroups = kThreads / LANES, kHeads = HEADS;
  grid_dependency_wait();
  grid_dependency_launch();
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int spread = kGroups >> p.token_shift;
  const int64_t token = ((int64_t)blockIdx.x << p.token_shift) + group / spread;
  if (token >= p.tokens) return;
  const int head0 = blockIdx.y * spread * kHeads + group % spread;
  const int all = p.heads + 2 * p.kv_heads;
  const bool live = lane * 16 < p.dim;                   // (a dimension that is no power of two)
  const bool turns = lane * 8 < p.half;
  // this lane's two pieces: partners of one another where it turns them, neighbours elsewhere
  const int c0 = turns && !INTERLEAVED ? lane * 8 : lane * 16;
  const int c1 = turns && !INTERLEAVED ? c0 + p.half : c0 + 8;

  uint4 x[kHeads][2];
  const uint8_t* src = p.qkv + token * p.ld_in;
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int h = head0 + u * spread;
    if (live && h < all) {
      x[u][0] = *reinterpret_cast<const uint4*>(src + (h * p.dim + c0) * 2);
      x[u][1] = *reinterpret_cast<const uint4*>(src + (h * p.dim + c1) * 2);
    }
  }
  const int pos = p.positions[token];
  const int slot = p.k_cache ? p.slots[token] : -1;
  if (pos < 0) return;                                    // a row of no token
  if (pos >= p.positions_in_table) {
    if (head0 == 0 && lane == 0) record_status(p.status, kBadPointer, kSitePosition, 0, (uint32_t)token, (uint64_t)pos);
    return;
  }
  if (slot >= p.cache_slots && head0 == 0 && lane == 0) record_status(p.status, kBadPointer, kSiteSlot, 0, (uint32_t)token, (uint64_t)slot);
  const bool keep = slot >= 0 && slot < p.cache_slots;
  const int64_t cached = keep ? (slot >> p.page_shift) * p.page_pitch + (slot & ((1 << p.page_shift) - 1)) * p.slot_pitch : 0;

  float2 cs[4], sn[4];
  if (turns) {
    const float* row = p.table + pos * p.ld_table + lane * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = *reinterpret_cast<const float4*>(row + 4 * i), s = *reinterpret_cast<const float4*>(row + p.half + 4 * i);
      cs[2 * i] = make_float2(c.x, c.y), cs[2 * i + 1] = make_float2(c.z, c.w);
      sn[2 * i] = make_float2(s.x, s.y), sn[2 * i + 1] = make_float2(s.z, s.w);
    }
  }
  uint8_t* dst = p.out + token * p.ld_out;
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int h = head0 + u * spread;
    if (h >= all) break;                                  // (the same for all lanes of a head)
    if (h < p.heads + p.kv_heads) {
      float2 y[2][4];                                     // the two pieces
      if (live) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[u][i]);
#pragma unroll
          for (int k = 0; k < 4; ++k) y[i][k] = unpack<F16>(w[k]);
        }
      }
      const uint8_t* weight = h < p.heads ? p.q_weight : p.k_weight;
      if (weight) {
        float2 ss = make_float2(0.f, 0.f);
        if (live) {
#pragma unroll
          for (int k = 0; k < 4; ++k) ss = fma2(y[0][k], y[0][k], fma2(y[1][k], y[1][k], ss));
        }
        float sum = ss.x + ss.y;
        // (the groups of a warp may have left the loop at different heads)
        const uint32_t lanes = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << (threadIdx.x & 31 & ~(LANES - 1));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(lanes, sum, o);
        const float scale = rsqrtf(sum / (float)p.dim + p.eps);
        if (live) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(weight + (i ? c1 : c0) * 2);
            const uint32_t* v = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
            for (int k = 0; k < 4; ++k) y[i][k] = mul2(y[i][k], mul2(unpack<F16>(v[k]), make_float2(scale, scale)));
          }
        }
      }
      if (turns) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (INTERLEAVED) {     // pairs 2 k and 2 k + 1 of the lane's eight: two neighbouring words of a piece
            float2 &f = y[k >> 1][2 * (k & 1)], &g = y[k >> 1][2 * (k & 1) + 1];
            float2 e = make_float2(f.x, g.x), d = make_float2(f.y, g.y);
            turn(e, d, cs[k], sn[k]);
            f = make_float2(e.x, d.x), g = make_float2(e.y, d.y);
          } else {
            turn(y[0][k], y[1][k], cs[k], sn[k]);
          }
        }
      }
      if (live) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          x[u][i] = make_uint4(pack<F16>(y[i][0]), pack<F16>(y[i][1]), pack<F16>(y[i][2]), pack<F16>(y[i][3]));
      }
    }
    if (!live) continue;
    if (h < p.out_heads) {
      *reinterpret_cast<uint4*>(dst + (h * p.dim + c0) * 2) = x[u][0];
      *reinterpret_cast<uint4*>(dst + (h * p.dim + c1) * 2) = x[u][1];
    }
    if (keep && h >= p.heads) {
      const bool key = h < p.heads + p.kv_heads;
      uint8_t* to = (key ? p.k_cache : p.v_cache) + cached + (h - p.heads - (key ? 0 : p.kv_heads)) * p.head_pitch;
      *reinterpret_cast<uint4*>(to + c0 * 2) = x[u][0];
      *reinterpret_cast<uint4*>(to + c1 * 2) = x[u][1];
    }
  }
}

thread_local char g_err[256] = "";

int refuse(const char* what) {
  snprintf(g_err, sizeof(g_err), "%s", what);
  return -1;
}

template <int LANES, int HEADS>
cudaError_t launch_as(const cudaLaunchConfig_t& cfg, const Params& p, int f16, int interleaved) {
  return f16 ? interleaved ? cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<LANES, true, true, HEADS>, p)
                           : cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<LANES, true, false, HEADS>, p)
             : interleaved ? cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<LANES, false, true, HEADS>, p)
                           : cudaLaunchKernelEx(&cfg, qk_norm_rope_kernel<LANES, false, false, HEADS>, p);
}

constexpr double kWorth[4] = {0., 0.80, 0.95, 1.00};   // of a place, by the heads of a lane (0.70 / 0.90 and 0.90 / 1.00: no better)
template <int LANES>
cudaError_t launch(Params& p, int64_t tokens, int f16, int interleaved, void* stream) {
  constexpr int kGroups = kThreads / LANES;
  const int all = p.heads + 2 * p.kv_heads;
  // groups of lanes to a token (a power of two, so one or more tokens to a block) and heads of a lane: the fewest places without a
  // head, and of those the most heads to a lane.  (16384 tokens: 32 + 8 + 8 heads of 128, always 32 groups to a token 101 us, so
  // 88; 8 + 1 + 1 heads, one head to a lane 30 us, so 22.)
  int blocks = 0, heads = 0;
  double best = 0.;
  for (int shift = 0; (kGroups >> shift) > 0; ++shift)
    for (int h = 1; h <= 3; ++h) {
      const int places = (kGroups >> shift) * h, n = (all + places - 1) / places;
      const double worth = (double)all / (n * places) * kWorth[h];
      if (worth > best) best = worth, blocks = n, heads = h, p.token_shift = shift;
    }
  p.tokens = tokens;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((tokens + (1 << p.token_shift) - 1) >> p.token_shift), blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return heads == 1   ? launch_as<LANES, 1>(cfg, p, f16, interleaved)
         : heads == 2 ? launch_as<LANES, 2>(cfg, p, f16, interleaved)
                      : launch_as<LANES, 3>(cfg, p, f16, interleaved);
}

}  // namespace rotary
}  // namespace iris

extern "C" {

const char* iris_rotary_last_error() { return iris::rotary::g_err; }

// The arguments of a call, packed (see paged_attention.cu).  qkv [tokens, (heads + 2 kv_heads) * dim], 16-bit (dtype 0 bf16,
// 1 fp16); out [tokens, out_heads * dim], or qkv itself with out_heads = heads + kv_heads.  table [positions_in_table, rotary]
// fp32, or null with rotary 0; positions, slots int32 [tokens].  Pitches in elements.
struct IrisQkNormRopeArgs {
  const void *qkv;
  void *out;
  const void *positions, *table, *q_weight, *k_weight;
  void *k_cache, *v_cache;
  const void *slots;
  void *status, *stream;
  int64_t ld_in, ld_out, ld_table, page_pitch, slot_pitch, head_pitch;
  int64_t out_heads, positions_in_table, rotary, interleaved, pages, page_size, tokens, heads, kv_heads, dim, dtype;
  double eps;
};

int iris_k_qk_norm_rope(const IrisQkNormRopeArgs* args) {
  using namespace iris::rotary;
  g_err[0] = 0;
  const auto [qkv, out, positions, table, q_weight, k_weight, k_cache, v_cache, slots, status, stream, ld_in0, ld_out0, ld_table0,
              page_pitch0, slot_pitch0, head_pitch0, out_heads, positions_in_table, rotary, interleaved, pages, page_size, tokens,
              heads, kv_heads, dim, dtype, eps] = *args;
  int64_t ld_in = ld_in0, ld_out = ld_out0, ld_table = ld_table0, page_pitch = page_pitch0, slot_pitch = slot_pitch0;
  int64_t head_pitch = head_pitch0;
  if (tokens < 1 || tokens > 0x7fffffff || heads < 1 || kv_heads < 1 || heads > 65536 || kv_heads > 65536) return refuse("sizes out of range");
  if (dim < 16 || dim > 512 || dim % 16) return refuse("head dimension must be a multiple of 16, at most 512");
  if (rotary < 0 || rotary > dim || rotary % 16 || (rotary && !table)) return refuse("rotated part must be a multiple of 16 within the head");
  if (dtype != 0 && dtype != 1) return refuse("dtype must be 0 (bf16) or 1 (fp16)");
  if (k_cache && (page_size < 1 || (page_size & (page_size - 1)) || page_size > (1 << 30) || pages < 1 || pages > 0x7fffffff))
    return refuse("page size must be a power of two");
  // a pitch along one element says nothing
  if (tokens == 1) ld_in = ld_out = 0;
  if (positions_in_table == 1) ld_table = 0;
  if (pages == 1) page_pitch = 0;
  if (page_size == 1) slot_pitch = 0;
  if (kv_heads == 1) head_pitch = 0;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(table) |
                          reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight) |
                          reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache);
  if (bases % 16 || (ld_in | ld_out) % 8 || ld_table % 4 || (k_cache && (page_pitch | slot_pitch | head_pitch) % 8))
    return refuse("rows must start on 16 bytes");
  {
    // what is written shares no memory with anything else, but for out in the place of qkv, which the caller looks after
    using namespace iris::overlap;
    const Rows in(qkv, (heads + 2 * kv_heads) * dim * 2, {tokens, ld_in * 2});
    const Rows to(out, out_heads * dim * 2, {tokens, ld_out * 2});
    const Rows keys(k_cache, dim * 2, {pages, page_pitch * 2}, {page_size, slot_pitch * 2}, {kv_heads, head_pitch * 2});
    const Rows values(v_cache, dim * 2, {pages, page_pitch * 2}, {page_size, slot_pitch * 2}, {kv_heads, head_pitch * 2});
    if (!apart(to) || !apart(keys) || meet(keys, values)) return refuse("rows of the cache, or of out, must not overlap");
    if (meet(keys, in) || meet(values, in) || meet(keys, to) || meet(values, to))
      return refuse("the cache must share no memory with qkv or out");
    const Rows read[] = {Rows(positions, tokens * 4), Rows(slots, tokens * 4), Rows(q_weight, dim * 2),
                         Rows(k_weight, dim * 2), Rows(table, rotary * 4, {positions_in_table, ld_table * 4})};
    for (const Rows& r : read)
      if (meet(to, r) || meet(keys, r) || meet(values, r))
        return refuse("out and the cache must share no memory with positions, slots, weights or the table");
  }
  Params p;
  memset(&p, 0, sizeof(p));
  p.qkv = static_cast<const uint8_t*>(qkv);
  p.out = static_cast<uint8_t*>(out);
  p.positions = static_cast<const int*>(positions);
  p.table = static_cast<const float*>(table);
  p.q_weight = static_cast<const uint8_t*>(q_weight);
  p.k_weight = static_cast<const uint8_t*>(k_weight);
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.slots = static_cast<const int*>(slots);
  p.status = static_cast<iris::StatusBlock*>(status);
  p.ld_in = ld_in * 2, p.ld_out = ld_out * 2, p.ld_table = ld_table;
  p.page_pitch = page_pitch * 2, p.slot_pitch = slot_pitch * 2, p.head_pitch = head_pitch * 2;
  p.cache_slots = k_cache ? pages * page_size : 0;
  p.positions_in_table = !table || positions_in_table > 0x7fffffff ? 0x7fffffff : (int)positions_in_table;
  p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.dim = (int)dim, p.half = (int)rotary / 2, p.out_heads = (int)out_heads;
  p.eps = (float)eps;
  while (k_cache && (1 << p.page_shift) < page_size) ++p.page_shift;
  const int pieces = (int)dim / 16;
  const cudaError_t e = pieces <= 4    ? launch<4>(p, tokens, (int)dtype, (int)interleaved, stream)
                        : pieces <= 8  ? launch<8>(p, tokens, (int)dtype, (int)interleaved, stream)
                        : pieces <= 16 ? launch<16>(p, tokens, (int)dtype, (int)interleaved, stream)
                                       : launch<32>(p, tokens, (int)dtype, (int)interleaved, stream);
  if (e == cudaSuccess) return 0;
  (void)cudaGetLastError();   // reported here: it must not turn up at someone else's launch
  snprintf(g_err, sizeof(g_err), "launch: %s", cudaGetErrorString(e));
  return -3;
}

}  // extern "C"
