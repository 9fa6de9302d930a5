// Attention of one new token per request over a paged key / value cache.
//   out[i, h, :] = softmax_t(scale q[i, h, :] . K[t, h / G, :]) V[t, h / G, :],  t < len_i; token t lies in page table[i][t / P] at place t % P
// G = query heads per key head. A request without tokens gets zeros. Every key and value is read once; the pass is bound by that.
//
// Split: the work is a list of tiles of tokens, ordered by (request, unit of heads, tile); each CTA takes an equally costly stretch of the list, whatever
// the lengths of the requests are (a long document next to short ones, few requests of many tokens); a (request, unit) costs as much as two tiles more than it has. A stretch that holds all tiles of a (request, unit)
// writes the result; one that holds some of them leaves its maximum, sum and unnormalised output in 32 bits, and a second small kernel joins those.
// A unit is a key head with up to 8 * MT of its query heads.
//
// Within a CTA four warps look the pages up and send for them, several tiles ahead, also across the end of a (request, unit); the others multiply, 16 tokens of a
// tile each, which are waited for and refilled by themselves. Rows beyond the length are filled with zeros and not read. The copies are the 16-byte
// asynchronous ones of the loading warps' lanes, which take any page size and any strides: boxes of 16 tokens x 128 bytes by TMA were issued and fetched at
// 5.0 to 5.9 TB/s without any product behind them, and boxes cannot be larger where a page holds 16 tokens.
// What a warp keeps per query head are the running maximum, sum and output in registers; the warps meet at the end of a (request, unit).
// bf16: products by warp-level matrix instructions (16 x 8 x 16). A decoding step has 1 to 32 rows per key head and is bound by memory: the
// larger tensor-memory instructions have nothing to win (64 rows at least, keys would pass through descriptors) and the sixteen rows here are only half used:
// rows 0..7 are 8 query heads with the weights rounded to bf16, rows 8..15 the same heads with what the rounding lost. Their sum weighs the
// values with 16 bits of mantissa at no further instruction; weights of 8 bits would add an error as large as the rounding of the result.
// fp32: products by fused multiply-adds.
#include "tcgen05.cuh"
#include <algorithm>

namespace {

using namespace rbt;

constexpr int kRows = 16;  // tokens of a warp in a tile

struct Args {
  const void *q, *k, *v;
  const int *table, *lens;
  void* out;
  float* part;   // [grid][2][unit heads][D + 4]: output, maximum (log2), sum
  int2* owners;  // [requests * units]: first and last CTA
  int* status;
  int64_t q_req, q_head, kp, kh, kt, vp, vh, vt, table_stride;
  int n, heads, kv_heads, d, page, blocks, num_pages, group, units_per_kv, unit_heads, grid;
  int q_words;  // queries can be read two features at a time
  int whole;  // 16 tokens from a multiple of 16 on lie in one page, and rows are as wide as in shared memory
  float scale_log2;
};

template <typename T, int DP>
struct Shape {
  static constexpr bool kBf16 = sizeof(T) == 2;
  static constexpr int kRowBytes = DP * (int)sizeof(T), kCols = 128 / (int)sizeof(T);  // features of a 128-byte row in shared memory
  static constexpr int kBlocks = kRowBytes / 128;
  static constexpr int kPart = kRows * kRowBytes;  // 16 tokens: blocks of 16 rows of 128 bytes, 16-byte pieces swizzled by the row
  static constexpr int kWarps = kRowBytes <= 256 ? 8 : kRowBytes <= 512 ? 4 : 2;
  static constexpr int kLoaders = std::min(4, kWarps), kThreads = (kWarps + kLoaders) * 32;
  static constexpr int kTile = kWarps * kRows;
  static constexpr int kStage = 2 * kWarps * kPart;  // keys, values
  static constexpr int kPitch = DP + 8;              // floats of a head where the warps meet (no bank conflicts)
  static constexpr int kMeet = 8 * kPitch + 16;      // of a warp: outputs, maxima, sums
  static constexpr int kExtra = kBf16 ? 0 : 8 * DP + kWarps * 8 * kRows;  // fp32: queries, weights of a tile
  static constexpr int kFloats = kWarps * kMeet + kExtra;
  static constexpr int kStages = std::min(6, (int)((227 * 1024 - 1024 - 1536 - kFloats * 4) / kStage));
  static constexpr int kSmem = kStages * kStage + kFloats * 4 + 1024;
};

struct Place {  // in the list of tiles
  int req, unit, tile, tiles, len;  // tiles: of the request
};

constexpr int kUnitCost = 2;  // of beginning and ending a (request, unit), in tiles: queries, the meeting of the warps, the result

__device__ __forceinline__ int length_of(const Args& a, int req) { return (int)min((int64_t)max(a.lens[req], 0), (int64_t)a.blocks * a.page); }
template <int kTile>
__device__ __forceinline__ int tiles_of(int len) { return (int)(((int64_t)len + kTile - 1) / kTile); }

// first tile of the next (request, unit)
template <int kTile>
__device__ __forceinline__ void next_unit(const Args& a, Place& p, int units) {
  p.tile = 0;
  if (++p.unit < units) return;
  p.unit = 0;
  do {
    if (++p.req >= a.n) {
      p.tiles = p.len = 0;
      return;
    }
    p.len = length_of(a, p.req);
    p.tiles = tiles_of<kTile>(p.len);
  } while (p.tiles == 0);
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool real) {  // zeros unless real
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// this thread's arrival at the barrier, once its copies so far are there
__device__ __forceinline__ void arrive_copied(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// exp2 of x - m where m may be -inf (nothing seen yet): 0
__device__ __forceinline__ float exp2_of(float x, float m) { return m == -INFINITY ? 0.f : exp2f(x - m); }

// What a warp knows of its 8 query heads: running maximum (of scores in units of log2), sum, unnormalised output.
// bf16: lane (g, j) = (lane / 4, lane % 4) has features 8 i + 2 j, + 1 of head g in rows g and g + 8 of accumulator i.
template <typename T, int DP>
struct State;

template <int DP>
struct State<__nv_bfloat16, DP> {
  using T = __nv_bfloat16;
  using S = Shape<T, DP>;
  static constexpr int kSteps = DP / 16, kTiles = DP / 8;
  uint32_t q[kSteps][2];
  float o[kTiles][4];
  float m, l;  // l: of this lane's columns

  __device__ __forceinline__ void fetch_queries(const Args& a, const Place& p, int m_tile) {
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const int kv = p.unit / a.units_per_kv, h = (p.unit % a.units_per_kv) * a.unit_heads + m_tile * 8 + g;
    const bool real = h < a.group && m_tile * 8 + g < a.unit_heads;
    const T* src = reinterpret_cast<const T*>(a.q) + p.req * a.q_req + (real ? (int64_t)(kv * a.group + h) * a.q_head : 0);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int e = s * 16 + b * 8 + j * 2;
        uint32_t x = 0u;
        if (real && e < a.d) {  // (D is a multiple of 8)
          const uint16_t* u = reinterpret_cast<const uint16_t*>(src) + e;
          x = a.q_words ? *reinterpret_cast<const uint32_t*>(u) : (uint32_t)u[0] | (uint32_t)u[1] << 16;
        }
        q[s][b] = x;
      }
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  // 16 tokens; bits: which of them there are
  __device__ __forceinline__ void add(const Args& a, uint32_t keys, uint32_t vals, uint32_t bits, const float*, float*) {
    const int lane = threadIdx.x & 31, j = lane & 3;
    // Fragments are fetched ahead of the products that use them, the first of the values ahead of the exponentials: fetched one by one, their latency was
    // a third of the time of a tile. Two accumulators per score halve the chain of products.
    constexpr int kDeep = kSteps < 8 ? kSteps : 8;
    float s[2][2][4] = {};
    const int turn = lane & 7;
    const uint32_t at_k = keys + ((lane & 7) + ((lane >> 4) << 3)) * 128, piece_k = (lane >> 3) & 1;
    const uint32_t at_v = vals + ((lane & 7) + ((lane >> 3) & 1) * 8) * 128, piece_v = lane >> 4;
#pragma unroll
    for (int k0 = 0; k0 < kSteps; k0 += kDeep) {
      uint32_t b[kDeep][4];
#pragma unroll
      for (int k = 0; k < kDeep; ++k) ldsm4(b[k], at_k + ((k0 + k) >> 2) * (kRows * 128) + ((((k0 + k) & 3) * 2 + piece_k) ^ turn) * 16);
#pragma unroll
      for (int k = 0; k < kDeep; ++k) {
        const uint32_t qa[4] = {q[k0 + k][0], 0u, q[k0 + k][1], 0u};
        mma(s[k & 1][0], qa, b[k][0], b[k][1]);
        mma(s[k & 1][1], qa, b[k][2], b[k][3]);
      }
    }
    constexpr int kVal = 4;  // pairs of accumulators fetched at a time
    auto fetch = [&](uint32_t (*b)[4], int i0) {
#pragma unroll
      for (int i = 0; i < kVal; ++i) ldsm4_t(b[i], at_v + ((i0 + i) >> 2) * (kRows * 128) + ((((i0 + i) & 3) * 2 + piece_v) ^ turn) * 16);
    };
    uint32_t vb[2][kVal][4];
    fetch(vb[0], 0);
    float x[4];
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9
      const int t = (c >> 1) * 8 + 2 * j + (c & 1);
      x[c] = bits >> t & 1 ? (s[0][c >> 1][c & 1] + s[1][c >> 1][c & 1]) * a.scale_log2 : -INFINITY;
      top = max_nan(top, x[c]);
    }
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float mn = max_nan(m, top);
    const float f = exp2_of(m, mn);
    m = mn;
    uint32_t hi[2], lo[2];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float p0 = exp2_of(x[2 * c], mn), p1 = exp2_of(x[2 * c + 1], mn);
      sum += p0 + p1;
      hi[c] = pack2(p0, p1);
      lo[c] = pack2(p0 - __uint_as_float(hi[c] << 16), p1 - __uint_as_float(hi[c] & 0xffff0000u));
    }
    l = l * f + sum;
    if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] *= f;
    }
    const uint32_t pa[4] = {hi[0], lo[0], hi[1], lo[1]};
#pragma unroll
    for (int i0 = 0; i0 < kTiles / 2; i0 += kVal) {
      const int now = i0 / kVal & 1;
      if (i0 + kVal < kTiles / 2) fetch(vb[now ^ 1], i0 + kVal);
#pragma unroll
      for (int i = 0; i < kVal; ++i) {
        mma(o[2 * (i0 + i)], pa, vb[now][i][0], vb[now][i][1]);
        mma(o[2 * (i0 + i) + 1], pa, vb[now][i][2], vb[now][i][3]);
      }
    }
  }

  __device__ __forceinline__ void finish() {  // sums over the lanes of a head, both roundings of the weights together
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      o[i][0] += o[i][2];
      o[i][1] += o[i][3];
    }
  }
  __device__ __forceinline__ void give(float* to) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) *reinterpret_cast<float2*>(to + g * S::kPitch + i * 8 + j * 2) = make_float2(o[i][0], o[i][1]);
    if (j == 0) {
      to[8 * S::kPitch + g] = m;
      to[8 * S::kPitch + 8 + g] = l;
    }
  }
};

// fp32: lanes l and l + 16 share token l's score (alternate groups of four features); lane has features lane, lane + 32, ... of the output of every head
template <int DP>
struct State<float, DP> {
  using S = Shape<float, DP>;
  static constexpr int kCols = DP / 32;
  float o[8][kCols];
  float m[8], l[8];  // l: of this lane's token

  // all multiplying warps; they meet afterwards
  __device__ __forceinline__ void share_queries(const Args& a, const Place& p, float* qs) {
    const int kv = p.unit / a.units_per_kv, h0 = (p.unit % a.units_per_kv) * a.unit_heads;
    for (int i = threadIdx.x; i < 8 * DP; i += S::kWarps * 32) {
      const int g = i / DP, e = i - g * DP;
      qs[i] = g < a.unit_heads && h0 + g < a.group && e < a.d
                  ? reinterpret_cast<const float*>(a.q)[p.req * a.q_req + (int64_t)(kv * a.group + h0 + g) * a.q_head + e] * a.scale_log2 : 0.f;
    }
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[g][c] = 0.f;
    }
  }
  __device__ __forceinline__ static float4 at(uint32_t from) {
    float4 r;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "r"(from) : "memory");
    return r;
  }
  __device__ __forceinline__ static float one_at(uint32_t from) {
    float r;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(from) : "memory");
    return r;
  }
  __device__ __forceinline__ void add(const Args& a, uint32_t keys, uint32_t vals, uint32_t bits, const float* qs, float* ps) {
    const int lane = threadIdx.x & 31, t = lane & 15, half = lane >> 4;
    float s[8] = {};
#pragma unroll 4
    for (int c = half; c < DP / 4; c += 2) {  // pieces of four features
      const float4 k = at(keys + (c >> 3) * (kRows * 128) + t * 128 + (((c & 7) ^ (t & 7)) << 4));
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        if (g < a.unit_heads) {
          const float4 q = *reinterpret_cast<const float4*>(qs + g * DP + c * 4);
          s[g] += k.x * q.x + k.y * q.y + k.z * q.z + k.w * q.w;
        }
      }
    }
    const bool there = bits >> t & 1;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g >= a.unit_heads) continue;
      float x = s[g] + __shfl_xor_sync(0xffffffffu, s[g], 16);
      x = there ? x : -INFINITY;
      float top = x;
#pragma unroll
      for (int w = 1; w < 16; w <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = max_nan(m[g], top), f = exp2_of(m[g], mn), p = exp2_of(x, mn);
      m[g] = mn;
      l[g] = l[g] * f + (half ? 0.f : p);
      if (!half) ps[g * kRows + t] = p;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[g][c] *= f;
    }
    __syncwarp();
#pragma unroll
    for (int t4 = 0; t4 < kRows; t4 += 4) {
      float v[4][kCols];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < kCols; ++c) v[r][c] = one_at(vals + c * (kRows * 128) + (t4 + r) * 128 + (((lane >> 2) ^ ((t4 + r) & 7)) << 4) + (lane & 3) * 4);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        if (g >= a.unit_heads) continue;
        const float4 p = *reinterpret_cast<const float4*>(ps + g * kRows + t4);
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[g][c] += p.x * v[0][c] + p.y * v[1][c] + p.z * v[2][c] + p.w * v[3][c];
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int g = 0; g < 8; ++g) l[g] = warp_sum(l[g]);
  }
  __device__ __forceinline__ void give(float* to) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) to[g * S::kPitch + c * 32 + lane] = o[g][c];
      if (lane == 0) {
        to[8 * S::kPitch + g] = m[g];
        to[8 * S::kPitch + 8 + g] = l[g];
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void put4(T* to, float4 v);
template <>
__device__ __forceinline__ void put4<float>(float* to, float4 v) { *reinterpret_cast<float4*>(to) = v; }
template <>
__device__ __forceinline__ void put4<__nv_bfloat16>(__nv_bfloat16* to, float4 v) { *reinterpret_cast<uint2*>(to) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w)); }

// MT: groups of 8 query heads in a unit; multiplying warp w has group w % MT of the tokens of share w / MT of a tile
template <typename T, int DP, int MT>
__global__ void __launch_bounds__(Shape<T, DP>::kThreads, 1)
attention_kernel(const Args a) {
  using S = Shape<T, DP>;
  constexpr int kWarps = S::kWarps, kShares = kWarps / MT, kStages = S::kStages, kLoaders = S::kLoaders;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  float* boxes = reinterpret_cast<float*>(smem + kStages * S::kStage);
  __shared__ uint64_t full[kStages][kWarps], empty[kStages][kWarps], meeting;
  __shared__ uint32_t notes[kStages][kWarps];  // of 16 tokens: those that there are as bits; bit 16: some lie within the length
  __shared__ long long warp_sums[kWarps + kLoaders][2], rank_shared[2], cost_shared;
  __shared__ Place start_shared;
  __shared__ int abort_shared;
  volatile int* abort = &abort_shared;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int units = a.kv_heads * a.units_per_kv;
  if (threadIdx.x == 0) {
    abort_shared = 0;
    for (int i = 0; i < kStages * kWarps; ++i) {
      mbar_init(&full[0][0] + i, 33);  // the lanes' copies, the note
      mbar_init(&empty[0][0] + i, MT);
    }
    mbar_init(&meeting, kWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  rb_pdl_wait();
  rb_pdl_launch();

  // This CTA's stretch of the list: prefix sums of cost and tiles over the requests, a run of them per thread. A place in the list is a cost; those that fall to the
  // beginning of a (request, unit) stand for its first tile.
  const int run = (a.n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int r0 = min((int64_t)a.n, (int64_t)threadIdx.x * run), r1 = min(a.n, r0 + run);
  auto cost_of = [&](int tiles) { return tiles ? (long long)(tiles + kUnitCost) * units : 0LL; };
  long long mine = 0, mine_tiles = 0;
  for (int r = r0; r < r1; ++r) {
    const int tiles = tiles_of<S::kTile>(length_of(a, r));
    mine += cost_of(tiles);
    mine_tiles += (long long)tiles * units;
  }
  long long inc = mine, inc_tiles = mine_tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, inc, o), y = __shfl_up_sync(0xffffffffu, inc_tiles, o);
    if (lane >= o) {
      inc += x;
      inc_tiles += y;
    }
  }
  if (lane == 31) {
    warp_sums[warp][0] = inc;
    warp_sums[warp][1] = inc_tiles;
  }
  __syncthreads();
  long long total = 0, total_tiles = 0, before = inc - mine, before_tiles = inc_tiles - mine_tiles;
#pragma unroll
  for (int w = 0; w < kWarps + kLoaders; ++w) {
    if (w < warp) {
      before += warp_sums[w][0];
      before_tiles += warp_sums[w][1];
    }
    total += warp_sums[w][0];
    total_tiles += warp_sums[w][1];
  }
  const long long per = max((total + a.grid - 1) / a.grid, 1LL);
  const long long first = per * blockIdx.x, last = min(total, first + per);
  if (first >= last) return;
  if (threadIdx.x == 0 && last == total) rank_shared[1] = total_tiles;
  for (int end = 0; end < 2; ++end) {
    const long long want = end ? last : first;
    if (!(before <= want && want < before + mine)) continue;
    long long c = before, k = before_tiles;
    for (int r = r0; r < r1; ++r) {
      const int len = length_of(a, r), tiles = tiles_of<S::kTile>(len);
      if (want < c + cost_of(tiles)) {
        const long long in = want - c;
        const int unit = (int)(in / (tiles + kUnitCost)), tile = max((int)(in % (tiles + kUnitCost)) - kUnitCost, 0);
        rank_shared[end] = k + (long long)unit * tiles + tile;
        if (!end) {
          start_shared = Place{r, unit, tile, tiles, len};
          cost_shared = c + (long long)unit * (tiles + kUnitCost);
        }
        break;
      }
      c += cost_of(tiles);
      k += (long long)tiles * units;
    }
  }
  __syncthreads();
  const int n_tiles = (int)(rank_shared[1] - rank_shared[0]);
  bool ok = true;

  if (warp >= kWarps) {
    // ---- loads. Loading warp w has the parts of 16 tokens w, w + kLoaders, ... of a tile; lane r looks the page of row r of a part up, a tile ahead
    constexpr int kMyParts = kWarps / kLoaders, kPer = 16 / (int)sizeof(T), kCopies = S::kRowBytes / 16;
    static_assert(kMyParts <= 2, "a lane per row");
    const int loader = warp - kWarps, my_row = (loader + (lane >> 4) * kLoaders) * kRows + (lane & 15);
    const bool mine_at_all = (lane >> 4) < kMyParts;
    Place p = start_shared, ahead = p;
    int pg = -1, at = 0, ahead_pg = -1, ahead_at = 0;
    auto look_up = [&]() {
      const int64_t t = (int64_t)ahead.tile * S::kTile + my_row;
      ahead_pg = -1;
      if (mine_at_all && t < ahead.len) {
        const int b = (int)t / a.page;
        ahead_at = (int)t - b * a.page;
        ahead_pg = a.table[(int64_t)ahead.req * a.table_stride + b];
      }
    };
    look_up();
    const int64_t k_step = a.kt * (int64_t)sizeof(T) * (32 / kCopies > 0 ? 32 / kCopies : 1), v_step = a.vt * (int64_t)sizeof(T) * (32 / kCopies > 0 ? 32 / kCopies : 1);
    int n = 0, s = 0, round = 0;
#pragma unroll 1
    for (; n < n_tiles; ++n) {
      p = ahead;
      pg = ahead_pg;
      at = ahead_at;
      if (n + 1 < n_tiles) {
        if (++ahead.tile == ahead.tiles) next_unit<S::kTile>(a, ahead, units);
        look_up();
      }
      const bool real = pg >= 0 && pg < a.num_pages;  // (no such token; or a page that is none: as if the token were not there)
      const uint32_t bits = __ballot_sync(0xffffffffu, real);
      const int64_t place = real ? at : 0, in = real ? pg : 0;
      const int kv = a.units_per_kv == 1 ? p.unit : p.unit / a.units_per_kv;
      const int64_t k_row = (int64_t)a.k + (int64_t)sizeof(T) * (in * a.kp + kv * a.kh + place * a.kt);
      const int64_t v_row = (int64_t)a.v + (int64_t)sizeof(T) * (in * a.vp + kv * a.vh + place * a.vt);
#pragma unroll
      for (int j = 0; j < kMyParts; ++j) {
        const int part = loader + j * kLoaders;
        if (round > 0) ok = ok && warp_wait(&empty[s][part], (round - 1) & 1, abort);
        if (!ok) break;
        const uint32_t to = smem_u32(smem) + s * S::kStage + part * S::kPart;
        const uint32_t mine = bits >> (16 * j);
        if (kCopies <= 32 && a.whole && (mine & 0xffffu) == 0xffffu) {  // 16 tokens of one page: rows at a fixed distance
          const int row0 = lane / kCopies, c = lane % kCopies;
          int64_t kr = __shfl_sync(0xffffffffu, k_row, 16 * j) + row0 * a.kt * (int64_t)sizeof(T) + c * 16;
          int64_t vr = __shfl_sync(0xffffffffu, v_row, 16 * j) + row0 * a.vt * (int64_t)sizeof(T) + c * 16;
#pragma unroll
          for (int i = 0; i < kRows * kCopies / 32; ++i) {
            const int row = i * (32 / kCopies) + row0;
            const uint32_t dst = to + (c >> 3) * (kRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
            copy16(dst, reinterpret_cast<const void*>(kr));
            copy16(dst + kWarps * S::kPart, reinterpret_cast<const void*>(vr));
            kr += k_step;
            vr += v_step;
          }
        } else {
#pragma unroll
        for (int i = 0; i < kRows * kCopies / 32; ++i) {
          const int id = i * 32 + lane, row = id / kCopies, c = id % kCopies;
          const int64_t kr = __shfl_sync(0xffffffffu, k_row, 16 * j + row), vr = __shfl_sync(0xffffffffu, v_row, 16 * j + row);
          const bool there = (mine >> row & 1) && (S::kRowBytes == a.d * (int)sizeof(T) || c * kPer < a.d);  // (features beyond D: zeros)
          const uint32_t dst = to + (c >> 3) * (kRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
          copy16(dst, reinterpret_cast<const void*>(kr + (there ? c * 16 : 0)), there);
          copy16(dst + kWarps * S::kPart, reinterpret_cast<const void*>(vr + (there ? c * 16 : 0)), there);
        }
        }
        arrive_copied(&full[s][part]);
        if (lane == 0) {
          const int64_t t0 = (int64_t)p.tile * S::kTile + part * kRows;
          notes[s][part] = (mine & 0xffffu) | (t0 < p.len ? 1u << 16 : 0u);
          arrive(&full[s][part]);
        }
      }
      if (!ok) break;
      if (++s == kStages) {
        s = 0;
        ++round;
      }
    }
    if (!ok) {  // a wait ran out
      *abort = 1;
      if (lane == 0 && a.status) atomicCAS(a.status, 0, (9 << 24) | 1);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // ---- products
  const int m_tile = warp % MT, share = warp / MT;
  float* qs = boxes + kWarps * S::kMeet;
  float* ps = qs + 8 * DP + warp * 8 * kRows;
  const uint32_t stages = smem_u32(smem);
  int meetings = 0;
  auto meet = [&]() {
    __syncwarp();
    if (lane == 0) arrive(&meeting);
    ok = warp_wait(&meeting, meetings++ & 1, abort);
  };
  State<T, DP> st;
  Place cur = start_shared;
  long long cost = cost_shared;  // where the present (request, unit) begins
  if constexpr (S::kBf16) st.fetch_queries(a, cur, m_tile);
  int n = 0, s = 0, round = 0;
#pragma unroll 1
  while (n < n_tiles) {
    const int count = min(cur.tiles - cur.tile, n_tiles - n);
    if constexpr (!S::kBf16) {
      st.share_queries(a, cur, qs);
      meet();
      if (!ok) break;
    }
    st.begin();
#pragma unroll 1
    for (int t = 0; t < count && ok; ++t) {
      constexpr int kMine = kWarps / kShares;  // parts of 16 tokens that are this warp's
#pragma unroll 1
      for (int i = 0; i < kMine; ++i) {
        const int w = share * kMine + i;
        ok = warp_wait(&full[s][w], round & 1, abort);
        if (!ok) break;
        const uint32_t word = notes[s][w];
        if (word >> 16) {
          const uint32_t keys = stages + s * S::kStage + w * S::kPart;
          st.add(a, keys, keys + kWarps * S::kPart, word & 0xffffu, qs, ps);
        }
        __syncwarp();
        if (lane == 0) arrive(&empty[s][w]);
      }
      if (++s == kStages) {
        s = 0;
        ++round;
      }
    }
    if (!ok) break;
    n += count;
    const Place done = cur;
    const bool ends = cur.tile + count == cur.tiles, whole = cur.tile == 0;
    if (n < n_tiles) {  // the next queries are under way while the warps meet
      next_unit<S::kTile>(a, cur, units);
      if constexpr (S::kBf16) st.fetch_queries(a, cur, m_tile);
    }
    // ---- the warps' outputs come together
    st.finish();
    if constexpr (S::kBf16) {
      meet();  // all have read what was there before
      if (!ok) break;
    }
    st.give(boxes + warp * S::kMeet);
    meet();
    if (!ok) break;
    const int kv = done.unit / a.units_per_kv, h0 = (done.unit % a.units_per_kv) * a.unit_heads;
    for (int i = threadIdx.x; i < 8 * MT * (DP / 4); i += kWarps * 32) {
      const int e = i % (DP / 4) * 4, g = i / (DP / 4) % 8, mt = i / (DP / 4) / 8, h = mt * 8 + g;
      if (e >= a.d || h >= a.unit_heads || h0 + h >= a.group) continue;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kShares; ++w) m = max_nan(m, boxes[(w * MT + mt) * S::kMeet + 8 * S::kPitch + g]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kShares; ++w) {
        const float* b = boxes + (w * MT + mt) * S::kMeet;
        const float f = exp2_of(b[8 * S::kPitch + g], m);
        const float4 x = *reinterpret_cast<const float4*>(b + g * S::kPitch + e);
        l += b[8 * S::kPitch + 8 + g] * f;
        o.x += x.x * f;
        o.y += x.y * f;
        o.z += x.z * f;
        o.w += x.w * f;
      }
      if (ends && whole) {
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        put4(reinterpret_cast<T*>(a.out) + ((int64_t)done.req * a.heads + kv * a.group + h0 + h) * a.d + e, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      } else {
        float* to = a.part + (((int64_t)blockIdx.x * 2 + (whole ? 1 : 0)) * a.unit_heads + h) * (a.d + 4);
        *reinterpret_cast<float4*>(to + e) = o;
        if (e == 0) *reinterpret_cast<float2*>(to + a.d) = make_float2(m, l);
      }
    }
    if (whole && threadIdx.x == 0)
      a.owners[(int64_t)done.req * units + done.unit] = make_int2((int)blockIdx.x, ends ? (int)blockIdx.x : (int)((cost + kUnitCost + done.tiles - 1) / per));
    cost += done.tiles + kUnitCost;
  }
  if (!ok) {
    *abort = 1;
    if (lane == 0 && a.status) atomicCAS(a.status, 0, (9 << 24) | 2);
  }
}

// joins the parts of a (request, unit) that several CTAs had, and writes the zeros of requests without tokens. A warp per query head.
template <typename T>
__global__ void __launch_bounds__(128)
join_kernel(const Args a, int units) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);  // (request, head)
  rb_pdl_wait();
  rb_pdl_launch();
  if (w >= (int64_t)a.n * a.heads) return;
  const int req = (int)(w / a.heads), head = (int)(w - (int64_t)req * a.heads);
  const int kv = head / a.group, in = head - kv * a.group, unit = kv * a.units_per_kv + in / a.unit_heads, row = in % a.unit_heads;
  T* out = reinterpret_cast<T*>(a.out) + w * a.d;
  if (length_of(a, req) == 0) {
    for (int e = lane; e < a.d; e += 32) out[e] = T(0.f);
    return;
  }
  const int2 own = a.owners[(int64_t)req * units + unit];
  if (own.x == own.y) return;  // one CTA had it all
  const int64_t pitch = (int64_t)a.unit_heads * (a.d + 4);
  // the first CTA's part is its last stretch (place 1), the others' their first (place 0)
  auto part = [&](int c) { return a.part + ((int64_t)c * 2 + (c == own.x ? 1 : 0)) * pitch + (int64_t)row * (a.d + 4); };
  float m = -INFINITY;
  for (int c = own.x + lane; c <= own.y; c += 32) m = max_nan(m, part(c)[a.d]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.f, acc[8] = {};
#pragma unroll 4
  for (int c = own.x; c <= own.y; ++c) {
    const float* p = part(c);
    const float f = exp2_of(p[a.d], m);
    l += p[a.d + 1] * f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < a.d) acc[k] += p[lane + 32 * k] * f;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (lane + 32 * k < a.d) out[lane + 32 * k] = T(acc[k] * inv);
}

template <typename T, int DP, int MT>
int launch(Args a, cudaStream_t stream) {
  using S = Shape<T, DP>;
  a.whole = a.page % kRows == 0 && a.d == DP;
  static_assert(S::kStages >= 2 && S::kSmem + 1536 <= 227 * 1024, "shared memory");
  static RbPerDevice ready;
  auto kernel = attention_kernel<T, DP, MT>;
  if (ready.needed()) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess) return rb_check_launch("paged_attention");
    ready.done();
  }
  rb_launch_pdl(kernel, dim3(a.grid), dim3(S::kThreads), (size_t)S::kSmem, stream, a);
  rb_launch_pdl(join_kernel<T>, dim3((unsigned)(((int64_t)a.n * a.heads + 3) / 4)), dim3(128), 0, stream, a, a.kv_heads * a.units_per_kv);
  return rb_check_launch("paged_attention");
}

template <typename T, int MT>
int by_dim(const Args& a, cudaStream_t stream) {
  if (a.d <= 64) return launch<T, 64, MT>(a, stream);
  if (a.d <= 128) return launch<T, 128, MT>(a, stream);
  return launch<T, 256, MT>(a, stream);
}

int units_of(int group, int bf16, int* unit_heads) {
  const int most = bf16 ? 32 : 8;
  const int units = (group + most - 1) / most;
  *unit_heads = (group + units - 1) / units;
  return units;
}

}  // namespace

// bytes of workspace for n requests: parts of the CTAs and the owners of the (request, unit)s
RB_EXPORT long long rb200_paged_attention_workspace(int n, int heads, int kv_heads, int d, int bf16) {
  int uh;
  const int units = kv_heads * units_of(heads / std::max(kv_heads, 1), bf16, &uh);
  return (long long)num_sms() * 2 * uh * (d + 4) * 4 + (long long)n * units * 8;
}

// q [n, heads, D]; k, v [pages, kv heads, page, D]; table [n][blocks] rows table_stride apart; out [n, heads, D] contiguous; strides: q request, head; k, v: page, head,
// token. Features have unit stride; caches start on 16 bytes and their strides are multiples of 16 bytes.
RB_EXPORT int rb200_paged_attention(const void* q, const void* k, const void* v, const int* table, long long table_stride, const int* lens, void* out,
                                    void* workspace, const long long* strides, int n, int heads, int kv_heads, int d, int page, int blocks, int num_pages, float scale,
                                    int bf16, int* status, cudaStream_t stream) {
  if (n <= 0 || heads <= 0) return RB_OK;
  const int unit = bf16 ? 8 : 4;
  bool ok = d >= 8 && d <= 256 && d % 8 == 0 && kv_heads >= 1 && heads % kv_heads == 0 && page >= 1 && blocks >= 0 && num_pages >= 0;
  for (int i = 2; i < 8; ++i) ok = ok && strides[i] % unit == 0 && strides[i] >= 0;
  ok = ok && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  if (!ok) {
    rb_set_error("paged_attention: head dim %d (a multiple of 8 up to 256), %d query heads over %d, page size %d, caches on 16 bytes", d, heads, kv_heads, page);
    return RB_ERR_UNSUPPORTED;
  }
  if (num_pages == 0 || blocks == 0) {  // no token anywhere
    if (cudaMemsetAsync(out, 0, (size_t)n * heads * d * (bf16 ? 2 : 4), stream) != cudaSuccess) return rb_check_launch("paged_attention");
    return RB_OK;
  }
  Args a = {};
  a.q = q; a.k = k; a.v = v; a.table = table; a.lens = lens; a.out = out; a.table_stride = table_stride; a.status = status;
  a.q_words = (reinterpret_cast<uintptr_t>(q) & 3) == 0 && strides[0] % 2 == 0 && strides[1] % 2 == 0;
  a.q_req = strides[0]; a.q_head = strides[1]; a.kp = strides[2]; a.kh = strides[3]; a.kt = strides[4]; a.vp = strides[5]; a.vh = strides[6]; a.vt = strides[7];
  a.n = n; a.heads = heads; a.kv_heads = kv_heads; a.d = d; a.page = page; a.blocks = blocks; a.num_pages = num_pages; a.group = heads / kv_heads;
  a.units_per_kv = units_of(a.group, bf16, &a.unit_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.grid = num_sms();
  a.part = reinterpret_cast<float*>(workspace);
  a.owners = reinterpret_cast<int2*>(a.part + (int64_t)a.grid * 2 * a.unit_heads * (d + 4));
  if (!bf16) return by_dim<float, 1>(a, stream);
  if (a.unit_heads <= 8) return by_dim<__nv_bfloat16, 1>(a, stream);
  if (a.unit_heads <= 16) return by_dim<__nv_bfloat16, 2>(a, stream);
  return by_dim<__nv_bfloat16, 4>(a, stream);
}
