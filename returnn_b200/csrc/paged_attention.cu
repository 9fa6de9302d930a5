// Attention of one new token per request over a paged key / value cache.
//   out[i, h, :] = softmax_t(scale q[i, h, :] . K[t, h / G, :]) V[t, h / G, :],  t < len_i; token t lies in page table[i][t / P] at place t % P
// G = query heads per key head. A request without tokens gets zeros. Every key and value is read once; the pass is bound by that.
//
// Split: the work is a list of tiles of tokens, ordered by (request, unit of heads, tile); each CTA takes an equal stretch of the list, whatever
// the lengths of the requests are (a long document next to short ones, few requests of many tokens). A stretch that holds all tiles of a (request, unit)
// writes the result; one that holds some of them leaves its maximum, sum and unnormalised output in 32 bits, and a second small kernel joins those.
// A unit is a key head with up to 8 * MT of its query heads.
//
// Within a CTA each warp loads 16 tokens of a tile by asynchronous copies of 16 bytes, several tiles ahead, also across the end of a (request, unit);
// rows beyond the length are filled with zeros and not read. What a warp keeps per query head are the running maximum, sum and output in registers.
// bf16: products by warp-level matrix instructions (16 x 8 x 16). A decoding step has 1 to 32 rows per key head and is bound by memory: the
// larger tensor-memory instructions have nothing to win (64 rows at least, keys would pass through descriptors) and the sixteen rows here are only half used:
// rows 0..7 are 8 query heads with the weights rounded to bf16, rows 8..15 the same heads with what the rounding lost. Their sum weighs the
// values with 16 bits of mantissa at no further instruction; weights of 8 bits would add an error as large as the rounding of the result.
// fp32: products by fused multiply-adds.
#include "common.cuh"
#include <algorithm>

namespace {

constexpr int kRows = 16;  // tokens of a warp in a tile

struct Args {
  const void *q, *k, *v;
  const int *table, *lens;
  void* out;
  float* part;   // [grid][2][unit heads][D + 2]: output, maximum (log2), sum
  int2* owners;  // [requests * units]: first and last CTA
  int64_t q_req, q_head, kp, kh, kt, vp, vh, vt, table_stride;
  int n, heads, kv_heads, d, page, blocks, num_pages, group, units_per_kv, unit_heads, grid;
  float scale_log2;
};

template <typename T, int DP>
struct Shape {
  static constexpr bool kBf16 = sizeof(T) == 2;
  static constexpr int kPitch = DP * (int)sizeof(T) + (kBf16 ? 16 : 32);  // bytes; the eight rows of a matrix load (bf16), four rows of two lanes (fp32) fall on different banks
  static constexpr int kStage = 2 * kRows * kPitch;                      // keys, values of one warp
  static constexpr int kWarps = DP * (int)sizeof(T) <= 256 ? 8 : DP * (int)sizeof(T) <= 512 ? 4 : 2;
  // outputs of half the warps, in their registers' order, with maximum and sum
  static constexpr int kOut = kBf16 ? DP / 8 * 2 : 8 * DP / 32;  // floats per lane
  static constexpr int kMerge = kWarps / 2 * (kOut * 32 + 16) * 4;
  static constexpr int kExtra = kBf16 ? 0 : (8 * DP + kWarps * 8 * kRows) * 4;  // fp32: queries, weights of a tile
  static constexpr int kStages = std::min(6, (int)((226 * 1024 - kMerge - kExtra) / (kWarps * kStage)));
  static constexpr int kSmem = kStages * kWarps * kStage + kMerge + kExtra;
  static constexpr int kTile = kWarps * kRows;
};

struct Place {  // in the list of tiles
  int req, unit, tile, tiles, len;
};

__device__ __forceinline__ int length_of(const Args& a, int req) { return (int)min((int64_t)max(a.lens[req], 0), (int64_t)a.blocks * a.page); }
template <int kTile>
__device__ __forceinline__ int tiles_of(int len) { return (int)(((int64_t)len + kTile - 1) / kTile); }

template <int kTile>
__device__ __forceinline__ void next(const Args& a, Place& p, int units) {
  if (++p.tile < p.tiles) return;
  p.tile = 0;
  if (++p.unit < units) return;
  p.unit = 0;
  do {
    if (++p.req >= a.n) {
      p.tiles = 0;
      return;
    }
    p.len = length_of(a, p.req);
    p.tiles = tiles_of<kTile>(p.len);
  } while (p.tiles == 0);
}

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_for() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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

// starts the copies of this warp's 16 tokens of a tile and leaves which of them there are, as bits
template <typename T, int DP>
__device__ __forceinline__ void load_tile(const Args& a, const Place& p, uint32_t stage, int warp, uint32_t* there) {
  using S = Shape<T, DP>;
  constexpr int kPer = 16 / sizeof(T), kCols = DP / kPer;  // copies of a row
  const int lane = threadIdx.x & 31;
  const int kv = p.unit / a.units_per_kv;
  const int64_t t0 = (int64_t)p.tile * S::kTile + warp * kRows;
  // lane r looks row r up
  int64_t ko = -1, vo = 0;
  if (lane < kRows && t0 + lane < p.len) {
    const int t = (int)t0 + lane, b = t / a.page;
    const int pg = a.table[(int64_t)p.req * a.table_stride + b];
    if (pg >= 0 && pg < a.num_pages) {  // (a page that is none: as if the token were not there)
      ko = pg * a.kp + kv * a.kh + (int64_t)(t - b * a.page) * a.kt;
      vo = pg * a.vp + kv * a.vh + (int64_t)(t - b * a.page) * a.vt;
    }
  }
  const uint32_t bits = __ballot_sync(0xffffffffu, ko >= 0);
  if (lane == 0) *there = bits;
#pragma unroll
  for (int i = 0; i < kRows * kCols / 32; ++i) {
    const int id = i * 32 + lane, row = id / kCols, col = (id - row * kCols) * kPer;
    const int64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
    const bool real = kr >= 0;
    if (col < a.d) {
      const uint32_t at = stage + row * S::kPitch + col * (int)sizeof(T);
      copy16(at, reinterpret_cast<const T*>(a.k) + (real ? kr + col : 0), real);
      copy16(at + kRows * S::kPitch, reinterpret_cast<const T*>(a.v) + (real ? vr + col : 0), real);
    }
  }
}

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

  __device__ __forceinline__ void begin(const Args& a, const Place& p, int m_tile, float*) {
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const int kv = p.unit / a.units_per_kv, h = (p.unit % a.units_per_kv) * a.unit_heads + m_tile * 8 + g;
    const bool real = h < a.group && m_tile * 8 + g < a.unit_heads;
    const T* src = reinterpret_cast<const T*>(a.q) + p.req * a.q_req + (real ? (int64_t)(kv * a.group + h) * a.q_head : 0);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int e = s * 16 + b * 8 + j * 2;
        const uint16_t* u = reinterpret_cast<const uint16_t*>(src);
        q[s][b] = real && e < a.d ? (uint32_t)u[e] | (uint32_t)u[e + 1] << 16 : 0u;  // (D is a multiple of 8)
      }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  // 16 tokens; bits: which of them there are
  __device__ __forceinline__ void add(const Args& a, uint32_t stage, uint32_t bits, const float*, float*) {
    const int lane = threadIdx.x & 31, j = lane & 3;
    float s[2][4] = {};
    {
      const uint32_t at = stage + ((lane & 7) + ((lane >> 4) << 3)) * S::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t b[4];
        ldsm4(b, at + k * 32);
        const uint32_t qa[4] = {q[k][0], 0u, q[k][1], 0u};
        mma(s[0], qa, b[0], b[1]);
        mma(s[1], qa, b[2], b[3]);
      }
    }
    float x[4];
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9
      const int t = (c >> 1) * 8 + 2 * j + (c & 1);
      x[c] = bits >> t & 1 ? s[c >> 1][c & 1] * a.scale_log2 : -INFINITY;
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
    const uint32_t at = stage + kRows * S::kPitch + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::kPitch + (lane >> 4) * 16;
#pragma unroll
    for (int i = 0; i < kTiles / 2; ++i) {
      uint32_t b[4];
      ldsm4_t(b, at + i * 32);
      mma(o[2 * i], pa, b[0], b[1]);
      mma(o[2 * i + 1], pa, b[2], b[3]);
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
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) reinterpret_cast<float2*>(to)[i * 32 + lane] = make_float2(o[i][0], o[i][1]);
    if ((lane & 3) == 0) {
      to[S::kOut * 32 + (lane >> 2)] = m;
      to[S::kOut * 32 + 8 + (lane >> 2)] = l;
    }
  }
  __device__ __forceinline__ void take(const float* from) {
    const int lane = threadIdx.x & 31;
    const float om = from[S::kOut * 32 + (lane >> 2)], ol = from[S::kOut * 32 + 8 + (lane >> 2)];
    const float mn = max_nan(m, om), f = exp2_of(m, mn), of = exp2_of(om, mn);
    m = mn;
    l = l * f + ol * of;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const float2 x = reinterpret_cast<const float2*>(from)[i * 32 + lane];
      o[i][0] = o[i][0] * f + x.x * of;
      o[i][1] = o[i][1] * f + x.y * of;
    }
  }
  __device__ __forceinline__ void write(const Args& a, const Place& p, int m_tile) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const int kv = p.unit / a.units_per_kv, h = (p.unit % a.units_per_kv) * a.unit_heads + m_tile * 8 + g;
    if (h >= a.group || m_tile * 8 + g >= a.unit_heads) return;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T* out = reinterpret_cast<T*>(a.out) + ((int64_t)p.req * a.heads + kv * a.group + h) * a.d;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int e = i * 8 + j * 2;
      if (e < a.d) *reinterpret_cast<uint32_t*>(out + e) = pack2(o[i][0] * inv, o[i][1] * inv);
    }
  }
  __device__ __forceinline__ void leave(const Args& a, float* part, int m_tile) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3, h = m_tile * 8 + g;
    if (h >= a.unit_heads) return;
    float* to = part + (int64_t)h * (a.d + 2);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int e = i * 8 + j * 2;
      if (e < a.d) *reinterpret_cast<float2*>(to + e) = make_float2(o[i][0], o[i][1]);
    }
    if (j == 0) *reinterpret_cast<float2*>(to + a.d) = make_float2(m, l);
  }
};

// fp32: two lanes share a token's score (alternate groups of four features); lane has features lane, lane + 32, ... of the output of every head
template <int DP>
struct State<float, DP> {
  using S = Shape<float, DP>;
  static constexpr int kCols = DP / 32;
  float o[8][kCols];
  float m[8], l[8];  // l: of this lane's token

  __device__ __forceinline__ void begin(const Args& a, const Place& p, int, float* qs) {  // (all threads of the CTA)
    const int kv = p.unit / a.units_per_kv, h0 = (p.unit % a.units_per_kv) * a.unit_heads;
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * DP; i += blockDim.x) {
      const int g = i / DP, e = i - g * DP;
      qs[i] = g < a.unit_heads && h0 + g < a.group && e < a.d
                  ? reinterpret_cast<const float*>(a.q)[p.req * a.q_req + (int64_t)(kv * a.group + h0 + g) * a.q_head + e] * a.scale_log2 : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[g][c] = 0.f;
    }
  }
  __device__ __forceinline__ void add(const Args& a, uint32_t stage_at, uint32_t bits, const float* qs, float* ps) {
    extern __shared__ __align__(128) uint8_t smem[];
    const uint8_t* stage = smem + (stage_at - smem_of(smem));
    const int lane = threadIdx.x & 31, t = lane >> 1, half = lane & 1;
    float s[8] = {};
    const float* key = reinterpret_cast<const float*>(stage + t * S::kPitch);
#pragma unroll 4
    for (int e = half * 4; e < DP; e += 8) {
      const float4 k = *reinterpret_cast<const float4*>(key + e);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        if (g < a.unit_heads) {
          const float4 q = *reinterpret_cast<const float4*>(qs + g * DP + e);
          s[g] += k.x * q.x + k.y * q.y + k.z * q.z + k.w * q.w;
        }
      }
    }
    const bool there = bits >> t & 1;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g >= a.unit_heads) continue;
      float x = s[g] + __shfl_xor_sync(0xffffffffu, s[g], 1);
      x = there ? x : -INFINITY;
      float top = x;
#pragma unroll
      for (int w = 2; w < 32; w <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = max_nan(m[g], top), f = exp2_of(m[g], mn), p = exp2_of(x, mn);
      m[g] = mn;
      l[g] = l[g] * f + (half ? 0.f : p);
      if (!half) ps[g * kRows + t] = p;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[g][c] *= f;
    }
    __syncwarp();
    const float* val = reinterpret_cast<const float*>(stage + kRows * S::kPitch);
#pragma unroll 4
    for (int t4 = 0; t4 < kRows; t4 += 4) {
      float v[4][kCols];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < kCols; ++c) v[r][c] = val[(t4 + r) * (S::kPitch / 4) + lane + 32 * c];
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
      for (int c = 0; c < kCols; ++c) to[(g * kCols + c) * 32 + lane] = o[g][c];
      if (lane == 0) {
        to[S::kOut * 32 + g] = m[g];
        to[S::kOut * 32 + 8 + g] = l[g];
      }
    }
  }
  __device__ __forceinline__ void take(const float* from) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const float om = from[S::kOut * 32 + g], ol = from[S::kOut * 32 + 8 + g];
      const float mn = max_nan(m[g], om), f = exp2_of(m[g], mn), of = exp2_of(om, mn);
      m[g] = mn;
      l[g] = l[g] * f + ol * of;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[g][c] = o[g][c] * f + from[(g * kCols + c) * 32 + lane] * of;
    }
  }
  __device__ __forceinline__ void write(const Args& a, const Place& p, int) const {
    const int lane = threadIdx.x & 31;
    const int kv = p.unit / a.units_per_kv, h0 = (p.unit % a.units_per_kv) * a.unit_heads;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g >= a.unit_heads || h0 + g >= a.group) continue;
      const float inv = l[g] > 0.f || l[g] != l[g] ? 1.f / l[g] : 0.f;
      float* out = reinterpret_cast<float*>(a.out) + ((int64_t)p.req * a.heads + kv * a.group + h0 + g) * a.d;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        if (lane + 32 * c < a.d) out[lane + 32 * c] = o[g][c] * inv;
    }
  }
  __device__ __forceinline__ void leave(const Args& a, float* part, int) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g >= a.unit_heads) continue;
      float* to = part + (int64_t)g * (a.d + 2);
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        if (lane + 32 * c < a.d) to[lane + 32 * c] = o[g][c];
      if (lane == 0) {
        to[a.d] = m[g];
        to[a.d + 1] = l[g];
      }
    }
  }
};

// MT: groups of 8 query heads in a unit; warp w has group w % MT of the tokens of share w / MT of a tile
template <typename T, int DP, int MT>
__global__ void __launch_bounds__(Shape<T, DP>::kWarps * 32, 1)
attention_kernel(const Args a) {
  using S = Shape<T, DP>;
  constexpr int kWarps = S::kWarps, kShares = kWarps / MT;
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + S::kStages * kWarps * S::kStage);
  float* qs = merge + S::kMerge / 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* ps = qs + 8 * DP + warp * 8 * kRows;
  const int m_tile = warp % MT, share = warp / MT;
  const int units = a.kv_heads * a.units_per_kv;
  if (a.d < DP) {  // features beyond D are never loaded: zeros
    const int cols = (DP - a.d) / 8, bytes = 8 * (int)sizeof(T);
    for (int i = threadIdx.x; i < S::kStages * kWarps * 2 * kRows * cols; i += kWarps * 32) {
      uint4* at = reinterpret_cast<uint4*>(smem + i / cols * S::kPitch + (a.d / 8 + i % cols) * bytes);
      for (int b = 0; b < bytes / 16; ++b) at[b] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  rb_pdl_wait();
  rb_pdl_launch();

  // this CTA's stretch of the list: prefix sums over the requests, a run of them per thread
  __shared__ long long warp_sums[kWarps];
  __shared__ Place start_shared;
  __shared__ uint32_t there[S::kStages][kWarps];
  const int run = (a.n + kWarps * 32 - 1) / (kWarps * 32);
  const int r0 = min(a.n, (int)threadIdx.x * run), r1 = min(a.n, r0 + run);
  long long mine = 0;
  for (int r = r0; r < r1; ++r) mine += (long long)tiles_of<S::kTile>(length_of(a, r)) * units;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  long long total = 0, before = inc - mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  const long long per = max((total + a.grid - 1) / a.grid, 1LL);
  const long long first = per * blockIdx.x, last = min(total, first + per);
  if (first >= last) return;
  if (before <= first && first < before + mine) {
    for (int r = r0; r < r1; ++r) {
      const int len = length_of(a, r), tiles = tiles_of<S::kTile>(len);
      const long long all = (long long)tiles * units;
      if (first < before + all) {
        const long long in = first - before;
        start_shared = Place{r, (int)(in / tiles), (int)(in % tiles), tiles, len};
        break;
      }
      before += all;
    }
  }
  __syncthreads();
  Place load = start_shared, cur = start_shared;
  const int n_tiles = (int)(last - first);

  const uint32_t stages = smem_of(smem);
  auto stage_of = [&](int i, int w) { return stages + (uint32_t)((i % S::kStages) * kWarps + w) * S::kStage; };
  int loaded = 0;
  auto load_next = [&]() {
    if (loaded < n_tiles) {
      load_tile<T, DP>(a, load, stage_of(loaded, warp), warp, &there[loaded % S::kStages][warp]);
      next<S::kTile>(a, load, units);
      ++loaded;
    }
    commit();
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) load_next();

  State<T, DP> st;
  bool fresh = true, whole = false;
  long long g0 = first - cur.tile;  // number of the first tile of the (request, unit) in the list
#pragma unroll 1
  for (int i = 0; i < n_tiles; ++i) {
    wait_for<S::kStages - 2>();
    if (MT == 1) __syncwarp();
    else __syncthreads();  // all warps' tokens are there, and all have left the tile before
    load_next();
    if (fresh) {
      st.begin(a, cur, m_tile, qs);
      whole = cur.tile == 0;
      fresh = false;
    }
    constexpr int kMine = kWarps / kShares;  // parts of 16 tokens that are this warp's: the same number as the groups of heads
#pragma unroll 1
    for (int s = 0; s < kMine; ++s) {
      const int w = share * kMine + s;
      const int64_t t0 = (int64_t)cur.tile * S::kTile + w * kRows;
      if (t0 >= cur.len) break;
      st.add(a, stage_of(i, w), there[i % S::kStages][w], qs, ps);
    }
    if (MT == 1) __syncwarp();
    const bool ends = cur.tile + 1 == cur.tiles;
    if (ends || i + 1 == n_tiles) {
      st.finish();
#pragma unroll
      for (int half = kShares / 2; half >= 1; half >>= 1) {
        __syncthreads();
        float* box = merge + ((share % half) * MT + m_tile) * (S::kOut * 32 + 16);
        if (share >= half && share < 2 * half) st.give(box);
        __syncthreads();
        if (share < half) st.take(box);
      }
      const int64_t at = (int64_t)cur.req * units + cur.unit;
      if (share == 0) {
        if (ends && whole) st.write(a, cur, m_tile);
        else st.leave(a, a.part + ((int64_t)blockIdx.x * 2 + (whole ? 1 : 0)) * a.unit_heads * (a.d + 2), m_tile);
      }
      if (whole && threadIdx.x == 0) a.owners[at] = make_int2((int)blockIdx.x, (int)((g0 + cur.tiles - 1) / per));
      fresh = true;
      g0 += cur.tiles;
    }
    next<S::kTile>(a, cur, units);
  }
  wait_for<0>();
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
  const int64_t pitch = (int64_t)a.unit_heads * (a.d + 2);
  // the first CTA's part is its last stretch (place 1), the others' their first (place 0)
  auto part = [&](int c) { return a.part + ((int64_t)c * 2 + (c == own.x ? 1 : 0)) * pitch + (int64_t)row * (a.d + 2); };
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
int launch(const Args& a, cudaStream_t stream) {
  using S = Shape<T, DP>;
  static_assert(S::kStages >= 2 && S::kSmem <= 226 * 1024, "shared memory");
  static RbPerDevice ready;
  auto kernel = attention_kernel<T, DP, MT>;
  if (ready.needed()) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess) return rb_check_launch("paged_attention");
    ready.done();
  }
  rb_launch_pdl(kernel, dim3(a.grid), dim3(S::kWarps * 32), (size_t)S::kSmem, stream, a);
  rb_launch_pdl(join_kernel<T>, dim3((unsigned)(((int64_t)a.n * a.heads + 3) / 4)), dim3(128), 0, stream, a, a.kv_heads * a.units_per_kv);
  return rb_check_launch("paged_attention");
}

template <typename T, int MT>
int by_dim(const Args& a, cudaStream_t stream) {
  if (a.d <= 32) return launch<T, 32, MT>(a, stream);
  if (a.d <= 64) return launch<T, 64, MT>(a, stream);
  if (a.d <= 96) return launch<T, 96, MT>(a, stream);
  if (a.d <= 128) return launch<T, 128, MT>(a, stream);
  return launch<T, 256, MT>(a, stream);
}

constexpr int kGrid = 148;

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
  return (long long)kGrid * 2 * uh * (d + 2) * 4 + (long long)n * units * 8;
}

// q [n, heads, D]; k, v [pages, kv heads, page, D]; table [n][blocks] rows table_stride apart; out [n, heads, D] contiguous; strides: q request, head; k, v: page, head,
// token. Features have unit stride; caches start on 16 bytes and their strides are multiples of 16 bytes.
RB_EXPORT int rb200_paged_attention(const void* q, const void* k, const void* v, const int* table, long long table_stride, const int* lens, void* out,
                                    void* workspace, const long long* strides, int n, int heads, int kv_heads, int d, int page, int blocks, int num_pages, float scale,
                                    int bf16, cudaStream_t stream) {
  if (n <= 0 || heads <= 0) return RB_OK;
  const int unit = bf16 ? 8 : 4;
  bool ok = d >= 8 && d <= 256 && d % 8 == 0 && kv_heads >= 1 && heads % kv_heads == 0 && page >= 1 && blocks >= 0 && num_pages >= 0;
  for (int i = 2; i < 8; ++i) ok = ok && strides[i] % unit == 0;
  ok = ok && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  if (!ok) {
    rb_set_error("paged_attention: head dim %d (a multiple of 8 up to 256), %d query heads over %d, page size %d, caches on 16 bytes", d, heads, kv_heads, page);
    return RB_ERR_UNSUPPORTED;
  }
  Args a = {};
  a.q = q; a.k = k; a.v = v; a.table = table; a.lens = lens; a.out = out; a.table_stride = table_stride;
  a.q_req = strides[0]; a.q_head = strides[1]; a.kp = strides[2]; a.kh = strides[3]; a.kt = strides[4]; a.vp = strides[5]; a.vh = strides[6]; a.vt = strides[7];
  a.n = n; a.heads = heads; a.kv_heads = kv_heads; a.d = d; a.page = page; a.blocks = blocks; a.num_pages = num_pages; a.group = heads / kv_heads;
  a.units_per_kv = units_of(a.group, bf16, &a.unit_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.grid = kGrid;
  a.part = reinterpret_cast<float*>(workspace);
  a.owners = reinterpret_cast<int2*>(a.part + (int64_t)kGrid * 2 * a.unit_heads * (d + 2));
  if (!bf16) return by_dim<float, 1>(a, stream);
  if (a.unit_heads <= 8) return by_dim<__nv_bfloat16, 1>(a, stream);
  if (a.unit_heads <= 16) return by_dim<__nv_bfloat16, 2>(a, stream);
  return by_dim<__nv_bfloat16, 4>(a, stream);
}
