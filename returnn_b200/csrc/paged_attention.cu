// Attention of one new token per request over a paged key / value cache.
//   out[i, h, :] = softmax_t(scale q[i, h, :] . K[t, h / G, :]) V[t, h / G, :],  t < len_i; token t lies in page table[i][t / P] at place t % P
// G = query heads per key head. A request without tokens gets zeros. Keys and values are read once for every 32 (bf16) or 8 (fp32) query heads of their key head; with up to
// that many in bf16, and up to 4 in fp32, the pass is bound by that where requests are long.
//
// Split: the work is a list of tiles, ordered by (request, group of units, tile); each CTA takes an equally costly stretch of the list, whatever the lengths
// of the requests are (a long document next to short ones, few requests of many tokens). A stretch that holds all tiles of a (request, group)
// writes the result; one that holds some of them leaves its maximum, sum and unnormalised output in 32 bits, and a second small kernel joins those.
// A unit is a key head with up to 8 * MT of its query heads. A tile is the parts of 16 tokens of the multiplying warps: of one unit, or of fewer tokens of 2, 4 or 8
// units where there are enough requests. Warps of one unit bring their outputs together at its end; with a unit for each warp there is nothing to bring
// together, and requests of a few tokens fill the warps (see group_of).
// Within a CTA four or eight warps look the pages up and send for them, several tiles ahead, also across the end of a (request, unit); the others multiply, 16 tokens of a
// tile each, which are waited for and refilled by themselves. Rows beyond the length are filled with zeros and not read. The copies are the 16-byte
// asynchronous ones of the loading warps' lanes, which take any page size and any strides: boxes of 16 tokens x 128 bytes by TMA were issued and fetched at
// 5.0 to 5.9 TB/s without any product behind them, and boxes cannot be larger where a page holds 16 tokens.
// What a warp keeps per query head are the running maximum, sum and output in registers.
// bf16: products by warp-level matrix instructions (16 x 8 x 16). A decoding step has 1 to 32 rows per key head and is bound by memory: the
// larger tensor-memory instructions have nothing to win (64 rows at least, keys would pass through descriptors) and the sixteen rows here are only half used:
// rows 0..7 are 8 query heads with the upper 16 bits of the weights, rows 8..15 the same heads with what is left of them in bf16. Their sum weighs the
// values with 16 bits of mantissa at no further instruction; weights of 8 bits would add an error as large as the rounding of the result.
// fp32: products by fused multiply-adds, a kernel for 1, 2, 4 and 8 heads of a unit (14 requests, 56340 tokens, D 128, 4 on each of 8 key heads: 88 us; with one kernel and the heads
// counted at run time 169). With 8 or more heads on a key head it is latency that sets the pace: 16 on one of 128, 14 x 4024 tokens, 45 us where one read of the cache takes 9 and
// the multiply-adds 6; 32 % of the issue slots, 18 % of the multiply-add units' and 30 % of the shared memory's rate are in use, with 12 warps on an SM.
// Measured (D 128, 4 query heads on each of 8 key heads, bf16): 64 requests of 122637 tokens together, 502 MB, 84 us (6.0 TB/s); two of 76484 and 131072, 850 MB, 132 us
// (6.4 TB/s). Small calls are at present two launches and a chain of length, page, token, product and join: one request of 1000 tokens, fp32, D 64, 8.2 us.
#include "packed_f32.cuh"
#include "tcgen05.cuh"
#include <algorithm>

namespace {

using namespace rbt;

constexpr int kJoin = 8;  // warps of a block that joins parts

struct Args {
  const void *q, *k, *v;
  const int *table, *lens;
  void* out;
  float* part;   // [grid][2][units of a group][unit heads][D + 4]: output, maximum (log2), sum
  int4* cuts;    // [grid]: the (request, group) that a CTA begins and others end, and the last of them; -1 if none
  int* status;
  int64_t q_req, q_head, kp, kh, kt, vp, vh, vt, table_stride;
  int n, heads, kv_heads, d, page, blocks, num_pages, group, units_per_kv, unit_heads, grid;
  int units, groups;  // units of a group (1, 2, 4 or 8), groups of a request
  int tile_shift;     // log2 of the tokens of a tile
  int group_cost;     // of beginning and ending a (request, group), in tiles: queries, the meeting of the warps, the result
  int q_words;  // queries can be read two features at a time
  int whole;  // 16 tokens from a multiple of 16 on lie in one page, and rows are as wide as in shared memory
  float scale_log2;
};

// H: query heads that a multiplying warp computes (bf16: the 8 of a product)
template <typename T, int DP, int H>
struct Shape {
  static constexpr bool kBf16 = sizeof(T) == 2;
  static constexpr int kRowBytes = DP * (int)sizeof(T);
  static constexpr int kRows = kRowBytes <= (kBf16 ? 512 : 256) ? 16 : 8;  // tokens of a part
  static constexpr int kPart = kRows * kRowBytes;          // blocks of kRows rows of 128 bytes, 16-byte pieces swizzled by the row
  static constexpr int kWarps = kRows * kRowBytes <= 4096 ? 8 : 4;
  static constexpr int kStage = 2 * kWarps * kPart;  // keys, values
  static constexpr int kPitch = DP + 8;              // floats of a head where the warps meet (no bank conflicts)
  static constexpr int kMeet = H * (kPitch + 2) + 7 & ~7;  // of a warp: outputs, maxima, sums; fp32: the queries before
  static constexpr int kFloats = kWarps * (kMeet + (kBf16 ? 0 : 2 * H * kRows));  // and fp32: weights of a part, each twice
  // loading warps: what they issue sets the pace of rows of 128 bytes with one group of heads (28 requests, 112680 tokens, 12 heads of 64, bf16: 68.4 us with four, 64.2 with eight; 64 over
  // 4 heads 33.5 and 36.1) and of four heads over parts of 8 rows (32 over 8 heads of 128, fp32: 165 and 152). Elsewhere four are enough and leave the registers
  // (32 over 8 of 128, bf16: 73.5 and 76.6).
  static constexpr int loaders(int mt) { return (kBf16 && kRowBytes == 128 && mt == 1) || (!kBf16 && kRowBytes == 512 && H == 4) ? 8 : std::min(4, kWarps); }
  static constexpr int threads(int mt) { return (kWarps + loaders(mt)) * 32; }
  static constexpr int kStages = std::min(6, (int)((227 * 1024 - 1024 - 1536 - kFloats * 4) / kStage));
  static constexpr int kSmem = kStages * kStage + kFloats * 4 + 1024;
};

struct Place {  // in the list of tiles
  int req, group, tile, tiles, len;  // tiles: of the request, in each group
};

__device__ __forceinline__ int length_of(const Args& a, int req) { return (int)min((int64_t)max(a.lens[req], 0), (int64_t)a.blocks * a.page); }
__device__ __forceinline__ int tiles_of(const Args& a, int len) { return (int)(((int64_t)len + (1 << a.tile_shift) - 1) >> a.tile_shift); }

// first tile of the next (request, group)
__device__ __forceinline__ void next_group(const Args& a, Place& p) {
  p.tile = 0;
  if (++p.group < a.groups) return;
  p.group = 0;
  do {
    if (++p.req >= a.n) {
      p.tiles = p.len = 0;
      return;
    }
    p.len = length_of(a, p.req);
    p.tiles = tiles_of(a, p.len);
  } while (p.tiles == 0);
}

struct Heads {  // of a unit: key head, first query head
  int kv, first, count;
  __device__ __forceinline__ Heads(const Args& a, int unit) {
    kv = a.units_per_kv == 1 ? unit : unit / a.units_per_kv;
    const int h0 = (unit - kv * a.units_per_kv) * a.unit_heads;
    first = kv * a.group + h0;
    count = min(a.unit_heads, a.group - h0);
  }
};

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
template <typename T, int DP, int H>
struct State;

template <int DP>
struct State<__nv_bfloat16, DP, 8> {
  using T = __nv_bfloat16;
  using S = Shape<T, DP, 8>;
  static constexpr int kRows = S::kRows;
  static constexpr int kSteps = DP / 16, kTiles = DP / 8;
  uint32_t q[kSteps][2];
  float o[kTiles][4];
  float m, l;  // l: of this lane's columns

  __device__ __forceinline__ void fetch_queries(const Args& a, int req, int unit, int m_tile) {
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const Heads of(a, unit);
    const bool real = m_tile * 8 + g < of.count;
    const T* src = reinterpret_cast<const T*>(a.q) + req * a.q_req + (real ? (int64_t)(of.first + m_tile * 8 + g) * a.q_head : 0);
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
      // the upper half of a weight as it stands, and what is left, which is then above zero: an infinite value has to meet two weights of one sign (2^-126 of the values is
      // added where nothing is left)
      hi[c] = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
      const __nv_bfloat162 rest = __floats2bfloat162_rn(p0 - __uint_as_float(hi[c] << 16), p1 - __uint_as_float(hi[c] & 0xffff0000u)),
                           least = __halves2bfloat162(__ushort_as_bfloat16(0x0080), __ushort_as_bfloat16(0x0080));
      const __nv_bfloat162 r = __hmax2(rest, least);
      lo[c] = *reinterpret_cast<const uint32_t*>(&r);
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

// fp32: 32 / kRows lanes share a token's score (groups of four features in turn); lane has features 2 lane, 2 lane + 1, 2 lane + 64, ... of the output of every head.
// Multiply-adds are packed, two features at a time.
template <int DP, int H>
struct State<float, DP, H> {
  using S = Shape<float, DP, H>;
  static constexpr int kRows = S::kRows, kSplit = 32 / kRows, kPairs = DP / 64;
  uint64_t o[H][kPairs];
  float m[H], l[H];  // l: of this lane's token
  float q[H][DP / 32];

  __device__ __forceinline__ void fetch_queries(const Args& a, int req, int unit, int) {
    const int lane = threadIdx.x & 31;
    const Heads of(a, unit);
    const float* src = reinterpret_cast<const float*>(a.q) + req * a.q_req + (int64_t)of.first * a.q_head + lane;
#pragma unroll
    for (int g = 0; g < H; ++g)
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) q[g][c] = g < of.count && lane + 32 * c < a.d ? src[g * a.q_head + 32 * c] * a.scale_log2 : 0.f;
  }
  __device__ __forceinline__ void share_queries(float* qs) const {  // in the warp
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < H; ++g)
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) qs[g * DP + c * 32 + lane] = q[g][c];
    __syncwarp();
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int g = 0; g < H; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int c = 0; c < kPairs; ++c) o[g][c] = 0;
    }
  }
  __device__ __forceinline__ static void at(uint32_t from, uint64_t& x, uint64_t& y) {
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(x), "=l"(y) : "r"(from) : "memory");
  }
  __device__ __forceinline__ static uint64_t pair_at(uint32_t from) {
    uint64_t r;
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(r) : "r"(from) : "memory");
    return r;
  }
  __device__ __forceinline__ void add(const Args& a, uint32_t keys, uint32_t vals, uint32_t bits, const float* qs, float* ps) {
    const int lane = threadIdx.x & 31, t = lane & (kRows - 1), part = lane / kRows;
    uint64_t s[H][2] = {};
    const uint32_t qa = smem_u32(qs), pa = smem_u32(ps);
#pragma unroll 4
    for (int c = part; c < DP / 4; c += kSplit) {  // pieces of four features
      uint64_t k0, k1;
      at(keys + (c >> 3) * (kRows * 128) + t * 128 + (((c & 7) ^ (t & 7)) << 4), k0, k1);
#pragma unroll
      for (int g = 0; g < H; ++g) {
        uint64_t q0, q1;
        at(qa + (g * DP + c * 4) * 4, q0, q1);
        s[g][0] = fma2(k0, q0, s[g][0]);
        s[g][1] = fma2(k1, q1, s[g][1]);
      }
    }
    const bool there = bits >> t & 1;
    float x[H], top[H], f[H];
#pragma unroll
    for (int g = 0; g < H; ++g) {
      float x0, x1;
      split(add2(s[g][0], s[g][1]), x0, x1);
      x[g] = x0 + x1;
    }
#pragma unroll
    for (int w = kRows; w < 32; w <<= 1)
#pragma unroll
      for (int g = 0; g < H; ++g) x[g] += __shfl_xor_sync(0xffffffffu, x[g], w);
#pragma unroll
    for (int g = 0; g < H; ++g) top[g] = x[g] = there ? x[g] : -INFINITY;
#pragma unroll
    for (int w = 1; w < kRows; w <<= 1)
#pragma unroll
      for (int g = 0; g < H; ++g) top[g] = max_nan(top[g], __shfl_xor_sync(0xffffffffu, top[g], w));
    bool more = false;
#pragma unroll
    for (int g = 0; g < H; ++g) {
      const float mn = max_nan(m[g], top[g]), p = exp2_of(x[g], mn);
      f[g] = exp2_of(m[g], mn);
      more |= f[g] != 1.f;
      m[g] = mn;
      l[g] = l[g] * f[g] + (part ? 0.f : p);
      if (!part) *reinterpret_cast<float2*>(ps + (g * kRows + t) * 2) = make_float2(p, p);
    }
    if (more) {  // (the same in all lanes)
#pragma unroll
      for (int g = 0; g < H; ++g)
#pragma unroll
        for (int c = 0; c < kPairs; ++c) o[g][c] = mul2(o[g][c], two(f[g], f[g]));
    }
    __syncwarp();
#pragma unroll
    for (int t4 = 0; t4 < kRows; t4 += 4) {
      uint64_t v[4][kPairs];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < kPairs; ++c) {
          const int e = 64 * c + 2 * lane;
          v[r][c] = pair_at(vals + (e >> 5) * (kRows * 128) + (t4 + r) * 128 + (((e >> 2 & 7) ^ ((t4 + r) & 7)) << 4) + (e & 3) * 4);
        }
#pragma unroll
      for (int g = 0; g < H; ++g) {
        uint64_t p[4];
        at(pa + (g * kRows + t4) * 8, p[0], p[1]);
        at(pa + (g * kRows + t4 + 2) * 8, p[2], p[3]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < kPairs; ++c) o[g][c] = fma2(p[r], v[r][c], o[g][c]);
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int g = 0; g < H; ++g) l[g] = warp_sum(l[g]);
  }
  __device__ __forceinline__ void give(float* to) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < H; ++g) {
#pragma unroll
      for (int c = 0; c < kPairs; ++c) *reinterpret_cast<uint64_t*>(to + g * S::kPitch + 64 * c + 2 * lane) = o[g][c];
      if (lane == 0) {
        to[H * S::kPitch + g] = m[g];
        to[H * S::kPitch + H + g] = l[g];
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

// MT: groups of H query heads in a unit. Multiplying warp (share, unit, m) has group m of the heads of a unit and MT parts of its tokens in a tile; the parts of a stage are
// ordered by unit and tokens
template <typename T, int DP, int MT, int H>
__global__ void __launch_bounds__(Shape<T, DP, H>::threads(MT), 1)
attention_kernel(const Args a) {
  using S = Shape<T, DP, H>;
  constexpr int kWarps = S::kWarps, kStages = S::kStages, kLoaders = S::loaders(MT), kRows = S::kRows;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  float* boxes = reinterpret_cast<float*>(smem + kStages * S::kStage);
  __shared__ uint64_t full[kStages][kWarps], empty[kStages][kWarps], meeting;
  __shared__ uint32_t notes[kStages][kWarps];  // of a part: the tokens that there are as bits; bit 16: some lie within the length
  __shared__ long long warp_sums[kWarps + kLoaders][2], rank_shared[2], cost_shared;
  __shared__ Place start_shared;
  __shared__ int abort_shared;
  volatile int* abort = &abort_shared;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token_parts = kWarps / a.units;  // of a unit in a tile
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
  // beginning of a (request, group) stand for its first tile.
  const int run = (a.n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int r0 = min((int64_t)a.n, (int64_t)threadIdx.x * run), r1 = min(a.n, r0 + run);
  auto cost_of = [&](int tiles) { return tiles ? (long long)(tiles + a.group_cost) * a.groups : 0LL; };
  long long mine = 0, mine_tiles = 0;
  for (int r = r0; r < r1; ++r) {
    const int tiles = tiles_of(a, length_of(a, r));
    mine += cost_of(tiles);
    mine_tiles += (long long)tiles * a.groups;
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
  if (threadIdx.x < kWarps * 32) {  // zeros of requests without tokens
    for (int r = blockIdx.x; r < a.n; r += a.grid) {
      if (length_of(a, r)) continue;
      T* out = reinterpret_cast<T*>(a.out) + (int64_t)r * a.heads * a.d;
      for (int e = threadIdx.x * 4; e < a.heads * a.d; e += kWarps * 128) put4(out + e, make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
  if (first >= last) {
    if (threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(0, 0, -1, 0);
    return;
  }
  if (threadIdx.x == 0 && last == total) rank_shared[1] = total_tiles;
  for (int end = 0; end < 2; ++end) {
    const long long want = end ? last : first;
    if (!(before <= want && want < before + mine)) continue;
    long long c = before, k = before_tiles;
    for (int r = r0; r < r1; ++r) {
      const int len = length_of(a, r), tiles = tiles_of(a, len);
      if (want < c + cost_of(tiles)) {
        const long long in = want - c;
        const int group = (int)(in / (tiles + a.group_cost)), tile = max((int)(in % (tiles + a.group_cost)) - a.group_cost, 0);
        rank_shared[end] = k + (long long)group * tiles + tile;
        if (!end) {
          start_shared = Place{r, group, tile, tiles, len};
          cost_shared = c + (long long)group * (tiles + a.group_cost);
        }
        break;
      }
      c += cost_of(tiles);
      k += (long long)tiles * a.groups;
    }
  }
  __syncthreads();
  const int n_tiles = (int)(rank_shared[1] - rank_shared[0]);
  bool ok = true;

  if (warp >= kWarps) {
    // ---- loads. Loading warp w has the parts w, w + kLoaders, ... of a tile; lane r looks the page of row r of a part up, a tile ahead
    constexpr int kMyParts = kWarps / kLoaders, kPer = 16 / (int)sizeof(T), kCopies = S::kRowBytes / 16;
    static_assert(kMyParts * kRows <= 32, "a lane per row");
    const int loader = warp - kWarps, my_part = loader + lane / kRows * kLoaders;
    const int my_unit = my_part / token_parts, my_row = (my_part & (token_parts - 1)) * kRows + lane % kRows;
    const bool mine_at_all = lane / kRows < kMyParts;
    Place p = start_shared, ahead = p;
    int pg = -1, at = 0, ahead_pg = -1, ahead_at = 0;
    auto look_up = [&]() {
      const int64_t t = ((int64_t)ahead.tile << a.tile_shift) + my_row;
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
        if (++ahead.tile == ahead.tiles) next_group(a, ahead);
        look_up();
      }
      const bool real = pg >= 0 && pg < a.num_pages;  // (no such token; or a page that is none: as if the token were not there)
      const uint32_t bits = __ballot_sync(0xffffffffu, real);
      const int64_t place = real ? at : 0, in = real ? pg : 0;
      const int unit = p.group * a.units + my_unit, kv = a.units_per_kv == 1 ? unit : unit / a.units_per_kv;
      const int64_t k_row = (int64_t)a.k + (int64_t)sizeof(T) * (in * a.kp + kv * a.kh + place * a.kt);
      const int64_t v_row = (int64_t)a.v + (int64_t)sizeof(T) * (in * a.vp + kv * a.vh + place * a.vt);
#pragma unroll
      for (int j = 0; j < kMyParts; ++j) {
        const int part = loader + j * kLoaders;
        if (round > 0) ok = ok && warp_wait(&empty[s][part], (round - 1) & 1, abort);
        if (!ok) break;
        const uint32_t to = smem_u32(smem) + s * S::kStage + part * S::kPart;
        const uint32_t mine = bits >> (kRows * j) & ((1u << kRows) - 1u);
        if (kCopies <= 32 && a.whole && mine == (1u << kRows) - 1u) {  // tokens of one page: rows at a fixed distance
          const int row0 = lane / kCopies, c = lane % kCopies;
          int64_t kr = __shfl_sync(0xffffffffu, k_row, kRows * j) + row0 * a.kt * (int64_t)sizeof(T) + c * 16;
          int64_t vr = __shfl_sync(0xffffffffu, v_row, kRows * j) + row0 * a.vt * (int64_t)sizeof(T) + c * 16;
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
          const int64_t kr = __shfl_sync(0xffffffffu, k_row, kRows * j + row), vr = __shfl_sync(0xffffffffu, v_row, kRows * j + row);
          const bool there = (mine >> row & 1) && (S::kRowBytes == a.d * (int)sizeof(T) || c * kPer < a.d);  // (features beyond D: zeros)
          const uint32_t dst = to + (c >> 3) * (kRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
          copy16(dst, reinterpret_cast<const void*>(kr + (there ? c * 16 : 0)), there);
          copy16(dst + kWarps * S::kPart, reinterpret_cast<const void*>(vr + (there ? c * 16 : 0)), there);
        }
        }
        arrive_copied(&full[s][part]);
        if (lane == 0) {
          const int64_t t0 = ((int64_t)p.tile << a.tile_shift) + (part & (token_parts - 1)) * kRows;
          notes[s][part] = mine | (t0 < p.len ? 1u << 16 : 0u);
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
  const int m_tile = warp % MT, slot = warp / MT, shares = token_parts / MT, my_unit = slot % a.units, share = slot / a.units;
  float* box = boxes + warp * S::kMeet;  // of (share, unit, m)
  float* ps = boxes + kWarps * S::kMeet + warp * 2 * H * kRows;
  const uint32_t stages = smem_u32(smem);
  int meetings = 0;
  auto meet = [&]() {  // of the multiplying warps, where some have the same unit
    __syncwarp();
    if (shares == 1) return;
    if (lane == 0) arrive(&meeting);
    ok = warp_wait(&meeting, meetings++ & 1, abort);
  };
  State<T, DP, H> st;
  Place cur = start_shared;
  long long cost = cost_shared;  // where the present (request, group) begins
  st.fetch_queries(a, cur.req, cur.group * a.units + my_unit, m_tile);
  int4 cut_here = make_int4(0, 0, -1, 0);
  int n = 0, s = 0, round = 0;
#pragma unroll 1
  while (n < n_tiles) {
    const int count = min(cur.tiles - cur.tile, n_tiles - n);
    if constexpr (!S::kBf16) {
      meet();  // all have read what was in the boxes
      if (!ok) break;
      st.share_queries(box);
    }
    st.begin();
#pragma unroll 1
    for (int t = 0; t < count && ok; ++t) {
#pragma unroll 1
      for (int i = 0; i < MT; ++i) {
        const int w = my_unit * token_parts + share * MT + i;
        ok = warp_wait(&full[s][w], round & 1, abort);
        if (!ok) break;
        const uint32_t word = notes[s][w];
        if (word >> 16) {
          const uint32_t keys = stages + s * S::kStage + w * S::kPart;
          st.add(a, keys, keys + kWarps * S::kPart, word & 0xffffu, box, ps);
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
    if (n < n_tiles) {  // the next queries are under way while the outputs come together
      next_group(a, cur);
      st.fetch_queries(a, cur.req, cur.group * a.units + my_unit, m_tile);
    }
    // ---- the outputs of a unit come together; a warp that has its unit alone writes it
    st.finish();
    if constexpr (S::kBf16) {
      meet();  // all have read what was in the boxes
      if (!ok) break;
    }
    st.give(box);
    meet();
    if (!ok) break;
    const int of = H * (DP / 4), all = shares == 1 ? of : of * MT * a.units;
    for (int i = shares == 1 ? lane : threadIdx.x; i < all; i += shares == 1 ? 32 : kWarps * 32) {
      const int e = i % (DP / 4) * 4, g = i / (DP / 4) % H;
      int mt = m_tile, un = my_unit;
      if (shares != 1) {
        mt = i / of % MT;
        un = i / of / MT;
      }
      const int h = mt * H + g;
      const Heads of_unit(a, done.group * a.units + un);
      if (e >= a.d || h >= of_unit.count) continue;
      const float* b = boxes + (un * MT + mt) * S::kMeet;
      const int pitch = a.units * MT * S::kMeet;  // to the next share
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps / MT; ++w) {
        if (w < shares) m = max_nan(m, b[w * pitch + H * S::kPitch + g]);
      }
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps / MT; ++w) {
        if (w >= shares) break;
        const float f = exp2_of(b[w * pitch + H * S::kPitch + g], m);
        const float4 x = *reinterpret_cast<const float4*>(b + w * pitch + g * S::kPitch + e);
        l += b[w * pitch + H * S::kPitch + H + g] * f;
        o.x += x.x * f;
        o.y += x.y * f;
        o.z += x.z * f;
        o.w += x.w * f;
      }
      if (ends && whole) {
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        put4(reinterpret_cast<T*>(a.out) + ((int64_t)done.req * a.heads + of_unit.first + h) * a.d + e, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      } else {
        float* to = a.part + ((((int64_t)blockIdx.x * 2 + (whole ? 1 : 0)) * a.units + un) * a.unit_heads + h) * (a.d + 4);
        *reinterpret_cast<float4*>(to + e) = o;
        if (e == 0) *reinterpret_cast<float2*>(to + a.d) = make_float2(m, l);
      }
    }
    if (shares == 1) __syncwarp();
    if (whole && !ends) cut_here = make_int4(done.req, done.group, (int)((cost + a.group_cost + done.tiles - 1) / per), 0);
    cost += done.tiles + a.group_cost;
  }
  if (threadIdx.x == 0) a.cuts[blockIdx.x] = cut_here;
  if (!ok) {
    *abort = 1;
    if (lane == 0 && a.status) atomicCAS(a.status, 0, (9 << 24) | 2);
  }
}

// joins the parts of a (request, group) that several CTAs had: block (c, y) the one that CTA c began (two requests of 5615 tokens, two units: 14 us with the pass; a thread
// per feature, part after part, took 27). A warp per query head: its lanes weigh a part each, then take
// four features each of all parts, several under way at a time.
template <typename T>
__global__ void __launch_bounds__(kJoin * 32)
join_kernel(const Args a) {
  const int lane = threadIdx.x & 31, began = blockIdx.x;
  const int w = blockIdx.y * kJoin + (threadIdx.x >> 5), in = w / a.unit_heads, row = w - in * a.unit_heads;
  rb_pdl_wait();
  rb_pdl_launch();
  const int4 cut = a.cuts[began];
  if (cut.z < 0 || in >= a.units) return;
  const Heads of(a, cut.y * a.units + in);
  if (row >= of.count) return;
  T* out = reinterpret_cast<T*>(a.out) + ((int64_t)cut.x * a.heads + of.first + row) * a.d;
  const int64_t pitch = (int64_t)a.units * a.unit_heads * (a.d + 4);
  const float* base = a.part + ((int64_t)in * a.unit_heads + row) * (a.d + 4);
  // the part of the one that began is its last stretch (place 1), the others' their first (place 0)
  auto part = [&](int c) { return base + ((int64_t)c * 2 + (c == began ? 1 : 0)) * pitch; };
  float m = -INFINITY, l = 0.f;
  float4 acc[2] = {};
  for (int c0 = began; c0 <= cut.z; c0 += 32) {
    const int count = min(32, cut.z + 1 - c0);
    constexpr int kAhead = 8;  // outputs that are under way with the maxima
    float4 ahead[kAhead];
#pragma unroll
    for (int c = 0; c < kAhead; ++c) ahead[c] = c < count && lane * 4 < a.d ? *reinterpret_cast<const float4*>(part(c0 + c) + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    float mine = -INFINITY, sum = 0.f;
    if (lane < count) {
      const float2 x = *reinterpret_cast<const float2*>(part(c0 + lane) + a.d);
      mine = x.x;
      sum = x.y;
    }
    float mn = max_nan(m, mine);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mn = max_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    const float f = lane < count ? exp2_of(mine, mn) : 0.f, old = exp2_of(m, mn);
    m = mn;
    l = l * old + warp_sum(sum * f);
#pragma unroll
    for (int k = 0; k < 2; ++k) acc[k] = make_float4(acc[k].x * old, acc[k].y * old, acc[k].z * old, acc[k].w * old);
    auto weigh = [&](float4& to, const float4& x, float by) {
      to.x += x.x * by;
      to.y += x.y * by;
      to.z += x.z * by;
      to.w += x.w * by;
    };
#pragma unroll
    for (int c = 0; c < kAhead; ++c)
      if (c < count) weigh(acc[0], ahead[c], __shfl_sync(0xffffffffu, f, c));
#pragma unroll 8
    for (int c = kAhead; c < count; ++c) {
      const float fc = __shfl_sync(0xffffffffu, f, c);
      if (lane * 4 < a.d) weigh(acc[0], *reinterpret_cast<const float4*>(part(c0 + c) + lane * 4), fc);
    }
    if (a.d > 128) {
#pragma unroll 8
      for (int c = 0; c < count; ++c) {
        const float fc = __shfl_sync(0xffffffffu, f, c);
        if (lane * 4 + 128 < a.d) weigh(acc[1], *reinterpret_cast<const float4*>(part(c0 + c) + lane * 4 + 128), fc);
      }
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int e = (lane + 32 * k) * 4;
    if (e < a.d) put4(out + e, make_float4(acc[k].x * inv, acc[k].y * inv, acc[k].z * inv, acc[k].w * inv));
  }
}

template <typename T, int DP, int MT, int H>
int launch(Args a, cudaStream_t stream) {
  using S = Shape<T, DP, H>;
  a.whole = a.page % S::kRows == 0 && a.d == DP;
  const int slots = S::kWarps / MT;
  a.units = std::min(a.units, slots);
  a.groups = a.kv_heads * a.units_per_kv / a.units;
  a.tile_shift = __builtin_ctz(S::kWarps / a.units * S::kRows);
  a.group_cost = a.units == slots ? 1 : 2;
  static_assert(S::kStages >= 2 && S::kSmem + 1536 <= 227 * 1024, "shared memory");
  static RbPerDevice ready;
  auto kernel = attention_kernel<T, DP, MT, H>;
  if (ready.needed()) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess) return rb_check_launch("paged_attention");
    ready.done();
  }
  rb_launch_pdl(kernel, dim3(a.grid), dim3(S::threads(MT)), (size_t)S::kSmem, stream, a);
  rb_launch_pdl(join_kernel<T>, dim3(a.grid, (a.units * a.unit_heads + kJoin - 1) / kJoin), dim3(kJoin * 32), 0, stream, a);
  return rb_check_launch("paged_attention");
}

template <typename T, int MT, int H>
int by_dim(const Args& a, cudaStream_t stream) {
  if (a.d <= 64) return launch<T, 64, MT, H>(a, stream);
  if (a.d <= 128) return launch<T, 128, MT, H>(a, stream);
  return launch<T, 256, MT, H>(a, stream);
}

int units_of(int group, int bf16, int* unit_heads) {
  const int most = bf16 ? 32 : 8;
  const int units = (group + most - 1) / most;
  *unit_heads = (group + units - 1) / units;
  return units;
}

}  // namespace

// units of a group: a power of two that divides the units, with which there is still a (request, group) for every other SM. Measured (bf16, 8 units) with 1, 2, 4 and 8:
// 378 requests of up to 11 tokens 57, 35, 24, 17 us; 64 of up to 4096 84.2, 83.7, 84.9, 85.9; 4 of up to 920 10.1, 10.7, 13.4, 15.8.
static int group_of(int n, int units) {
  int g = 1;
  while (g < 8 && units % (2 * g) == 0 && (long long)n * units / (2 * g) >= num_sms() / 2) g *= 2;
  return g;
}

// bytes of workspace for n requests: cuts and parts of the CTAs. None for shapes that are not computed
RB_EXPORT long long rb200_paged_attention_workspace(int n, int heads, int kv_heads, int d, int bf16) {
  if (n <= 0 || kv_heads <= 0 || heads < kv_heads) return 0;  // (no heads: no units to share them between)
  int uh;
  const int units = kv_heads * units_of(heads / kv_heads, bf16, &uh);
  return (long long)num_sms() * (16 + 2 * group_of(n, units) * uh * (d + 4) * 4);
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
  a.cuts = reinterpret_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(a.cuts + a.grid);
  a.units = group_of(n, kv_heads * a.units_per_kv);
  if (!bf16) {
    if (a.unit_heads == 1) return by_dim<float, 1, 1>(a, stream);
    if (a.unit_heads == 2) return by_dim<float, 1, 2>(a, stream);
    return a.unit_heads <= 4 ? by_dim<float, 1, 4>(a, stream) : by_dim<float, 1, 8>(a, stream);
  }
  if (a.unit_heads <= 8) return by_dim<__nv_bfloat16, 1, 8>(a, stream);
  if (a.unit_heads <= 16) return by_dim<__nv_bfloat16, 2, 8>(a, stream);
  return by_dim<__nv_bfloat16, 4, 8>(a, stream);
}
