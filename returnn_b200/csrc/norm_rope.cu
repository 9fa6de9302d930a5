// Norm per head and rotary positions of queries and keys in one pass, with its gradient and a form that leaves keys and values in a paged cache.
//   y = w x / sqrt(mean x^2 + eps) per (token, head) row of D features (without a norm: y = x)
//   z = c R(p f) y on the first R features, whose pairs (a, b) are (2i, 2i + 1) or (i, i + R / 2):
//       a' = c (a cos t - b sin t), b' = c (a sin t + b cos t), t = p f_i for the token's position p; the other features stay.
// Backward: dy = c R(-t) dz; with u = x / sqrt(mean x^2 + eps): dx = (dy w - u mean(dy w u)) / sqrt(mean x^2 + eps), dw = sum dy u.
//
// The angle of a far position does not fit the 24 bits of a float (position 100000 would be off by 0.004 of a radian): p f / (2 pi) is taken in 64
// bits, its whole turns dropped, and the sine and cosine of the rest taken in 32. One pair of them per (token, pair of features) serves all heads,
// so a CTA owns whole tokens and keeps the table of its tokens in shared memory.
// Rows are read once and written once. A row of D features sits in the next power of two of D / 8 lanes, 8 features a lane, chosen so that both features of a pair
// are the lane's own: 8 in a row for pairs (2i, 2i + 1), 4 of each half for pairs (i, i + R / 2). The mean is a few shuffles. Head dims, rotated parts and
// alignments that do not fit this take a warp per row with single elements.
// Measured, both passes with the norm: 25000 x 16 heads of 64, bf16, 256 MB, 62 us (4.1 TB/s; a copy of as many bytes takes 42), bound by latency: 57 to 65 % of the issue
// slots and 28 to 40 % of the memory's rate are in use, with 45 % of the warps that an SM holds; 8191 x 40 of 128, fp32, 839 MB, 138.5 us (6.1 TB/s, what the memory gives).
#include "packed_f32.cuh"
#include <algorithm>
#include <cstdlib>
#include <initializer_list>
#include <type_traits>

namespace {

constexpr int kMaxDim = 256;
constexpr int kThreads = 256;
constexpr int kTurnsBf16 = 4, kTurnsF32 = 2, kBackBf16 = 2, kBackF32 = 1;  // rows of a group that are under way at a time, forward and backward
constexpr int kCtasBf16 = 4, kCtasF32 = 4, kBackCtasBf16 = 4, kBackCtasF32 = 4;  // of an SM, forward and backward

struct Rows {        // of queries, keys or values
  const void* x;     // input; backward: of the norm (null without one)
  const void* dz;    // backward: incoming gradient
  const void* w;     // [D] scale or null
  void* out;         // [N, heads, D] or the cache
  int64_t tok, head, dz_tok, dz_head;  // strides in elements
  int64_t page, page_head, page_tok;   // of the cache
  int heads;
};

struct Args {
  Rows r[3];                        // queries, keys, values (cache form)
  const void* positions;            // [num_pos], token t has number t % num_pos
  const float* freq;                // [R / 2]
  float* part;                      // backward: [gridDim.x][2][D] partial sums of dw
  const int* slots;
  int64_t num_slots, num_pos;
  int64_t n;
  int d, rot, page, pos64, w_bf16, interleaved;
  int tokens;                       // of a CTA's tile
  int split;                        // groups that share a row's tokens where fewer rows are left than groups
  uint32_t split_inverse, half_inverse;
  float eps, amp, inv_d;
};

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t token) {
  if (a.num_pos < a.n) token %= a.num_pos;
  return a.pos64 ? reinterpret_cast<const long long*>(a.positions)[token] : reinterpret_cast<const int*>(a.positions)[token];
}
// turns per position
__device__ __forceinline__ double turns_of(const Args& a, int i) { return (double)a.freq[i] * 0.15915494309189533577; }
__device__ __forceinline__ float2 turn_of(const Args& a, int64_t position, double turns) {
  double t = (double)position * turns;
  t -= rint(t);
  float s, c;
  sincospif((float)(2.0 * t), &s, &c);
  return make_float2(c * a.amp, s * a.amp);
}
__device__ __forceinline__ float weight_at(const void* w, int i, int bf16) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]) : reinterpret_cast<const float*>(w)[i];
}
template <typename T>
__device__ __forceinline__ float one(const void* x, int64_t i) { return (float)reinterpret_cast<const T*>(x)[i]; }
template <typename T>
__device__ __forceinline__ void put(void* x, int64_t i, float v) { reinterpret_cast<T*>(x)[i] = T(v); }
template <typename T>
constexpr int is_bf16() { return sizeof(T) == 2; }

// where a token's place in the cache starts; -1: nowhere (a token without a slot)
__device__ __forceinline__ int64_t cache_at(const Args& a, const Rows& r, int64_t token) {
  const int64_t slot = a.slots[token];
  if (slot < 0 || slot >= a.num_slots) return -1;
  const int pg = (int)(slot / a.page);
  return pg * r.page + (slot - (int64_t)pg * a.page) * r.page_tok;
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
struct P4 {  // a lane's 8 features in pairs; rotated ones: first the four a of the pairs (a, b), then the four b
  uint64_t v[4];
};
__device__ __forceinline__ P4 scaled(const P4& x, float f) {
  const uint64_t g = two(f, f);
  return P4{{mul2(x.v[0], g), mul2(x.v[1], g), mul2(x.v[2], g), mul2(x.v[3], g)}};
}
__device__ __forceinline__ P4 product(const P4& x, const P4& y) {
  return P4{{mul2(x.v[0], y.v[0]), mul2(x.v[1], y.v[1]), mul2(x.v[2], y.v[2]), mul2(x.v[3], y.v[3])}};
}
__device__ __forceinline__ float dot_of(const P4& x, const P4& y) {
  uint64_t s = mul2(x.v[0], y.v[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j) s = fma2(x.v[j], y.v[j], s);
  float a, b;
  split(s, a, b);
  return a + b;
}
// eight scales from shared memory
__device__ __forceinline__ P4 scales_at(const float* p) {
  const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(p), b = *reinterpret_cast<const ulonglong2*>(p + 4);
  return P4{{a.x, a.y, b.x, b.y}};
}

// the same, but from shared memory each time: kept for all rows of a head they are registers that the rows under way need
__device__ __forceinline__ P4 scales_at(uint32_t p) {
  P4 r;
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(r.v[0]), "=l"(r.v[1]) : "r"(p) : "memory");
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(r.v[2]), "=l"(r.v[3]) : "r"(p + 16) : "memory");
  return r;
}

// A lane's 8 features as they lie in memory: 8 in a row, or twice 4 (kInter false)
template <typename T, bool kInter>
struct Raw8;
template <bool kInter>
struct Raw8<__nv_bfloat16, kInter> {
  uint4 u;
  __device__ __forceinline__ void load(const char* p, int gap) {
    if (kInter) {
      u = *reinterpret_cast<const uint4*>(p);
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(p), y = *reinterpret_cast<const uint2*>(p + gap);
      u = make_uint4(x.x, x.y, y.x, y.y);
    }
  }
  __device__ __forceinline__ static float lo(uint32_t w) { return __uint_as_float(w << 16); }
  __device__ __forceinline__ static float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  __device__ __forceinline__ P4 get() const {
    if (kInter) return P4{{two(lo(u.x), lo(u.y)), two(lo(u.z), lo(u.w)), two(hi(u.x), hi(u.y)), two(hi(u.z), hi(u.w))}};
    return P4{{two(lo(u.x), hi(u.x)), two(lo(u.y), hi(u.y)), two(lo(u.z), hi(u.z)), two(lo(u.w), hi(u.w))}};
  }
  __device__ __forceinline__ static uint32_t word(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ __forceinline__ static void store(char* p, int gap, const P4& x) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) split(x.v[j], f[2 * j], f[2 * j + 1]);
    if (kInter) {
      *reinterpret_cast<uint4*>(p) = make_uint4(word(f[0], f[4]), word(f[1], f[5]), word(f[2], f[6]), word(f[3], f[7]));
    } else {
      *reinterpret_cast<uint2*>(p) = make_uint2(word(f[0], f[1]), word(f[2], f[3]));
      *reinterpret_cast<uint2*>(p + gap) = make_uint2(word(f[4], f[5]), word(f[6], f[7]));
    }
  }
};
template <bool kInter>
struct Raw8<float, kInter> {
  float4 a, b;
  __device__ __forceinline__ void load(const char* p, int gap) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + gap);
  }
  __device__ __forceinline__ P4 get() const {
    if (kInter) return P4{{two(a.x, a.z), two(b.x, b.z), two(a.y, a.w), two(b.y, b.w)}};
    return P4{{two(a.x, a.y), two(a.z, a.w), two(b.x, b.y), two(b.z, b.w)}};
  }
  __device__ __forceinline__ static void store(char* p, int gap, const P4& x) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) split(x.v[j], f[2 * j], f[2 * j + 1]);
    if (kInter) {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[4], f[1], f[5]);
      *reinterpret_cast<float4*>(p + gap) = make_float4(f[2], f[6], f[3], f[7]);
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(p + gap) = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
};

// What a lane is: features `at` .. + 3 and `at + gap` .. + 3 of the rows of its group; rotated: its pairs are 4 `sub` .. + 3 of the table
struct Lane {
  int sub, at, gap, group;
  bool real, turned;
};
template <bool kInter, int kLanes>
__device__ __forceinline__ Lane lane_of(const Args& a) {
  Lane l;
  const int lane = threadIdx.x & 31;
  l.sub = lane & (kLanes - 1);
  l.group = lane / kLanes;
  l.real = l.sub * 8 < a.d;
  l.turned = l.sub * 8 < a.rot;
  l.at = l.sub * 8;
  l.gap = 4;
  if (!kInter && l.turned) {
    l.at = l.sub * 4;
    l.gap = a.rot >> 1;
  }
  return l;
}

// the four pairs of a lane turned; t: their four cosines and four sines
__device__ __forceinline__ void rotate4(P4& x, const float* t) {
  const P4 cs = scales_at(t);
  const uint64_t minus = two(-1.f, -1.f);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint64_t a = x.v[j], b = x.v[2 + j], c = cs.v[j], s = cs.v[2 + j];
    x.v[j] = fma2(a, c, mul2(mul2(b, minus), s));
    x.v[2 + j] = fma2(a, s, mul2(b, c));
  }
}

// A CTA has the rows (token, head) of a few tokens. A group of kLanes lanes keeps to one head at a time, of the queries' or then the keys' or the values', and goes through the
// tokens: scale, strides and addresses stay, a row costs no selection. Where fewer heads are left than groups, `split` groups share the tokens of a head. (With the rows of a
// tile counted through, token after token, half of the instructions were addresses and choices: 25000 tokens x 16
// heads of 64, bf16, both passes, 70.4 us, by heads 65.0.)
struct Turn {
  int tk, row, split;  // first token of this group, its head, tokens to the next
  bool mine;
  __device__ __forceinline__ Turn(const Args& a, int row0, int rows, int group, int groups) {
    const bool whole = rows - row0 >= groups;
    const int left = whole ? groups : rows - row0;
    tk = whole ? 0 : left == 1 ? group : (int)__umulhi((uint32_t)group, a.split_inverse);
    row = row0 + group - tk * left;
    split = whole ? 1 : a.split;
    mine = tk < split;
  }
};

// feature that a lane has in place `in` of its 8
template <bool kInter>
__device__ __forceinline__ int feature_at(const Args& a, int sub, int in) {
  if (kInter) return sub * 8 + (in < 4 ? 2 * in : 2 * in - 7);
  if (sub * 8 < a.rot) return in < 4 ? sub * 4 + in : (a.rot >> 1) + sub * 4 + in - 4;
  return sub * 8 + in;
}
// shared memory: the scales of queries and keys in fp32 in the lanes' order, [2][kLanes * 8]; then the cosines and sines of the tile's tokens, [tokens][R / 8][2][4]
template <bool kInter, int kLanes>
__device__ __forceinline__ void fill_scales(const Args& a, float* scales) {
  if (!a.r[0].w) return;
  for (int i = threadIdx.x; i < 2 * kLanes * 8; i += kThreads) {
    const int e = i % (kLanes * 8);
    scales[i] = e < a.d ? weight_at(i < kLanes * 8 ? a.r[0].w : a.r[1].w, feature_at<kInter>(a, e >> 3, e & 7), a.w_bf16) : 0.f;
  }
}
__device__ __forceinline__ void fill_table(const Args& a, float* table, int64_t t0, int nt, float sign) {
  const int half = a.rot >> 1;
  if (!half) return;
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int tk = (int)__umulhi(i, a.half_inverse), pair = i - tk * half;  // (half is 4 at least)
    const float2 t = turn_of(a, position_of(a, t0 + tk), turns_of(a, pair));
    float* to = table + tk * a.rot + (pair >> 2) * 8 + (pair & 3);
    to[0] = t.x;
    to[4] = t.y * sign;
  }
}

template <typename T, bool kInter, bool kCache, int kLanes>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? kCtasBf16 : kCtasF32)
forward_kernel(const Args a) {
  extern __shared__ __align__(16) float smem[];
  float* table = smem + 2 * kLanes * 8;
  rb_pdl_wait();
  rb_pdl_launch();
  constexpr int kTurns = sizeof(T) == 2 ? kTurnsBf16 : kTurnsF32, kSize = sizeof(T), kGroups = kThreads / kLanes;
  using Raw = Raw8<T, kInter>;
  const Lane l = lane_of<kInter, kLanes>(a);
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int nt = (int)min((int64_t)a.tokens, a.n - t0);
  const int hq = a.r[0].heads, hk = a.r[1].heads, rows = hq + hk + (kCache ? hk : 0), groups = gridDim.y * kGroups;
  const bool norm = a.r[0].w != nullptr;
  const int gap = l.gap * kSize;
  bool ready = false;
  for (int row0 = 0; row0 < rows; row0 += groups) {
    const Turn turn(a, row0, rows, blockIdx.y * kGroups + threadIdx.x / kLanes, groups);
    const bool is_q = turn.row < hq, is_v = kCache && turn.row >= hq + hk, mine = turn.mine && l.real;
    const Rows& w = a.r[is_q ? 0 : is_v ? 2 : 1];
    const int h = is_q ? turn.row : is_v ? turn.row - hq - hk : turn.row - hq;
    const char* from = reinterpret_cast<const char*>(w.x) + ((t0 + turn.tk) * w.tok + h * w.head + l.at) * kSize;
    const int step = turn.split * (int)w.tok * kSize, out_step = turn.split * w.heads * a.d * kSize;
    char* to = reinterpret_cast<char*>(w.out) + (kCache && !is_q ? h * w.page_head + l.at : ((t0 + turn.tk) * w.heads + h) * a.d + l.at) * kSize;
    P4 scales;
    for (int t = 0; t < nt; t += kTurns * turn.split) {
      Raw raw[kTurns] = {};
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        if (mine && turn.tk + t + u * turn.split < nt) raw[u].load(from, gap);
        from += step;
      }
      if (!ready) {  // while the first rows are under way
        fill_scales<kInter, kLanes>(a, smem);
        fill_table(a, table, t0, nt, 1.f);
        __syncthreads();
        ready = true;
      }
      if (norm && t == 0) scales = scales_at(smem + (is_q ? 0 : kLanes * 8) + l.sub * 8);
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        if (t + u * turn.split < nt) {
          const int tk = turn.tk + t + u * turn.split;
          P4 y = raw[u].get();
          if (norm) {
            const float inv = rsqrtf(group_sum(dot_of(y, y), kLanes) * a.inv_d + a.eps);
            if (!is_v) y = product(scaled(y, inv), scales);
          }
          if (mine && tk < nt) {
            if (!is_v && l.turned) rotate4(y, table + tk * a.rot + l.sub * 8);
            if (!kCache || is_q) {
              Raw::store(to, gap, y);
            } else {
              const int64_t at = cache_at(a, w, t0 + tk);
              if (at >= 0) Raw::store(to + at * kSize, gap, y);
            }
          }
          if (!kCache || is_q) to += out_step;
        }
      }
    }
  }
}

// kNorm: x is read again and the weights have gradients (sums per CTA, added up in order by the kernel below)
template <typename T, bool kInter, bool kNorm, int kLanes>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? kBackCtasBf16 : kBackCtasF32)
backward_kernel(const Args a) {
  extern __shared__ __align__(16) float smem[];
  float* table = smem + 2 * kLanes * 8;
  rb_pdl_wait();
  rb_pdl_launch();
  constexpr int kTurns = sizeof(T) == 2 ? kBackBf16 : kBackF32, kSize = sizeof(T), kGroups = kThreads / kLanes;
  using Raw = Raw8<T, kInter>;
  const Lane l = lane_of<kInter, kLanes>(a);
  const int hq = a.r[0].heads, hk = a.r[1].heads, rows = hq + hk;
  const int gap = l.gap * kSize;
  // sums of the scales' gradients: this thread's 8 of queries and of keys, touched once per head and tile
  float* sums = smem + 2 * kLanes * 8 + a.tokens * a.rot;
  ulonglong2* mine_q = reinterpret_cast<ulonglong2*>(sums) + threadIdx.x * 2;  // [2][groups][lanes * 8]
  ulonglong2* mine_k = mine_q + kThreads * 2;
  if (kNorm) mine_q[0] = mine_q[1] = mine_k[0] = mine_k[1] = make_ulonglong2(0, 0);
  bool have_scales = false;
  for (int64_t t0 = (int64_t)blockIdx.x * a.tokens; t0 < a.n; t0 += (int64_t)gridDim.x * a.tokens) {
    const int nt = (int)min((int64_t)a.tokens, a.n - t0);
    for (int row0 = 0; row0 < rows; row0 += gridDim.y * kGroups) {
      const Turn turn(a, row0, rows, blockIdx.y * kGroups + threadIdx.x / kLanes, gridDim.y * kGroups);
      const bool is_q = turn.row < hq, mine = turn.mine && l.real;
      const Rows& w = a.r[is_q ? 0 : 1];
      const int h = is_q ? turn.row : turn.row - hq;
      const char* from_z = reinterpret_cast<const char*>(w.dz) + ((t0 + turn.tk) * w.dz_tok + h * w.dz_head + l.at) * kSize;
      const char* from_x = reinterpret_cast<const char*>(w.x) + ((t0 + turn.tk) * w.tok + h * w.head + l.at) * kSize;
      const int step_z = turn.split * (int)w.dz_tok * kSize, step_x = turn.split * (int)w.tok * kSize, out_step = turn.split * w.heads * a.d * kSize;
      char* to = reinterpret_cast<char*>(w.out) + (((t0 + turn.tk) * w.heads + h) * a.d + l.at) * kSize;
      P4 sum = {};
      const uint32_t at_scales = (uint32_t)__cvta_generic_to_shared(smem + (is_q ? 0 : kLanes * 8) + l.sub * 8);
      for (int t = 0; t < nt; t += kTurns * turn.split) {
        Raw raw_z[kTurns] = {}, raw_x[kNorm ? kTurns : 1] = {};
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
          if (mine && turn.tk + t + u * turn.split < nt) {
            raw_z[u].load(from_z, gap);
            if (kNorm) raw_x[u].load(from_x, gap);
          }
          from_z += step_z;
          if (kNorm) from_x += step_x;
        }
        if (row0 == 0 && t == 0) {
          __syncthreads();  // (the table of the tokens before has been read)
          if (!have_scales) fill_scales<kInter, kLanes>(a, smem);
          have_scales = true;
          fill_table(a, table, t0, nt, -1.f);
          __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
          if (t + u * turn.split < nt) {
            const int tk = turn.tk + t + u * turn.split;
            const bool live = mine && tk < nt;
            P4 g = raw_z[u].get();
            if (live && l.turned) rotate4(g, table + tk * a.rot + l.sub * 8);
            if (kNorm) {
              const P4 x = raw_x[u].get();
              const float square = group_sum(dot_of(x, x), kLanes) * a.inv_d + a.eps;
              const float inv = turn.mine && tk < nt ? rsqrtf(square) : 0.f;  // (no row here: without an epsilon the zeros would have no norm)
              const P4 v = scaled(x, inv);
#pragma unroll
              for (int j = 0; j < 4; ++j) sum.v[j] = fma2(g.v[j], v.v[j], sum.v[j]);  // (zeros in lanes and groups without a row)
              const P4 y = product(g, scales_at(at_scales));
              const float dot = -group_sum(dot_of(y, v), kLanes) * a.inv_d * inv;
              const uint64_t by = two(inv, inv), off = two(dot, dot);
#pragma unroll
              for (int j = 0; j < 4; ++j) g.v[j] = fma2(v.v[j], off, mul2(y.v[j], by));
            }
            if (live) Raw::store(to, gap, g);
            to += out_step;
          }
        }
      }
      if (kNorm) {
        ulonglong2* to_sum = is_q ? mine_q : mine_k;
        const ulonglong2 s0 = to_sum[0], s1 = to_sum[1];
        to_sum[0] = make_ulonglong2(add2(s0.x, sum.v[0]), add2(s0.y, sum.v[1]));
        to_sum[1] = make_ulonglong2(add2(s1.x, sum.v[2]), add2(s1.y, sum.v[3]));
      }
    }
  }
  if (kNorm) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
      const int e = i < a.d ? i : i - a.d, half = a.rot >> 1;
      int at = e;  // where the lanes have feature e
      if (kInter) at = (e & ~7) + (e & 1) * 4 + ((e & 7) >> 1);
      else if (e < a.rot) at = e < half ? (e >> 2) * 8 + (e & 3) : ((e - half) >> 2) * 8 + 4 + ((e - half) & 3);
      if (i >= a.d) at += kThreads * 8;
      float s = 0.f;
      for (int g = 0; g < kThreads / kLanes; ++g) s += sums[g * kLanes * 8 + at];
      a.part[(int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.d + i] = s;
    }
  }
}

// ---- any even rotated part, any head dim up to kMaxDim, any alignment: a warp per row, lane l has the features l, l + 32, ...
__device__ __forceinline__ int partner(int e, int rot, int interleaved, int* pair, float* sign) {
  if (interleaved) {
    *pair = e >> 1;
    *sign = e & 1 ? 1.f : -1.f;
    return e ^ 1;
  }
  const int half = rot >> 1;
  *pair = e < half ? e : e - half;
  *sign = e < half ? -1.f : 1.f;
  return e < half ? e + half : e - half;
}

template <typename T, bool kCache>
__global__ void __launch_bounds__(kThreads)
forward_any_kernel(const Args a) {
  const int lane = threadIdx.x & 31;
  const int rows = a.r[0].heads + a.r[1].heads + (kCache ? a.r[2].heads : 0);
  const int64_t total = a.n * rows;
  rb_pdl_wait();
  rb_pdl_launch();
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t token = i / rows;
    int h = (int)(i - token * rows), which = 0;
    if (h >= a.r[0].heads) {
      h -= a.r[0].heads;
      which = 1;
      if (kCache && h >= a.r[1].heads) {
        h -= a.r[1].heads;
        which = 2;
      }
    }
    const Rows& r = a.r[which];
    const int64_t base = token * r.tok + h * r.head;
    float inv = 1.f;
    if (r.w) {
      float s = 0.f;
      for (int e = lane; e < a.d; e += 32) {
        const float f = one<T>(r.x, base + e);
        s += f * f;
      }
      inv = rsqrtf(warp_sum(s) * a.inv_d + a.eps);
    }
    int64_t to = (token * r.heads + h) * a.d;
    if (kCache && which) {
      to = cache_at(a, r, token);
      if (to < 0) continue;
      to += h * r.page_head;
    }
    const int64_t pos = a.rot && which < 2 ? position_of(a, token) : 0;
    for (int e = lane; e < a.d; e += 32) {
      float y = one<T>(r.x, base + e);
      if (r.w) y *= inv * weight_at(r.w, e, a.w_bf16);
      if (which < 2 && e < a.rot) {
        int pair;
        float sign;
        const int o = partner(e, a.rot, a.interleaved, &pair, &sign);
        float other = one<T>(r.x, base + o);
        if (r.w) other *= inv * weight_at(r.w, o, a.w_bf16);
        const float2 t = turn_of(a, pos, turns_of(a, pair));
        y = y * t.x + sign * other * t.y;
      }
      put<T>(r.out, to + e, y);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
backward_any_kernel(const Args a) {
  __shared__ float sums[kThreads / 32][2][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = a.r[0].heads + a.r[1].heads;
  const int64_t total = a.n * rows;
  const bool norm = a.r[0].w != nullptr;
  rb_pdl_wait();
  rb_pdl_launch();
  float gq[kMaxDim / 32] = {}, gk[kMaxDim / 32] = {};
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + warp; i < total; i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t token = i / rows;
    int h = (int)(i - token * rows);
    const bool is_q = h < a.r[0].heads;
    if (!is_q) h -= a.r[0].heads;
    const Rows& r = a.r[is_q ? 0 : 1];
    const int64_t gb = token * r.dz_tok + h * r.dz_head, xb = token * r.tok + h * r.head, to = (token * r.heads + h) * a.d;
    const int64_t pos = a.rot ? position_of(a, token) : 0;
    float inv = 1.f, dot = 0.f;
    float dy[kMaxDim / 32], u[kMaxDim / 32];
    if (norm) {
      float s = 0.f;
      for (int e = lane; e < a.d; e += 32) {
        const float f = one<T>(r.x, xb + e);
        s += f * f;
      }
      inv = rsqrtf(warp_sum(s) * a.inv_d + a.eps);
    }
#pragma unroll
    for (int j = 0; j < kMaxDim / 32; ++j) {
      const int e = lane + 32 * j;
      dy[j] = u[j] = 0.f;
      if (e >= a.d) continue;
      dy[j] = one<T>(r.dz, gb + e);
      if (e < a.rot) {
        int pair;
        float sign;
        const int o = partner(e, a.rot, a.interleaved, &pair, &sign);
        const float2 t = turn_of(a, pos, turns_of(a, pair));
        dy[j] = dy[j] * t.x - sign * one<T>(r.dz, gb + o) * t.y;
      }
      if (norm) {
        u[j] = one<T>(r.x, xb + e) * inv;
        if (is_q) gq[j] += dy[j] * u[j]; else gk[j] += dy[j] * u[j];
        dy[j] *= weight_at(r.w, e, a.w_bf16);
        dot += dy[j] * u[j];
      }
    }
    if (norm) dot = warp_sum(dot) * a.inv_d;
#pragma unroll
    for (int j = 0; j < kMaxDim / 32; ++j) {
      const int e = lane + 32 * j;
      if (e < a.d) put<T>(r.out, to + e, norm ? inv * (dy[j] - u[j] * dot) : dy[j]);
    }
  }
  if (norm) {
#pragma unroll
    for (int j = 0; j < kMaxDim / 32; ++j) {
      sums[warp][0][lane + 32 * j] = gq[j];
      sums[warp][1][lane + 32 * j] = gk[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
      float s = 0.f;
      for (int w = 0; w < kThreads / 32; ++w) s += sums[w][i / a.d][i % a.d];
      a.part[(int64_t)blockIdx.x * 2 * a.d + i] = s;
    }
  }
}

// the partial sums of all CTAs in order -> gradients in the type of the weights. A CTA has 32 columns, its warps every 32nd of the rows, ten of which are asked for at a
// time: what bounds it is the memory's latency, twice (592 rows; 8 warps with 8 at a time waited ten times, which made
// passes of 25000 x 16 rows of 64 in bf16 and 8191 x 40 of 128 in fp32 3 and 7 us longer).
constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(kSumWarps * 32)
weight_sum_kernel(const float* __restrict__ part, int parts, int d, void* __restrict__ dwq, void* __restrict__ dwk, int w_bf16) {
  constexpr int kAhead = 10;
  __shared__ float sh[kSumWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  rb_pdl_wait();
  rb_pdl_launch();
  float s = 0.f;
  if (col < 2 * d) {
    for (int p0 = warp; p0 < parts; p0 += kAhead * kSumWarps) {
      float v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = p0 + k * kSumWarps < parts ? part[(int64_t)(p0 + k * kSumWarps) * 2 * d + col] : 0.f;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) s += v[k];
    }
  }
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < 2 * d) {
#pragma unroll
    for (int w = 1; w < kSumWarps; ++w) s += sh[w][lane];
    void* out = col < d ? dwq : dwk;
    const int at = col < d ? col : col - d;
    if (w_bf16) put<__nv_bfloat16>(out, at, s);
    else put<float>(out, at, s);
  }
}

// f of the lanes of a row, 1 to 32, as a constant
template <typename F>
auto with_lanes(int d, F f) {
  if (d <= 8) return f(std::integral_constant<int, 1>());
  if (d <= 16) return f(std::integral_constant<int, 2>());
  if (d <= 32) return f(std::integral_constant<int, 4>());
  if (d <= 64) return f(std::integral_constant<int, 8>());
  if (d <= 128) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}
int lanes_of(int d) {
  return with_lanes(d, [](auto l) { return (int)decltype(l)::value; });
}

bool aligned(const void* p, std::initializer_list<int64_t> strides, int unit, int bytes) {
  if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
  for (int64_t s : strides)
    if (s % unit) return false;
  return true;
}

int bad_shape(const Args& a) {
  if (a.d >= 1 && a.d <= kMaxDim && a.rot >= 0 && a.rot <= a.d && a.rot % 2 == 0 && a.r[0].heads >= 0 && a.r[1].heads >= 0 && (a.rot == 0 || a.num_pos > 0 || a.n <= 0)) return 0;
  rb_set_error("norm_rope: head dim %d (1 to %d), rotated part %d (even, at most the head dim)", a.d, kMaxDim, a.rot);
  return 1;
}

// 8 features a lane, whole pairs, vector accesses (16 bytes; pairs (i, i + R / 2) in bf16: 8)
bool fits(const Args& a, int bf16, bool backward, bool cache) {
  const int bytes = bf16 && !a.interleaved ? 8 : 16, unit = bytes / (bf16 ? 2 : 4);
  if (a.d % 8 || a.rot % 8) return false;
  bool ok = true;
  for (int i = 0; i < (cache ? 3 : 2); ++i) {
    const Rows& r = a.r[i];
    ok = ok && aligned(r.out, {}, unit, bytes);
    if (!backward || a.r[0].w) ok = ok && aligned(r.x, {r.tok, r.head}, unit, bytes);
    if (backward) ok = ok && aligned(r.dz, {r.dz_tok, r.dz_head}, unit, bytes);
    if (cache && i) ok = ok && aligned(r.out, {r.page, r.page_head, r.page_tok}, unit, bytes);
    // steps of up to 256 tokens in 32 bits, group numbers in 16
    ok = ok && std::max({std::abs(r.tok), std::abs(r.dz_tok), (int64_t)a.d * r.heads}) * 256 * 4 < (int64_t)1 << 31 && r.heads < 16384;
  }
  return ok;
}

// A tile is as many tokens as fill the table with an angle per thread; fewer where that leaves SMs without any. Each has a beginning that costs about as much as two rows of a group:
// tiles are up to four times as large where the turns in which the SMs take them are the shorter for it (bf16, us, 8191 tokens x 40 rows of 128, both passes: 103.6 with 4 tokens,
// 97.1 with 16 in the backward pass; forward 38.3 and 35.6; 100000 x 40 of 128 forward 405 and 364; 20000 x 24 of 64 take 8: 5 turns of those are shorter than 3 of 16, 26.6 and
// 34.6). Not so for fp32 forward, whose rows are bound by the memory (8191 x 40 of 128: 56 and 64), nor for a turn and a half (6000 x 16 of 64: 7.4 and 8.4).
// Where all tiles are on the SMs at once, their heads are shared by as many CTAs as it takes for every group to have one head (returned): all rows are then asked for at the
// beginning.
int tile_of(Args& a, int rows, int groups, int ctas, bool may_grow) {
  const int need = std::max(1, (rows + groups - 1) / groups);
  auto tiles = [&]() { return (a.n + a.tokens - 1) / a.tokens; };
  a.tokens = a.rot ? std::max(1, kThreads / (a.rot / 2)) : 8;
  const int64_t slots = ctas * 148;
  if (may_grow && tiles() * 2 >= slots * 3) {
    const int least = a.tokens;
    auto turns = [&]() { return (tiles() + slots - 1) / slots * (a.tokens * (int64_t)rows + 2 * groups); };
    int best = least;
    int64_t cost = turns();
    for (int more = 2; more <= 4; more *= 2) {
      a.tokens = least * more;
      if (tiles() < 2 * 148 || turns() >= cost) continue;
      best = a.tokens;
      cost = turns();
    }
    a.tokens = best;
  }
  while (a.tokens > 1 && tiles() * need < 2 * 148) a.tokens /= 2;
  const int shared_by = tiles() * need <= ctas * 148 ? need : 1;
  while (a.tokens > 1 && tiles() * shared_by < 2 * 148) a.tokens /= 2;
  const int left = rows % (groups * shared_by);
  a.split = left ? groups * shared_by / left : 1;
  a.split_inverse = left > 1 ? (uint32_t)(((1ull << 32) + left - 1) / left) : 0u;
  a.half_inverse = a.rot ? (uint32_t)(((1ull << 32) + a.rot / 2 - 1) / (a.rot / 2)) : 0u;
  return shared_by;
}
size_t smem_of(const Args& a) { return (size_t)lanes_of(a.d) * 16 * sizeof(float) + (size_t)a.tokens * (a.rot / 2) * sizeof(float2); }

constexpr int kParts = 148 * std::max(kBackCtasBf16, kBackCtasF32);

int forward(Args& a, int bf16, bool cache, cudaStream_t stream) {
  if (bad_shape(a)) return RB_ERR_UNSUPPORTED;
  const int rows = a.r[0].heads + a.r[1].heads * (cache ? 2 : 1);
  if (a.n <= 0 || rows == 0) return RB_OK;
  a.inv_d = 1.f / a.d;
  if (fits(a, bf16, false, cache)) {
    const int gy = tile_of(a, rows, kThreads / lanes_of(a.d), bf16 ? kCtasBf16 : kCtasF32, bf16);
    const int64_t gx = (a.n + a.tokens - 1) / a.tokens;
    if (gx > 0x7fffffff) {
      rb_set_error("norm_rope: %lld tokens", (long long)a.n);
      return RB_ERR_UNSUPPORTED;
    }
    auto pick = [&](auto t) {
      return with_lanes(a.d, [&](auto l) {
        using T = decltype(t);
        constexpr int kL = decltype(l)::value;
        return a.interleaved ? (cache ? forward_kernel<T, true, true, kL> : forward_kernel<T, true, false, kL>)
                             : (cache ? forward_kernel<T, false, true, kL> : forward_kernel<T, false, false, kL>);
      });
    };
    auto kernel = bf16 ? pick(__nv_bfloat16()) : pick(float());
    rb_launch_pdl(kernel, dim3((unsigned)gx, gy), dim3(kThreads), smem_of(a), stream, a);
  } else {
    const int64_t ctas = (a.n * rows + kThreads / 32 - 1) / (kThreads / 32);
    auto kernel = bf16 ? (cache ? forward_any_kernel<__nv_bfloat16, true> : forward_any_kernel<__nv_bfloat16, false>)
                       : (cache ? forward_any_kernel<float, true> : forward_any_kernel<float, false>);
    rb_launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(ctas, 148 * 8)), dim3(kThreads), 0, stream, a);
  }
  return rb_check_launch("norm_rope");
}

Rows rows_of(const void* x, int64_t tok, int64_t head, int heads, const void* w, void* out) {
  Rows r = {};
  r.x = x; r.tok = tok; r.head = head; r.heads = heads; r.w = w; r.out = out;
  return r;
}
void common(Args& a, const void* positions, long long num_pos, const float* freq, long long n, int d, int rot, int pos64, int w_bf16, int interleaved, float eps, float amp) {
  a.positions = positions; a.num_pos = num_pos; a.freq = freq; a.n = n; a.d = d; a.rot = rot; a.pos64 = pos64; a.w_bf16 = w_bf16; a.interleaved = interleaved;
  a.eps = eps; a.amp = amp;
}

}  // namespace

RB_EXPORT int rb200_norm_rope_fwd(const void* q, const void* k, const void* positions, long long num_pos, const float* freq, const void* wq, const void* wk, void* out_q,
                                  void* out_k, const long long* strides /* q token, q head, k token, k head */, long long n, int hq, int hk, int d, int rot,
                                  int bf16, int pos64, int w_bf16, int interleaved, float eps, float amp, cudaStream_t stream) {
  Args a = {};
  a.r[0] = rows_of(q, strides[0], strides[1], hq, wq, out_q);
  a.r[1] = rows_of(k, strides[2], strides[3], hk, wk, out_k);
  common(a, positions, num_pos, freq, n, d, rot, pos64, w_bf16, interleaved, eps, amp);
  return forward(a, bf16, false, stream);
}

RB_EXPORT int rb200_norm_rope_cache(const void* q, const void* k, const void* v, const void* positions, long long num_pos, const float* freq, const void* wq, const void* wk,
                                    void* out_q, void* cache_k, void* cache_v, const int* slots,
                                    const long long* strides /* q, k, v: token, head; cache k, cache v: page, head, token */, long long n, int hq, int hk, int d,
                                    int rot, int page, long long num_slots, int bf16, int pos64, int w_bf16, int interleaved, float eps, float amp,
                                    cudaStream_t stream) {
  Args a = {};
  if (page < 1) {
    rb_set_error("norm_rope: page size %d", page);
    return RB_ERR_ARG;
  }
  a.r[0] = rows_of(q, strides[0], strides[1], hq, wq, out_q);
  a.r[1] = rows_of(k, strides[2], strides[3], hk, wk, cache_k);
  a.r[2] = rows_of(v, strides[4], strides[5], hk, nullptr, cache_v);
  for (int i = 0; i < 2; ++i) {
    a.r[1 + i].page = strides[6 + 3 * i];
    a.r[1 + i].page_head = strides[7 + 3 * i];
    a.r[1 + i].page_tok = strides[8 + 3 * i];
  }
  a.slots = slots; a.page = page; a.num_slots = num_slots;
  common(a, positions, num_pos, freq, n, d, rot, pos64, w_bf16, interleaved, eps, amp);
  return forward(a, bf16, true, stream);
}

// partial sums that the backward pass leaves: rows of 2 D floats
RB_EXPORT int rb200_norm_rope_parts() { return kParts; }

// part: [rb200_norm_rope_parts()][2][D] floats with a norm, else unused; dwq, dwk [D] in the type of the weights
RB_EXPORT int rb200_norm_rope_bwd(const void* dq, const void* dk, const void* q, const void* k, const void* positions, long long num_pos, const float* freq, const void* wq,
                                  const void* wk, void* out_q, void* out_k, float* part, void* dwq, void* dwk,
                                  const long long* strides /* dq, dk, q, k: token, head */, long long n, int hq, int hk, int d, int rot, int bf16, int pos64,
                                  int w_bf16, int interleaved, float eps, float amp, cudaStream_t stream) {
  Args a = {};
  a.r[0] = rows_of(q, strides[4], strides[5], hq, wq, out_q);
  a.r[1] = rows_of(k, strides[6], strides[7], hk, wk, out_k);
  a.r[0].dz = dq; a.r[0].dz_tok = strides[0]; a.r[0].dz_head = strides[1];
  a.r[1].dz = dk; a.r[1].dz_tok = strides[2]; a.r[1].dz_head = strides[3];
  a.part = part;
  common(a, positions, num_pos, freq, n, d, rot, pos64, w_bf16, interleaved, eps, amp);
  if (bad_shape(a)) return RB_ERR_UNSUPPORTED;
  const bool norm = wq != nullptr;
  const int rows = hq + hk;
  if (n <= 0 || rows == 0) {  // sums of nothing; a launch for it would have as many groups as there are heads, more than places in `part`
    const size_t bytes = (size_t)d * (w_bf16 ? 2 : 4);
    if (norm && (cudaMemsetAsync(dwq, 0, bytes, stream) != cudaSuccess || cudaMemsetAsync(dwk, 0, bytes, stream) != cudaSuccess)) return rb_check_launch("norm_rope_bwd");
    return RB_OK;
  }
  a.inv_d = 1.f / d;
  int64_t grid;
  int gy = 1;
  if (fits(a, bf16, true, false)) {
    const int ctas = bf16 ? kBackCtasBf16 : kBackCtasF32;
    gy = tile_of(a, rows, kThreads / lanes_of(d), ctas, true);
    grid = std::min<int64_t>((n + a.tokens - 1) / a.tokens, 148 * ctas / gy);  // (gy: 148 * ctas at most, there is a tile)
    const size_t sums = norm ? (size_t)kThreads * 2 * 8 * sizeof(float) : 0;
    auto pick = [&](auto t) {
      return with_lanes(d, [&](auto l) {
        using T = decltype(t);
        constexpr int kL = decltype(l)::value;
        return interleaved ? (norm ? backward_kernel<T, true, true, kL> : backward_kernel<T, true, false, kL>)
                           : (norm ? backward_kernel<T, false, true, kL> : backward_kernel<T, false, false, kL>);
      });
    };
    auto kernel = bf16 ? pick(__nv_bfloat16()) : pick(float());
    rb_launch_pdl(kernel, dim3((unsigned)grid, (unsigned)gy), dim3(kThreads), smem_of(a) + sums, stream, a);
  } else {
    grid = std::min<int64_t>((n * rows + kThreads / 32 - 1) / (kThreads / 32), kParts);
    auto kernel = bf16 ? backward_any_kernel<__nv_bfloat16> : backward_any_kernel<float>;
    rb_launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  }
  if (norm) rb_launch_pdl(weight_sum_kernel, dim3((2 * d + 31) / 32), dim3(kSumWarps * 32), 0, stream, (const float*)part, (int)grid * gy, d, dwq, dwk, w_bf16);
  return rb_check_launch("norm_rope_bwd");
}
