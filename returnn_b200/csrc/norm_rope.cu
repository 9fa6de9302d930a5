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
// What bounds it is the instructions around 16 bytes: each turn of a warp has addresses that only go on by a fixed step.
#include "packed_f32.cuh"
#include <algorithm>
#include <cstdlib>
#include <initializer_list>
#include <type_traits>

namespace {

constexpr int kMaxDim = 256;
constexpr int kThreads = 256;
constexpr int kTurnsBf16 = 4, kTurnsF32 = 2, kBackBf16 = 2, kBackF32 = 1;  // rows of a group that are under way at a time, forward and backward
constexpr int kBackCtas = 4;                                               // of an SM

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
  int step_tk, step_h;              // of a row of a tile: tokens and heads to the next of its group
  uint32_t rows_inverse, half_inverse;
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
struct P4 {  // 8 numbers in pairs
  uint64_t v[4];
};
__device__ __forceinline__ P4 pairs(const F8& x) { return P4{{two(x.v[0], x.v[1]), two(x.v[2], x.v[3]), two(x.v[4], x.v[5]), two(x.v[6], x.v[7])}}; }
__device__ __forceinline__ F8 single(const P4& x) {
  F8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) split(x.v[j], r.v[2 * j], r.v[2 * j + 1]);
  return r;
}
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
  __device__ __forceinline__ F8 get() const {
    F8 r;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.v[2 * i] = __uint_as_float(w[i] << 16);
      r.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    return r;
  }
  __device__ __forceinline__ static void store(char* p, int gap, const F8& f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.v[2 * i], f.v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if (kInter) {
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(p + gap) = make_uint2(w[2], w[3]);
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
  __device__ __forceinline__ F8 get() const { return F8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}}; }
  __device__ __forceinline__ static void store(char* p, int gap, const F8& f) {
    *reinterpret_cast<float4*>(p) = make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
    *reinterpret_cast<float4*>(p + gap) = make_float4(f.v[4], f.v[5], f.v[6], f.v[7]);
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

// the four pairs of a lane turned (sign -1: back)
template <bool kInter>
__device__ __forceinline__ void rotate4(F8& x, const float2* table, const Lane& l, float sign) {
  if (!l.turned) return;
  const float4* t = reinterpret_cast<const float4*>(table + l.sub * 4);
  const float4 t0 = t[0], t1 = t[1];
  const float c[4] = {t0.x, t0.z, t1.x, t1.z}, s[4] = {t0.y * sign, t0.w * sign, t1.y * sign, t1.w * sign};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float &p = x.v[kInter ? 2 * j : j], &q = x.v[kInter ? 2 * j + 1 : 4 + j];
    const float u = p * c[j] - q * s[j];
    q = p * s[j] + q * c[j];
    p = u;
  }
}

// A CTA has the rows (token, head) of a few tokens, queries' heads before keys' and values', a row per group of kLanes lanes and turn. Rows go on by whole steps, so that token
// and head cost no division; offsets within a tile of tokens are 32 bits wide (see fits).
struct Walk {
  int tk, h;
  __device__ __forceinline__ Walk(int start, uint32_t inverse, int of) {  // inverse: 2^32 / of, rounded up; start below 2^16
    tk = of == 1 ? start : (int)__umulhi((uint32_t)start, inverse);
    h = start - tk * of;
  }
  __device__ __forceinline__ void go(const Args& a, int of) {
    tk += a.step_tk;
    h += a.step_h;
    if (h >= of) {
      h -= of;
      ++tk;
    }
  }
};

// shared memory: the scales of queries and keys in fp32 in the lanes' order, [2][kLanes * 8]; then the angles of the tile's tokens, [tokens][R / 2]
template <bool kInter, int kLanes>
__device__ __forceinline__ void fill_scales(const Args& a, float* scales) {
  if (!a.r[0].w) return;
  for (int i = threadIdx.x; i < 2 * kLanes * 8; i += kThreads) {
    const int e = i % (kLanes * 8), sub = e >> 3, in = e & 7;
    int at = e;
    if (!kInter && sub * 8 < a.rot) at = in < 4 ? sub * 4 + in : (a.rot >> 1) + sub * 4 + in - 4;
    scales[i] = e < a.d ? weight_at(i < kLanes * 8 ? a.r[0].w : a.r[1].w, at, a.w_bf16) : 0.f;
  }
}
__device__ __forceinline__ void fill_table(const Args& a, float2* table, int64_t t0, int nt) {
  const int half = a.rot >> 1;
  if (!half) return;
  const Walk w(threadIdx.x, a.half_inverse, half);  // (an angle per thread: see tile_of)
  if (w.tk < nt) table[threadIdx.x] = turn_of(a, position_of(a, t0 + w.tk), turns_of(a, w.h));
}

template <typename T, bool kInter, bool kCache, int kLanes>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 5 : 4)
forward_kernel(const Args a) {
  extern __shared__ __align__(16) float smem[];
  float2* table = reinterpret_cast<float2*>(smem + 2 * kLanes * 8);
  rb_pdl_wait();
  rb_pdl_launch();
  constexpr int kTurns = sizeof(T) == 2 ? kTurnsBf16 : kTurnsF32, kSize = sizeof(T), kGroups = kThreads / kLanes;
  using Raw = Raw8<T, kInter>;
  const Lane l = lane_of<kInter, kLanes>(a);
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int nt = (int)min((int64_t)a.tokens, a.n - t0);
  const int hq = a.r[0].heads, hk = a.r[1].heads, rows = hq + hk + (kCache ? hk : 0), half = a.rot >> 1;
  const bool norm = a.r[0].w != nullptr;
  const int gap = l.gap * kSize;
  const char* in_q = reinterpret_cast<const char*>(a.r[0].x) + (t0 * a.r[0].tok + l.at) * kSize;
  const char* in_k = reinterpret_cast<const char*>(a.r[1].x) + (t0 * a.r[1].tok + l.at) * kSize;
  const char* in_v = kCache ? reinterpret_cast<const char*>(a.r[2].x) + (t0 * a.r[2].tok + l.at) * kSize : nullptr;
  char* out_q = reinterpret_cast<char*>(a.r[0].out) + (t0 * hq * a.d + l.at) * kSize;
  char* out_k = kCache ? nullptr : reinterpret_cast<char*>(a.r[1].out) + (t0 * hk * a.d + l.at) * kSize;
  const int total = nt * rows, step = gridDim.y * kGroups;
  Walk fetch(blockIdx.y * kGroups + threadIdx.x / kLanes, a.rows_inverse, rows), use = fetch;
  bool ready = false;
  for (int r = blockIdx.y * kGroups; r < total; r += kTurns * step) {
    Raw raw[kTurns] = {};
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      if (fetch.tk < nt && l.real) {
        const bool is_q = fetch.h < hq, is_v = kCache && fetch.h >= hq + hk;
        const int tok = (int)(is_q ? a.r[0].tok : is_v ? a.r[2].tok : a.r[1].tok), head = (int)(is_q ? a.r[0].head : is_v ? a.r[2].head : a.r[1].head);
        const int h = is_q ? fetch.h : is_v ? fetch.h - hq - hk : fetch.h - hq;
        raw[u].load((is_q ? in_q : is_v ? in_v : in_k) + (fetch.tk * tok + h * head) * kSize, gap);
      }
      fetch.go(a, rows);
    }
    if (!ready) {  // while the first rows are under way
      fill_scales<kInter, kLanes>(a, smem);
      fill_table(a, table, t0, nt);
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      if (r + u * step < total) {
        const bool live = use.tk < nt && l.real, is_q = use.h < hq, is_v = kCache && use.h >= hq + hk;
        F8 y = raw[u].get();
        if (norm) {
          const P4 x = pairs(y);
          const float inv = rsqrtf(group_sum(dot_of(x, x), kLanes) * a.inv_d + a.eps);
          if (!is_v) y = single(product(scaled(x, inv), scales_at(smem + (is_q ? 0 : kLanes * 8) + l.sub * 8)));
        }
        if (live) {
          if (!is_v) rotate4<kInter>(y, table + use.tk * half, l, 1.f);
          char* out;
          if (is_q) {
            out = out_q + (use.tk * hq + use.h) * (a.d * kSize);
          } else if (!kCache) {
            out = out_k + (use.tk * hk + use.h - hq) * (a.d * kSize);
          } else {
            const Rows& k = is_v ? a.r[2] : a.r[1];
            const int64_t at = cache_at(a, k, t0 + use.tk);
            out = at < 0 ? nullptr : reinterpret_cast<char*>(k.out) + (at + (is_v ? use.h - hq - hk : use.h - hq) * k.page_head + l.at) * kSize;
          }
          if (!kCache || out) Raw::store(out, gap, y);
        }
        use.go(a, rows);
      }
    }
  }
}

// kNorm: x is read again and the weights have gradients (sums per CTA, added up in order by the kernel below)
template <typename T, bool kInter, bool kNorm, int kLanes>
__global__ void __launch_bounds__(kThreads, kBackCtas)
backward_kernel(const Args a) {
  extern __shared__ __align__(16) float smem[];
  float2* table = reinterpret_cast<float2*>(smem + 2 * kLanes * 8);
  rb_pdl_wait();
  rb_pdl_launch();
  constexpr int kTurns = sizeof(T) == 2 ? kBackBf16 : kBackF32, kSize = sizeof(T), kGroups = kThreads / kLanes;
  using Raw = Raw8<T, kInter>;
  const Lane l = lane_of<kInter, kLanes>(a);
  const int hq = a.r[0].heads, hk = a.r[1].heads, rows = hq + hk, half = a.rot >> 1;
  const int gap = l.gap * kSize;
  P4 gq = {}, gk = {};
  bool have_scales = false;
  for (int64_t t0 = (int64_t)blockIdx.x * a.tokens; t0 < a.n; t0 += (int64_t)gridDim.x * a.tokens) {
    const int nt = (int)min((int64_t)a.tokens, a.n - t0);
    const char* dz_q = reinterpret_cast<const char*>(a.r[0].dz) + (t0 * a.r[0].dz_tok + l.at) * kSize;
    const char* dz_k = reinterpret_cast<const char*>(a.r[1].dz) + (t0 * a.r[1].dz_tok + l.at) * kSize;
    const char* in_q = reinterpret_cast<const char*>(a.r[0].x) + (t0 * a.r[0].tok + l.at) * kSize;
    const char* in_k = reinterpret_cast<const char*>(a.r[1].x) + (t0 * a.r[1].tok + l.at) * kSize;
    char* out_q = reinterpret_cast<char*>(a.r[0].out) + (t0 * hq * a.d + l.at) * kSize;
    char* out_k = reinterpret_cast<char*>(a.r[1].out) + (t0 * hk * a.d + l.at) * kSize;
    const int total = nt * rows;
    Walk fetch(threadIdx.x / kLanes, a.rows_inverse, rows), use = fetch;
    for (int r = 0; r < total; r += kTurns * kGroups) {
      Raw raw_g[kTurns] = {}, raw_x[kNorm ? kTurns : 1] = {};
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        if (fetch.tk < nt && l.real) {
          const bool is_q = fetch.h < hq;
          const int h = is_q ? fetch.h : fetch.h - hq;
          raw_g[u].load((is_q ? dz_q : dz_k) + (fetch.tk * (int)(is_q ? a.r[0].dz_tok : a.r[1].dz_tok) + h * (int)(is_q ? a.r[0].dz_head : a.r[1].dz_head)) * kSize, gap);
          if (kNorm) raw_x[u].load((is_q ? in_q : in_k) + (fetch.tk * (int)(is_q ? a.r[0].tok : a.r[1].tok) + h * (int)(is_q ? a.r[0].head : a.r[1].head)) * kSize, gap);
        }
        fetch.go(a, rows);
      }
      if (r == 0) {
        __syncthreads();  // (the table of the tokens before has been read)
        if (!have_scales) fill_scales<kInter, kLanes>(a, smem);
        have_scales = true;
        fill_table(a, table, t0, nt);
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        if (r + u * kGroups < total) {
          const bool live = use.tk < nt && l.real, is_q = use.h < hq;
          F8 g = raw_g[u].get();
          if (live) rotate4<kInter>(g, table + use.tk * half, l, -1.f);
          if (kNorm) {
            const P4 x = pairs(raw_x[u].get());
            const float inv = rsqrtf(group_sum(dot_of(x, x), kLanes) * a.inv_d + a.eps);
            const P4 v = scaled(x, inv), dy = pairs(g);
            const uint64_t yes = two(is_q ? 1.f : 0.f, is_q ? 1.f : 0.f), no = two(is_q ? 0.f : 1.f, is_q ? 0.f : 1.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint64_t e = mul2(dy.v[j], v.v[j]);  // (zeros in lanes and groups without a row)
              gq.v[j] = fma2(e, yes, gq.v[j]);
              gk.v[j] = fma2(e, no, gk.v[j]);
            }
            const P4 w = product(dy, scales_at(smem + (is_q ? 0 : kLanes * 8) + l.sub * 8));
            const float dot = -group_sum(dot_of(w, v), kLanes) * a.inv_d * inv;
            const uint64_t by = two(inv, inv), off = two(dot, dot);
            P4 r;
#pragma unroll
            for (int j = 0; j < 4; ++j) r.v[j] = fma2(v.v[j], off, mul2(w.v[j], by));
            g = single(r);
          }
          if (live) Raw::store(is_q ? out_q + (use.tk * hq + use.h) * (a.d * kSize) : out_k + (use.tk * hk + use.h - hq) * (a.d * kSize), gap, g);
          use.go(a, rows);
        }
      }
    }
  }
  if (kNorm) {
    float* sums = smem;  // [groups][2][lanes * 8] in the lanes' order; at least as large as this (see the launch)
    __syncthreads();
    float* mine = sums + threadIdx.x / kLanes * 2 * kLanes * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      reinterpret_cast<uint64_t*>(mine + l.sub * 8)[j] = gq.v[j];
      reinterpret_cast<uint64_t*>(mine + kLanes * 8 + l.sub * 8)[j] = gk.v[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
      const int e = i < a.d ? i : i - a.d, half = a.rot >> 1;
      int at = e;  // where the lanes have feature e
      if (!kInter && e < a.rot) at = e < half ? (e >> 2) * 8 + (e & 3) : ((e - half) >> 2) * 8 + 4 + ((e - half) & 3);
      if (i >= a.d) at += kLanes * 8;
      float s = 0.f;
      for (int g = 0; g < kThreads / kLanes; ++g) s += sums[g * 2 * kLanes * 8 + at];
      a.part[(int64_t)blockIdx.x * 2 * a.d + i] = s;
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

// 8 features a lane, whole pairs, vector accesses (16 bytes; pairs (i, i + R / 2) in bf16: 8), tiles below 2^31 bytes
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
    // offsets within a tile of up to 256 tokens
    const int64_t widest = std::max({std::abs(r.head), std::abs(r.dz_head), (int64_t)a.d}) * r.heads + std::max(std::abs(r.tok), std::abs(r.dz_tok)) * 256;
    ok = ok && widest * 4 < (int64_t)1 << 31 && (int64_t)a.d * r.heads * 256 * 4 < (int64_t)1 << 31;
  }
  return ok;
}

// A tile is as many tokens as fill the table with an angle per thread; fewer where that leaves SMs without any
void tile_of(Args& a) {
  a.tokens = a.rot ? std::max(1, kThreads / (a.rot / 2)) : 8;
  while (a.tokens > 1 && (a.n + a.tokens - 1) / a.tokens < 2 * 148) a.tokens /= 2;
}
// rows of a tile, `step` groups at a time
void walk_of(Args& a, int rows, int step) {
  a.step_tk = step / rows;
  a.step_h = step % rows;
  a.rows_inverse = rows > 1 ? (uint32_t)(((1ull << 32) + rows - 1) / rows) : 0u;
  a.half_inverse = a.rot > 2 ? (uint32_t)(((1ull << 32) + a.rot / 2 - 1) / (a.rot / 2)) : 0u;
}
size_t smem_of(const Args& a) { return (size_t)lanes_of(a.d) * 16 * sizeof(float) + (size_t)a.tokens * (a.rot / 2) * sizeof(float2); }

constexpr int kParts = 148 * kBackCtas;

int forward(Args& a, int bf16, bool cache, cudaStream_t stream) {
  if (bad_shape(a)) return RB_ERR_UNSUPPORTED;
  const int rows = a.r[0].heads + a.r[1].heads * (cache ? 2 : 1);
  if (a.n <= 0 || rows == 0) return RB_OK;
  a.inv_d = 1.f / a.d;
  if (fits(a, bf16, false, cache)) {
    tile_of(a);
    const int groups = kThreads / lanes_of(a.d);
    const int64_t gx = (a.n + a.tokens - 1) / a.tokens;
    int gy = 1;  // where tokens are few their rows are shared by several CTAs
    while (gx * gy < 148 && gy * groups < a.tokens * rows) gy *= 2;
    walk_of(a, rows, gy * groups);
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
  if (!norm && (n <= 0 || rows == 0)) return RB_OK;
  a.inv_d = 1.f / d;
  int64_t grid;  // (without any row one CTA leaves sums of zero)
  if (fits(a, bf16, true, false)) {
    tile_of(a);
    walk_of(a, std::max(rows, 1), kThreads / lanes_of(d));
    grid = std::max<int64_t>(1, std::min<int64_t>((n + a.tokens - 1) / a.tokens, kParts));
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
    rb_launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), std::max(smem_of(a), sums), stream, a);
  } else {
    grid = std::max<int64_t>(1, std::min<int64_t>((n * rows + kThreads / 32 - 1) / (kThreads / 32), kParts));
    auto kernel = bf16 ? backward_any_kernel<__nv_bfloat16> : backward_any_kernel<float>;
    rb_launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  }
  if (norm) rb_launch_pdl(weight_sum_kernel, dim3((2 * d + 31) / 32), dim3(kSumWarps * 32), 0, stream, (const float*)part, (int)grid, d, dwq, dwk, w_bf16);
  return rb_check_launch("norm_rope_bwd");
}
