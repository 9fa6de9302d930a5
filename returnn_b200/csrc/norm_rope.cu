// Norm per head and rotary positions of queries and keys in one pass, with its gradient and a form that leaves keys and values in a paged cache.
//   y = w x / sqrt(mean x^2 + eps) per (token, head) row of D features (without a norm: y = x)
//   z = c R(p f) y on the first R features, whose pairs (a, b) are (2i, 2i + 1) or (i, i + R / 2):
//       a' = c (a cos t - b sin t), b' = c (a sin t + b cos t), t = p f_i for the token's position p; the other features stay.
// Backward: dy = c R(-t) dz; with u = x / sqrt(mean x^2 + eps): dx = (dy w - u mean(dy w u)) / sqrt(mean x^2 + eps), dw = sum dy u.
//
// The angle of a far position does not fit the 24 bits of a float (position 100000 would be off by 0.004 of a radian): p f / (2 pi) is taken in 64
// bits, its whole turns dropped, and the sine and cosine of the rest taken in 32. One pair of them per (token, pair of features) serves all heads,
// so a CTA owns whole tokens and keeps the table of its tokens in shared memory.
// Rows are read once and written once. A row of D features sits in the next power of two of D / 8 lanes, 8 features (16 bytes of bf16) a lane: the mean
// is a few shuffles, pairs (2i, 2i + 1) are a lane's own, pairs (i, i + R / 2) one shuffle away. Head dims, rotated parts and alignments that do
// not fit this take a warp per row with single elements.
#include "common.cuh"
#include <algorithm>
#include <initializer_list>

namespace {

constexpr int kMaxDim = 256;
constexpr int kThreads = 256;

struct Args {
  const void *q, *k, *v;            // forward: inputs. backward: x of the norm (null without one)
  const void *dq, *dk;              // backward: incoming gradients
  void *out_q, *out_k;              // [N, Hq, D], [N, Hk, D]
  void *cache_k, *cache_v;          // cache form: where k and v go
  const void *positions;            // [num_pos], token t has number t % num_pos
  const float* freq;                // [R / 2]
  const void *wq, *wk;              // [D] or null
  float* part;                      // backward: [gridDim.x][2][D] partial sums of dw
  const int* slots;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, dq_tok, dq_head, dk_tok, dk_head;
  int64_t ck_page, ck_head, ck_tok, cv_page, cv_head, cv_tok;
  int64_t num_slots, num_pos;
  int64_t n;
  int hq, hk, d, rot, page, pos64, w_bf16, interleaved, tokens_per_cta;
  float eps, amp;
};

__device__ __forceinline__ float2 turn_of(const Args& a, int64_t token, int i) {
  if (a.num_pos < a.n) token %= a.num_pos;
  const int64_t p = a.pos64 ? reinterpret_cast<const long long*>(a.positions)[token] : reinterpret_cast<const int*>(a.positions)[token];
  double t = (double)p * (double)a.freq[i] * 0.15915494309189533577;  // turns
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

// where row `head` of `token` goes in the cache form; -1: nowhere (a token without a slot)
__device__ __forceinline__ int64_t cache_at(const Args& a, int64_t token, int head, int64_t page_stride, int64_t head_stride, int64_t tok_stride) {
  const int64_t slot = a.slots[token];
  if (slot < 0 || slot >= a.num_slots) return -1;
  const int64_t pg = slot / a.page;
  return pg * page_stride + head * head_stride + (slot - pg * a.page) * tok_stride;
}

// the 8 features of this lane turned by the token's angles (sign -1: back)
template <bool kInter>
__device__ __forceinline__ void rotate8(F8& x, const float2* tab, int sub, int rot, float sign) {
  const int e0 = sub * 8;
  if (kInter) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (e0 + 2 * j < rot) {
        const float2 t = tab[(e0 >> 1) + j];
        const float p = x.v[2 * j], r = x.v[2 * j + 1], s = t.y * sign;
        x.v[2 * j] = p * t.x - r * s;
        x.v[2 * j + 1] = p * s + r * t.x;
      }
    }
  } else {
    const int half = rot >> 1, step = half >> 3;  // half is a multiple of 8 here
    const bool first = e0 < half, in = e0 < rot;
    const int lane = threadIdx.x & 31;
    const int src = in ? (first ? lane + step : lane - step) : lane;
    const float s = first ? -sign : sign;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float other = __shfl_sync(0xffffffffu, x.v[j], src);
      if (in) {
        const float2 t = tab[(first ? e0 : e0 - half) + j];
        x.v[j] = x.v[j] * t.x + other * t.y * s;
      }
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float squares(const F8& x) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += x.v[j] * x.v[j];
  return s;
}

template <typename T, bool kInter, bool kCache>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const Args a, int lanes) {
  extern __shared__ float2 table[];  // [tokens_per_cta][R / 2]
  rb_pdl_wait();
  rb_pdl_launch();
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_cta;
  const int nt = (int)min((int64_t)a.tokens_per_cta, a.n - t0);
  const int half = a.rot >> 1;
  for (int i = threadIdx.x; i < nt * half; i += kThreads) table[i] = turn_of(a, t0 + i / half, i % half);
  __syncthreads();
  const int sub = threadIdx.x & (lanes - 1);
  const bool real = sub * 8 < a.d;
  const bool norm = a.wq != nullptr;
  F8 wq, wk;
  if (norm && real) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wq.v[j] = weight_at(a.wq, sub * 8 + j, a.w_bf16);
      wk.v[j] = weight_at(a.wk, sub * 8 + j, a.w_bf16);
    }
  }
  const int rows = a.hq + a.hk + (kCache ? a.hk : 0);
  const int groups = kThreads / lanes;
  const int total = nt * rows;
  // (all lanes of a warp go round together: the shuffles want them)
  for (int r0 = blockIdx.y * groups; r0 < total; r0 += gridDim.y * groups) {
    const int r = r0 + threadIdx.x / lanes;
    const bool live = r < total && real;
    const int tk = live ? r / rows : 0;
    const int h = live ? r - tk * rows : 0;
    const int64_t token = t0 + tk;
    F8 x = {};
    if (live) {
      if (h < a.hq) x = load8(a.q, token * a.q_tok + h * a.q_head + sub * 8, is_bf16<T>());
      else if (h < a.hq + a.hk) x = load8(a.k, token * a.k_tok + (h - a.hq) * a.k_head + sub * 8, is_bf16<T>());
      else x = load8(a.v, token * a.v_tok + (h - a.hq - a.hk) * a.v_head + sub * 8, is_bf16<T>());
    }
    const bool value = kCache && h >= a.hq + a.hk;
    if (norm) {
      const float inv = rsqrtf(group_sum(squares(x), lanes) / a.d + a.eps);
      if (live && !value) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x.v[j] *= inv * (h < a.hq ? wq.v[j] : wk.v[j]);
      }
    }
    F8 y = x;
    rotate8<kInter>(y, table + tk * half, sub, a.rot, 1.f);
    if (!live) continue;
    if (h < a.hq) {
      store8(a.out_q, (token * a.hq + h) * a.d + sub * 8, y, is_bf16<T>());
    } else if (!kCache) {
      store8(a.out_k, (token * a.hk + h - a.hq) * a.d + sub * 8, y, is_bf16<T>());
    } else if (!value) {
      const int64_t at = cache_at(a, token, h - a.hq, a.ck_page, a.ck_head, a.ck_tok);
      if (at >= 0) store8(a.cache_k, at + sub * 8, y, is_bf16<T>());
    } else {
      const int64_t at = cache_at(a, token, h - a.hq - a.hk, a.cv_page, a.cv_head, a.cv_tok);
      if (at >= 0) store8(a.cache_v, at + sub * 8, x, is_bf16<T>());
    }
  }
}

// kNorm: x is read again and the weights have gradients (sums per CTA, added up in order by the kernel below)
template <typename T, bool kInter, bool kNorm>
__global__ void __launch_bounds__(kThreads)
backward_kernel(const Args a, int lanes) {
  extern __shared__ float2 table[];
  rb_pdl_wait();
  rb_pdl_launch();
  const int half = a.rot >> 1;
  const int sub = threadIdx.x & (lanes - 1);
  const bool real = sub * 8 < a.d;
  F8 wq = {}, wk = {}, gq = {}, gk = {};
  if (kNorm && real) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wq.v[j] = weight_at(a.wq, sub * 8 + j, a.w_bf16);
      wk.v[j] = weight_at(a.wk, sub * 8 + j, a.w_bf16);
    }
  }
  const int rows = a.hq + a.hk;
  const int groups = kThreads / lanes;
  for (int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_cta; t0 < a.n; t0 += (int64_t)gridDim.x * a.tokens_per_cta) {
    const int nt = (int)min((int64_t)a.tokens_per_cta, a.n - t0);
    __syncthreads();
    for (int i = threadIdx.x; i < nt * half; i += kThreads) table[i] = turn_of(a, t0 + i / half, i % half);
    __syncthreads();
    const int total = nt * rows;
    for (int r0 = 0; r0 < total; r0 += groups) {
      const int r = r0 + threadIdx.x / lanes;
      const bool live = r < total && real;
      const int tk = live ? r / rows : 0;
      const int h = live ? r - tk * rows : 0;
      const int64_t token = t0 + tk;
      const bool is_q = h < a.hq;
      F8 g = {}, x = {};
      if (live) {
        g = is_q ? load8(a.dq, token * a.dq_tok + h * a.dq_head + sub * 8, is_bf16<T>())
                 : load8(a.dk, token * a.dk_tok + (h - a.hq) * a.dk_head + sub * 8, is_bf16<T>());
        if (kNorm) x = is_q ? load8(a.q, token * a.q_tok + h * a.q_head + sub * 8, is_bf16<T>())
                            : load8(a.k, token * a.k_tok + (h - a.hq) * a.k_head + sub * 8, is_bf16<T>());
      }
      rotate8<kInter>(g, table + tk * half, sub, a.rot, -1.f);
      if (kNorm) {
        const float inv = rsqrtf(group_sum(squares(x), lanes) / a.d + a.eps);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x.v[j] *= inv;
          const float c = g.v[j] * x.v[j];  // (zeros in idle lanes)
          if (is_q) gq.v[j] += c; else gk.v[j] += c;
          g.v[j] *= is_q ? wq.v[j] : wk.v[j];
          dot += g.v[j] * x.v[j];
        }
        dot = group_sum(dot, lanes) / a.d;
#pragma unroll
        for (int j = 0; j < 8; ++j) g.v[j] = inv * (g.v[j] - x.v[j] * dot);
      }
      if (live) {
        if (is_q) store8(a.out_q, (token * a.hq + h) * a.d + sub * 8, g, is_bf16<T>());
        else store8(a.out_k, (token * a.hk + h - a.hq) * a.d + sub * 8, g, is_bf16<T>());
      }
    }
  }
  if (kNorm) {
    float* sums = reinterpret_cast<float*>(table);  // [groups][2][lanes * 8]; at least as large as this (see the launch)
    __syncthreads();
    float* mine = sums + (threadIdx.x / lanes) * 2 * lanes * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mine[sub * 8 + j] = gq.v[j];
      mine[lanes * 8 + sub * 8 + j] = gk.v[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
      const int at = i < a.d ? i : lanes * 8 + i - a.d;
      float s = 0.f;
      for (int g = 0; g < groups; ++g) s += sums[g * 2 * lanes * 8 + at];
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
  const int rows = a.hq + a.hk + (kCache ? a.hk : 0);
  const int64_t total = a.n * rows;
  rb_pdl_wait();
  rb_pdl_launch();
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); r < total; r += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t token = r / rows;
    const int h = (int)(r - token * rows);
    const bool is_q = h < a.hq, value = h >= a.hq + a.hk;
    const void* x = is_q ? a.q : value ? a.v : a.k;
    const int64_t base = is_q ? token * a.q_tok + h * a.q_head
                              : value ? token * a.v_tok + (h - a.hq - a.hk) * a.v_head : token * a.k_tok + (h - a.hq) * a.k_head;
    const void* w = is_q ? a.wq : a.wk;
    float inv = 1.f;
    if (w && !value) {
      float s = 0.f;
      for (int e = lane; e < a.d; e += 32) {
        const float f = one<T>(x, base + e);
        s += f * f;
      }
      inv = rsqrtf(warp_sum(s) / a.d + a.eps);
    }
    void* out = is_q ? a.out_q : kCache ? (value ? a.cache_v : a.cache_k) : a.out_k;
    int64_t to;
    if (is_q) to = (token * a.hq + h) * a.d;
    else if (!kCache) to = (token * a.hk + h - a.hq) * a.d;
    else if (!value) to = cache_at(a, token, h - a.hq, a.ck_page, a.ck_head, a.ck_tok);
    else to = cache_at(a, token, h - a.hq - a.hk, a.cv_page, a.cv_head, a.cv_tok);
    if (to < 0) continue;
    for (int e = lane; e < a.d; e += 32) {
      float y = one<T>(x, base + e);
      if (!value) {
        if (w) y *= inv * weight_at(w, e, a.w_bf16);
        if (e < a.rot) {
          int pair;
          float sign;
          const int o = partner(e, a.rot, a.interleaved, &pair, &sign);
          float other = one<T>(x, base + o);
          if (w) other *= inv * weight_at(w, o, a.w_bf16);
          const float2 t = turn_of(a, token, pair);
          y = y * t.x + sign * other * t.y;
        }
      }
      put<T>(out, to + e, y);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
backward_any_kernel(const Args a) {
  __shared__ float sums[kThreads / 32][2][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = a.hq + a.hk;
  const int64_t total = a.n * rows;
  const bool norm = a.wq != nullptr;
  rb_pdl_wait();
  rb_pdl_launch();
  float gq[kMaxDim / 32] = {}, gk[kMaxDim / 32] = {};
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + warp; r < total; r += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t token = r / rows;
    const int h = (int)(r - token * rows);
    const bool is_q = h < a.hq;
    const void* g = is_q ? a.dq : a.dk;
    const int64_t gb = is_q ? token * a.dq_tok + h * a.dq_head : token * a.dk_tok + (h - a.hq) * a.dk_head;
    const void* x = is_q ? a.q : a.k;
    const int64_t xb = is_q ? token * a.q_tok + h * a.q_head : token * a.k_tok + (h - a.hq) * a.k_head;
    const void* w = is_q ? a.wq : a.wk;
    void* out = is_q ? a.out_q : a.out_k;
    const int64_t to = is_q ? (token * a.hq + h) * a.d : (token * a.hk + h - a.hq) * a.d;
    float inv = 1.f, dot = 0.f;
    float dy[kMaxDim / 32], u[kMaxDim / 32];
    if (norm) {
      float s = 0.f;
      for (int e = lane; e < a.d; e += 32) {
        const float f = one<T>(x, xb + e);
        s += f * f;
      }
      inv = rsqrtf(warp_sum(s) / a.d + a.eps);
    }
#pragma unroll
    for (int j = 0; j < kMaxDim / 32; ++j) {
      const int e = lane + 32 * j;
      dy[j] = u[j] = 0.f;
      if (e >= a.d) continue;
      dy[j] = one<T>(g, gb + e);
      if (e < a.rot) {
        int pair;
        float sign;
        const int o = partner(e, a.rot, a.interleaved, &pair, &sign);
        const float2 t = turn_of(a, token, pair);
        dy[j] = dy[j] * t.x - sign * one<T>(g, gb + o) * t.y;
      }
      if (norm) {
        u[j] = one<T>(x, xb + e) * inv;
        if (is_q) gq[j] += dy[j] * u[j]; else gk[j] += dy[j] * u[j];
        dy[j] *= weight_at(w, e, a.w_bf16);
        dot += dy[j] * u[j];
      }
    }
    if (norm) dot = warp_sum(dot) / a.d;
#pragma unroll
    for (int j = 0; j < kMaxDim / 32; ++j) {
      const int e = lane + 32 * j;
      if (e < a.d) put<T>(out, to + e, norm ? inv * (dy[j] - u[j] * dot) : dy[j]);
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

// the partial sums of all CTAs in order -> gradients in the type of the weights. A CTA has 32 columns, its warps a stretch of the rows each.
__global__ void __launch_bounds__(256)
weight_sum_kernel(const float* __restrict__ part, int parts, int d, void* __restrict__ dwq, void* __restrict__ dwk, int w_bf16) {
  __shared__ float sh[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  rb_pdl_wait();
  rb_pdl_launch();
  float s = 0.f;
  if (col < 2 * d) {
    const int each = (parts + 7) / 8;
    const int end = min(parts, (warp + 1) * each);
#pragma unroll 8
    for (int p = warp * each; p < end; ++p) s += part[(int64_t)p * 2 * d + col];
  }
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < 2 * d) {
#pragma unroll
    for (int w = 1; w < 8; ++w) s += sh[w][lane];
    void* out = col < d ? dwq : dwk;
    const int at = col < d ? col : col - d;
    if (w_bf16) put<__nv_bfloat16>(out, at, s);
    else put<float>(out, at, s);
  }
}

int lanes_of(int d) {
  int l = 1;
  while (l * 8 < d) l *= 2;
  return l;
}

bool aligned(const void* p, std::initializer_list<int64_t> strides, int unit) {
  if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  for (int64_t s : strides)
    if (s % unit) return false;
  return true;
}

int bad_shape(const Args& a, int backward) {
  if (a.d < 1 || a.d > kMaxDim || a.rot < 0 || a.rot > a.d || a.rot % 2 || a.hq < 0 || a.hk < 0) {
    rb_set_error("norm_rope%s: head dim %d (1 to %d), rotated part %d (even, at most the head dim)", backward ? " backward" : "", a.d, kMaxDim, a.rot);
    return 1;
  }
  return 0;
}

// 8 features a lane: whole groups of 8, rotated pairs within a lane or a whole number of lanes apart, 16-byte accesses
bool fits(const Args& a, int bf16, bool backward, bool cache) {
  const int unit = bf16 ? 8 : 4;
  if (a.d % 8 || (!a.interleaved && a.rot % 16)) return false;
  bool ok = aligned(a.out_q, {}, unit);
  if (backward) ok = ok && aligned(a.dq, {a.dq_tok, a.dq_head}, unit) && aligned(a.dk, {a.dk_tok, a.dk_head}, unit) && aligned(a.out_k, {}, unit);
  if (!backward || a.wq) ok = ok && aligned(a.q, {a.q_tok, a.q_head}, unit) && aligned(a.k, {a.k_tok, a.k_head}, unit);
  if (cache)
    ok = ok && aligned(a.v, {a.v_tok, a.v_head}, unit) && aligned(a.cache_k, {a.ck_page, a.ck_head, a.ck_tok}, unit) &&
         aligned(a.cache_v, {a.cv_page, a.cv_head, a.cv_tok}, unit);
  else if (!backward) ok = ok && aligned(a.out_k, {}, unit);
  return ok;
}

int forward(Args& a, int bf16, bool cache, cudaStream_t stream) {
  if (bad_shape(a, 0)) return RB_ERR_UNSUPPORTED;
  const int rows = a.hq + a.hk * (cache ? 2 : 1);
  if (a.n <= 0 || rows == 0) return RB_OK;
  if (fits(a, bf16, false, cache)) {
    const int lanes = lanes_of(a.d), groups = kThreads / lanes, half = a.rot / 2;
    // a table entry or two per thread, fewer tokens where that leaves SMs without any; then the rows of a token are shared by several CTAs too
    int tb = half ? max(1, kThreads / half) : 8;
    while (tb > 1 && (a.n + tb - 1) / tb < 2 * 148) tb /= 2;
    a.tokens_per_cta = tb;
    const int64_t gx = (a.n + tb - 1) / tb;
    int gy = 1;
    while (gx * gy < 148 && gy * groups * 2 <= tb * rows) gy *= 2;
    if (gx > 0x7fffffff) {
      rb_set_error("norm_rope: %lld tokens", (long long)a.n);
      return RB_ERR_UNSUPPORTED;
    }
    auto pick = [&](auto t) {
      using T = decltype(t);
      return a.interleaved ? (cache ? forward_kernel<T, true, true> : forward_kernel<T, true, false>)
                           : (cache ? forward_kernel<T, false, true> : forward_kernel<T, false, false>);
    };
    auto kernel = bf16 ? pick(__nv_bfloat16()) : pick(float());
    rb_launch_pdl(kernel, dim3((unsigned)gx, gy), dim3(kThreads), (size_t)tb * half * sizeof(float2), stream, a, lanes);
  } else {
    const int64_t ctas = (a.n * rows + kThreads / 32 - 1) / (kThreads / 32);
    auto kernel = bf16 ? (cache ? forward_any_kernel<__nv_bfloat16, true> : forward_any_kernel<__nv_bfloat16, false>)
                       : (cache ? forward_any_kernel<float, true> : forward_any_kernel<float, false>);
    rb_launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(ctas, 148 * 8)), dim3(kThreads), 0, stream, a);
  }
  return rb_check_launch("norm_rope");
}

}  // namespace

RB_EXPORT int rb200_norm_rope_fwd(const void* q, const void* k, const void* positions, long long num_pos, const float* freq, const void* wq, const void* wk, void* out_q,
                                  void* out_k, const long long* strides /* q token, q head, k token, k head */, long long n, int hq, int hk, int d, int rot,
                                  int bf16, int pos64, int w_bf16, int interleaved, float eps, float amp, cudaStream_t stream) {
  Args a = {};
  a.q = q; a.k = k; a.positions = positions; a.num_pos = num_pos; a.freq = freq; a.wq = wq; a.wk = wk; a.out_q = out_q; a.out_k = out_k;
  a.q_tok = strides[0]; a.q_head = strides[1]; a.k_tok = strides[2]; a.k_head = strides[3];
  a.n = n; a.hq = hq; a.hk = hk; a.d = d; a.rot = rot; a.pos64 = pos64; a.w_bf16 = w_bf16; a.interleaved = interleaved; a.eps = eps; a.amp = amp;
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
  a.q = q; a.k = k; a.v = v; a.positions = positions; a.num_pos = num_pos; a.freq = freq; a.wq = wq; a.wk = wk; a.out_q = out_q;
  a.cache_k = cache_k; a.cache_v = cache_v; a.slots = slots; a.page = page; a.num_slots = num_slots;
  a.q_tok = strides[0]; a.q_head = strides[1]; a.k_tok = strides[2]; a.k_head = strides[3]; a.v_tok = strides[4]; a.v_head = strides[5];
  a.ck_page = strides[6]; a.ck_head = strides[7]; a.ck_tok = strides[8]; a.cv_page = strides[9]; a.cv_head = strides[10]; a.cv_tok = strides[11];
  a.n = n; a.hq = hq; a.hk = hk; a.d = d; a.rot = rot; a.pos64 = pos64; a.w_bf16 = w_bf16; a.interleaved = interleaved; a.eps = eps; a.amp = amp;
  return forward(a, bf16, true, stream);
}

// partial sums that the backward pass leaves: rows of 2 D floats
RB_EXPORT int rb200_norm_rope_parts() { return 148 * 4; }

// part: [rb200_norm_rope_parts()][2][D] floats with a norm, else unused; dwq, dwk [D] in the type of the weights
RB_EXPORT int rb200_norm_rope_bwd(const void* dq, const void* dk, const void* q, const void* k, const void* positions, long long num_pos, const float* freq, const void* wq,
                                  const void* wk, void* out_q, void* out_k, float* part, void* dwq, void* dwk,
                                  const long long* strides /* dq, dk, q, k: token, head */, long long n, int hq, int hk, int d, int rot, int bf16, int pos64,
                                  int w_bf16, int interleaved, float eps, float amp, cudaStream_t stream) {
  Args a = {};
  a.dq = dq; a.dk = dk; a.q = q; a.k = k; a.positions = positions; a.num_pos = num_pos; a.freq = freq; a.wq = wq; a.wk = wk; a.out_q = out_q; a.out_k = out_k; a.part = part;
  a.dq_tok = strides[0]; a.dq_head = strides[1]; a.dk_tok = strides[2]; a.dk_head = strides[3];
  a.q_tok = strides[4]; a.q_head = strides[5]; a.k_tok = strides[6]; a.k_head = strides[7];
  a.n = n; a.hq = hq; a.hk = hk; a.d = d; a.rot = rot; a.pos64 = pos64; a.w_bf16 = w_bf16; a.interleaved = interleaved; a.eps = eps; a.amp = amp;
  if (bad_shape(a, 1)) return RB_ERR_UNSUPPORTED;
  const bool norm = wq != nullptr;
  const int rows = hq + hk;
  if (!norm && (n <= 0 || rows == 0)) return RB_OK;
  int64_t grid;  // (without any row one CTA leaves sums of zero)
  if (fits(a, bf16, true, false)) {
    const int lanes = lanes_of(d), half = rot / 2;
    int tb = half ? max(1, kThreads / half) : 8;
    while (tb > 1 && (n + tb - 1) / tb < 2 * 148) tb /= 2;
    a.tokens_per_cta = tb;
    grid = std::max<int64_t>(1, (n + tb - 1) / tb);
    if (norm) grid = std::min<int64_t>(grid, rb200_norm_rope_parts());
    grid = std::min<int64_t>(grid, 0x7fffffff);
    const size_t table = (size_t)tb * half * sizeof(float2), sums = norm ? (size_t)kThreads * 2 * 8 * sizeof(float) : 0;
    auto pick = [&](auto t) {
      using T = decltype(t);
      return interleaved ? (norm ? backward_kernel<T, true, true> : backward_kernel<T, true, false>)
                         : (norm ? backward_kernel<T, false, true> : backward_kernel<T, false, false>);
    };
    auto kernel = bf16 ? pick(__nv_bfloat16()) : pick(float());
    rb_launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), std::max(table, sums), stream, a, lanes);
  } else {
    grid = std::max<int64_t>(1, std::min<int64_t>((n * rows + kThreads / 32 - 1) / (kThreads / 32), rb200_norm_rope_parts()));
    auto kernel = bf16 ? backward_any_kernel<__nv_bfloat16> : backward_any_kernel<float>;
    rb_launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  }
  if (norm) rb_launch_pdl(weight_sum_kernel, dim3((2 * d + 31) / 32), dim3(256), 0, stream, (const float*)part, (int)grid, d, dwq, dwk, w_bf16);
  return rb_check_launch("norm_rope_bwd");
}
