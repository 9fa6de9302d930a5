// Log probabilities of given tokens over rows of logits, with the entropy of each row and its K best labels, and the gradient of all three.
//   with the maximum m: S = sum exp(x - m), lp = (x_y - m) - log S, H = log S - sum exp(x - m) (x - m) / S  (differences to the maximum: no cancellation)
//   best: the K largest logits, the lowest label first among equal ones (NaN counts as the largest), as log probabilities
//   dx_j = g (d_jy - p_j) + sum_k g_k (d_j,best_k - p_j) - g_H p_j (log p_j + H)
// A target outside 0 .. V - 1 has log probability 0 and no gradient of it. A label of logit -inf has probability 0; a row of nothing else has entropy 0,
// log probabilities -inf and no gradient.
//
// Forward: one CTA per row, one pass with a running maximum, sum and sum of exp(z) z; the logits are read once. A label costs an exponential and, by packed
// arithmetic, five more instructions; they are what bounds rows of bf16 next to the memory. The K best come without a sort and almost without a second
// read: the K-th largest of the maxima of 32 groups of threads bounds the K-th largest logit from below, so that only the threads whose maximum reaches the bound
// have their logits looked through again, and the few logits above it are ranked by counting.
// Backward: one pass, p from the maximum and the sum; the labels that have a gradient of their own are written once more at the end.
#include "class_rows.cuh"
#include "packed_f32.cuh"
#include <algorithm>
#include <type_traits>

namespace {

using rows::Chunk;
using rows::ld;
using rows::row_head;

constexpr int kBack = 256;  // threads of the backward pass
constexpr int kMaxTop = 32;
constexpr int kCand = 512;  // logits that are ranked
// Up to this many best the bound comes from 32 groups of threads (32 shuffles; 12 of 32 are reached by 15 logits on the average, 24 by 44), beyond from the threads
// themselves (a search bit by bit, two microseconds of one warp; 32 of 32 groups would be reached by 130). Few rows wait for the search, many for the instructions.
// Groups and threads, us: 1500 rows x 10001 fp32, 8 best 16.0 and 17.0, 20 best 20.3 and 19.6, 28 best 27.1 and 21.5; 16 rows x 32000, 20 best 6.1 and 8.1, 24 best 6.5 and 8.1.
template <int kThreads, int kBatch>
constexpr int kFewTop = kThreads == 1024 || kBatch == 8 ? 24 : 12;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* x;
  int64_t pitch;
  const void* target;  // null: no log probabilities of tokens
  int target64, v, top;
  float *lp, *norm, *entropy, *top_lp;  // norm: [rows][2], the maximum m and log S
  int* top_label;
};

// order of the logits as whole numbers; NaN is the largest, -0 and what is below the normal numbers count as 0 (as for the maxima)
__device__ __forceinline__ uint32_t rank_of(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t a = __float_as_uint(f), u = (a & 0x7fffffffu) < 0x00800000u ? 0u : a;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ long long target_of(const Args& a, int64_t row) {
  return a.target64 ? reinterpret_cast<const long long*>(a.target)[row] : reinterpret_cast<const int*>(a.target)[row];
}

// running maximum, sum of e = exp(x - m), sum of e (x - m). Before the first logit above -inf the sums are 0 (or NaN).
struct Stat {
  float m, s, w;
  __device__ __forceinline__ void to(float nm) {
    if (m != -INFINITY) {
      const float d = m - nm, f = exp2f(d * kLog2e);
      w = f == 0.f ? 0.f * w : f * (w + s * d);  // (not 0 times a difference beyond the range; NaN stays)
      s *= f;
    }
    m = nm;
  }
};
// A logit so far below the maximum that its e is 0: with the entropy, logits are raised to it, so that e = 0 does not meet an infinity. Near the end of
// the range there is no such number, and the products are guarded one by one.
__device__ __forceinline__ bool is_far(float m) { return !(fabsf(m) < 1e38f); }
__device__ __forceinline__ float floor_of(float m) { return m - 1e4f - 0.01f * fabsf(m); }
// The difference to the maximum first: its exponent is 0 whatever its size, up to the type's lowest value. (One fused multiply-add, x / ln 2 - m / ln 2, would round
// the second product by 2^-24 of the maximum and overflow at the end of the range.)
template <bool kEntropy>
__device__ __forceinline__ void add(float x, float m, float& s, float& w) {
  const float z = x - m;
  const float e = exp2f(z * kLog2e);
  s += e;
  if (kEntropy) w += e == 0.f ? 0.f : e * z;
}
// the logits of a chunk as pairs, raised to `least`
template <bool kRaise>
__device__ __forceinline__ void in_pairs(const Chunk<true>& u, float least, uint64_t* p) {
  const uint32_t w[4] = {u.u.x, u.u.y, u.u.z, u.u.w};
  const __nv_bfloat162 f = __float2bfloat162_rn(least);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v = w[i];
    if (kRaise) {
      const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), f);
      v = *reinterpret_cast<const uint32_t*>(&r);
    }
    p[i] = two(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
}
template <bool kRaise>
__device__ __forceinline__ void in_pairs(const Chunk<false>& u, float least, uint64_t* p) {
#pragma unroll
  for (int i = 0; i < 2; ++i) p[i] = kRaise ? two(max_nan(u.at(2 * i), least), max_nan(u.at(2 * i + 1), least)) : two(u.at(2 * i), u.at(2 * i + 1));
}

// K-th largest of the CTA's whole numbers in shared memory, by one warp, bit by bit (`bits` leading ones may differ)
template <int kThreads>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* key, int k, int bits) {
  const int lane = threadIdx.x & 31;
  uint32_t found = 0;
  for (int b = 31; b >= 32 - bits; --b) {
    const uint32_t want = found | 1u << b;
    int n = 0;
    for (int j = 0; j < kThreads / 32; ++j) n += key[j * 32 + lane] >= want;
    if ((int)__reduce_add_sync(0xffffffffu, n) >= k) found = want;
  }
  return found;
}
// K-th largest of the 32 whole numbers of a warp
__device__ __forceinline__ uint32_t kth_of_warp(uint32_t mine, int k) {
  const int lane = threadIdx.x & 31;
  int above = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const uint32_t other = __shfl_sync(0xffffffffu, mine, j);
    above += other > mine || (other == mine && j < lane);
  }
  return __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, above == k - 1)) - 1);
}

struct Row {
  const void* x;
  int64_t base;
  int head, v8, v;
};

template <int kThreads>
struct Best {
  uint32_t key[kThreads], group[32];
  uint64_t cand[kCand];  // rank of the logit, and the label counted from above
  uint64_t last;
  uint32_t bound;
  int count, hits, found[kThreads / 32];
};

// orders logits by rank, then by label from the lowest; below ~0
__device__ __forceinline__ uint64_t composite(uint32_t rank, int label) { return (uint64_t)rank << 32 | (0xfffffffeu - (uint32_t)label); }
__device__ __forceinline__ int label_of(uint64_t c) { return (int)(0xfffffffeu - (uint32_t)c); }

template <int kThreads>
__device__ __forceinline__ void consider(Best<kThreads>& b, float x, int label) {
  const uint32_t r = rank_of(x);
  if (r >= b.bound) {
    const int at = atomicAdd(&b.count, 1);  // (the order does not matter: they are ranked)
    if (at < kCand) b.cand[at] = composite(r, label);
  }
}

// logits of the threads whose maximum reaches the bound, and those outside the chunks; given up where they are too many. b.count and b.hits are 0 before. All threads look
// the chunks of those threads through, two at a time: a warp for its own threads, one after another, waited for the memory at each (1500 x 10001 fp32, 8 best:
// 18.1 and 15.8 us; 2740 x 1001 fp32, 20 best: 22.9 and 12.4).
template <int kThreads, bool kBf16>
__device__ __forceinline__ void collect(Best<kThreads>& b, const Row& r, uint32_t key) {
  constexpr int kN = Chunk<kBf16>::kN, kAhead = 2;
  const int lane = threadIdx.x & 31;
  const uint32_t bound = b.bound, who = __ballot_sync(0xffffffffu, key >= bound);
  int at = 0;
  if (lane == 0 && who) at = atomicAdd(&b.hits, __popc(who));
  at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
  if (key >= bound) b.key[at] = threadIdx.x | (key == 0xffffffffu ? 1u << 31 : 0u);  // (a maximum passes a NaN by)
  const int rest = r.v - (r.v8 - r.head);
  if ((int)threadIdx.x < rest) {
    const int c = (int)threadIdx.x < r.head ? threadIdx.x : threadIdx.x + (r.v8 - r.head);
    consider(b, ld(r.x, r.base + c, kBf16), c);
  }
  __syncthreads();
  const int hits = b.hits, chunks = (r.v8 - r.head + kThreads * kN - 1) / (kThreads * kN);
  for (int i0 = threadIdx.x; i0 < hits * chunks && *(volatile int*)&b.count <= kCand; i0 += kAhead * kThreads) {
    Chunk<kBf16> u[kAhead];
    int c[kAhead];
    bool odd[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int i = i0 + q * kThreads, k = i / hits;
      const uint32_t t = k < chunks ? b.key[i - k * hits] : 0u;
      odd[q] = t >> 31;
      c[q] = r.head + ((int)(t & 0x7fffffffu) + kThreads * k) * kN;
      if (k < chunks && c[q] < r.v8) u[q].load(r.x, r.base + c[q]);
      else c[q] = -1;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (c[q] < 0 || (!odd[q] && rank_of(u[q].max()) < bound)) continue;
#pragma unroll
      for (int k = 0; k < kN; ++k) consider(b, u[q].at(k), c[q] + k);
    }
  }
}

// a thread's key: the rank of its largest logit (its chunks, and one outside). `odd`: its sum is no number, the maximum may be one.
template <int kThreads, bool kBf16>
__device__ __forceinline__ uint32_t key_of(const Row& r, float mx, bool odd) {
  uint32_t key = rank_of(mx);
  if (odd) {
    constexpr int kN = Chunk<kBf16>::kN;
    const int rest = r.v - (r.v8 - r.head);
    if ((int)threadIdx.x < rest) key = max(key, rank_of(ld(r.x, r.base + ((int)threadIdx.x < r.head ? threadIdx.x : threadIdx.x + (r.v8 - r.head)), kBf16)));
    for (int64_t c = r.head + (int)threadIdx.x * kN; c < r.v8; c += kThreads * kN)
      for (int k = 0; k < kN; ++k) key = max(key, rank_of(ld(r.x, r.base + c + k, kBf16)));
  }
  return key;
}

// K-th largest of the threads' keys, by the first warp
template <int kThreads, bool kBf16>
__device__ __forceinline__ uint32_t bound_of_threads(const Best<kThreads>& b, int top) {
  // (the lower half of a bf16 value's rank follows from the upper: zeros, ones where the value is negative or no number)
  uint32_t bound = kth_largest<kThreads>(b.key, top, kBf16 ? 16 : 32);
  if (kBf16 && (bound < 0x80000000u || bound == 0xffff0000u)) bound |= 0xffffu;
  return bound;
}

// The K best labels of a row in b.cand, in no order; returns how many there are (at least K, all above the K-th and itself among them). b.bound: at most the rank of the
// K-th largest logit; b.count, b.hits: 0
template <int kThreads, bool kBf16>
__device__ int select(Best<kThreads>& b, const Row& r, int top, uint32_t key) {
  collect<kThreads, kBf16>(b, r, key);
  __syncthreads();
  if (b.count <= kCand) return b.count;
  // Many equal logits at the bound (masks), or large ones in few groups. With the K-th largest of the threads' maxima as the bound, the logits above it lie in fewer than K
  // threads; of those equal to it the lowest labels are taken, in order, a stretch of labels after another.
  __syncthreads();
  b.key[threadIdx.x] = key;
  if (threadIdx.x == 0) b.count = b.hits = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    const uint32_t bound = bound_of_threads<kThreads, kBf16>(b, top);
    if (threadIdx.x == 0) b.bound = bound;
  }
  __syncthreads();
  const uint32_t bound = b.bound;
  __syncthreads();
  if (threadIdx.x == 0) b.bound = bound + 1;
  __syncthreads();
  if (bound != 0xffffffffu) collect<kThreads, kBf16>(b, r, key);  // (nothing is above a NaN)
  __syncthreads();
  int have = b.count;
  if (have <= kCand) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int c0 = 0; c0 < r.v && have < top; c0 += kThreads) {
      const int c = c0 + threadIdx.x;
      const uint32_t yes = __ballot_sync(0xffffffffu, c < r.v && rank_of(ld(r.x, r.base + c, kBf16)) == bound);
      if (lane == 0) b.found[warp] = __popc(yes);
      __syncthreads();
      int at = have, all = have;
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) at += b.found[w];
        all += b.found[w];
      }
      at += __popc(yes & ((1u << lane) - 1u));
      if ((yes >> lane & 1) && at < top) b.cand[at] = composite(bound, c);
      have = all;
      __syncthreads();
    }
    return min(have, max(b.count, top));
  }
  // more logits above the bound than are ranked (all in few threads' share): the K best one after another
  uint64_t before = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int c = threadIdx.x; c < r.v; c += kThreads) {
      const uint64_t q = composite(rank_of(ld(r.x, r.base + c, kBf16)), c);
      if (q < before && q > best) best = q;
    }
    __syncthreads();
    if (threadIdx.x == 0) b.last = 0;
    __syncthreads();
    atomicMax(reinterpret_cast<unsigned long long*>(&b.last), (unsigned long long)best);
    __syncthreads();
    before = b.last;
    if (threadIdx.x == 0) b.cand[k] = before;
  }
  __syncthreads();
  return top;
}

__device__ __forceinline__ float value_of(uint64_t c) {
  const uint32_t r = (uint32_t)(c >> 32);
  return __uint_as_float(r & 0x80000000u ? r & 0x7fffffffu : ~r);  // (NaN: the largest rank is a NaN again)
}

__device__ __forceinline__ float log_prob(float x, float2 norm) {
  return x == -INFINITY && norm.y == norm.y ? -INFINITY : (x - norm.x) - norm.y;
}

// kBatch: chunks of 16 bytes that a thread has in flight
template <int kThreads, bool kBf16, bool kEntropy, bool kTop, int kBatch>
__global__ void __launch_bounds__(kThreads, kThreads == 1024 ? 1 : kBatch == 8 ? 4 : 1536 / kThreads)
forward_kernel(const Args a) {
  constexpr int kN = Chunk<kBf16>::kN, kWarps = kThreads / 32;
  __shared__ float sh_m[kWarps], sh_s[kWarps], sh_w[kWarps];
  __shared__ float2 sh_norm;
  __shared__ Best<kTop ? kThreads : 32> best;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  rb_pdl_wait();
  rb_pdl_launch();
  Row r;
  r.x = a.x;
  r.base = row * a.pitch;
  r.v = a.v;
  r.head = row_head(a.x, r.base, a.v, kBf16 ? 2 : 4);
  r.v8 = r.head + ((a.v - r.head) & ~7);
  // asked for early, used late: the target's logit (by the thread that finishes the sums), the logits outside the chunks
  constexpr int kLast = 32;  // of the second warp; the first one looks for the bound
  long long y = -1;
  float xy = 0.f, xr = 0.f;
  if (threadIdx.x == kLast && a.target) {
    y = target_of(a, row);
    if (y >= 0 && y < a.v) xy = ld(a.x, r.base + y, kBf16);
  }
  const int rest = a.v - (r.v8 - r.head);  // fewer than the threads
  if ((int)threadIdx.x < rest) xr = ld(a.x, r.base + ((int)threadIdx.x < r.head ? threadIdx.x : threadIdx.x + (r.v8 - r.head)), kBf16);
  Stat st{-INFINITY, 0.f, 0.f};
  // kAll: every piece lies in the row
  auto batch = [&](int64_t c0, auto all) {
    constexpr bool kAll = decltype(all)::value;
    Chunk<kBf16> u[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int64_t c = c0 + q * kThreads * kN;
      if (kAll || c < r.v8) u[q].load(a.x, r.base + c);
      else u[q].fill_neg_inf();
    }
    float lm = u[0].max();
#pragma unroll
    for (int q = 1; q < kBatch; ++q) lm = fmaxf(lm, u[q].max());
    if (lm > st.m) st.to(lm);
    const float m = st.m == -INFINITY ? 0.f : st.m;
    if (!is_far(m)) {
      const float least = kEntropy ? floor_of(m) : 0.f;
      const uint64_t minus = two(-m, -m), l2 = two(kLog2e, kLog2e);
      uint64_t s = 0, w = 0;
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        if (kAll || q == 0 || c0 + q * kThreads * kN < r.v8) {
          uint64_t p[kN / 2];
          in_pairs<kEntropy>(u[q], least, p);
#pragma unroll
          for (int k = 0; k < kN / 2; ++k) {
            const uint64_t z = add2(p[k], minus);
            float t0, t1;
            split(mul2(z, l2), t0, t1);
            const uint64_t e = two(exp2f(t0), exp2f(t1));
            s = add2(s, e);
            if (kEntropy) w = fma2(e, z, w);
          }
        }
      }
      float s0, s1;
      split(s, s0, s1);
      st.s += s0 + s1;
      if (kEntropy) {
        split(w, s0, s1);
        st.w += s0 + s1;
      }
    } else {
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (kAll || q == 0 || c0 + q * kThreads * kN < r.v8)
          for (int k = 0; k < kN; ++k) add<kEntropy>(u[q].at(k), m, st.s, st.w);
    }
  };
  int64_t c0 = r.head + (int)threadIdx.x * kN;
  // whole batches without a check for each piece, where registers allow the second copy of the body (4 x 128000 fp32, 8 best: 10.7 and 9.5 us; with 128 threads, 6001 x 10001
  // fp32, 40.2 and 42.2)
  if (kThreads != 128)
    for (; c0 + (kBatch - 1) * kThreads * kN < r.v8; c0 += kBatch * kThreads * kN) batch(c0, std::true_type());
  for (; c0 < r.v8; c0 += kBatch * kThreads * kN) batch(c0, std::false_type());
  if ((int)threadIdx.x < rest) {
    if (xr > st.m) st.to(xr);
    add<kEntropy>(xr, st.m == -INFINITY ? 0.f : st.m, st.s, st.w);
  }
  uint32_t key = 0;
  if constexpr (kTop) {
    key = key_of<kThreads, kBf16>(r, st.m, st.s != st.s);
    if (a.top <= kFewTop<kThreads, kBatch>) {
      uint32_t g = key;  // of this thread's group: a warp, or 8 lanes of it
      if (kThreads == 1024) {
        g = __reduce_max_sync(0xffffffffu, g);
        if (lane == 0) best.group[warp] = g;
      } else {
        constexpr int kOf = kThreads / 32;  // threads of a group
#pragma unroll
        for (int o = 1; o < kOf; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (lane % kOf == 0) best.group[threadIdx.x / kOf] = g;
      }
    } else {
      best.key[threadIdx.x] = key;
    }
  }
  {
    const float m = warp_max(st.m);
    if (m > st.m) st.to(m);
    st.m = m;
    st.s = warp_sum(st.s);
    if (kEntropy) st.w = warp_sum(st.w);
  }
  if (lane == 0) {
    sh_m[warp] = st.m;
    sh_s[warp] = st.s;
    sh_w[warp] = st.w;
  }
  __syncthreads();
  if constexpr (kTop) {
    if (warp == 0) {
    const uint32_t bound = a.top <= kFewTop<kThreads, kBatch> ? kth_of_warp(best.group[lane], a.top) : bound_of_threads<kThreads, kBf16>(best, a.top);
    if (lane == 0) {
      best.bound = bound;
      best.count = best.hits = 0;
    }
    }
  }
  if (warp == kLast / 32) {  // the warps' sums; one lane after another's would be a microsecond for 32
    st = lane < kWarps ? Stat{sh_m[lane], sh_s[lane], sh_w[lane]} : Stat{-INFINITY, 0.f, 0.f};
    const float m = warp_max(st.m);
    if (m > st.m) st.to(m);
    st.m = m;
    st.s = warp_sum(st.s);
    if (kEntropy) st.w = warp_sum(st.w);
  }
  if (threadIdx.x == kLast) {
    const bool none = st.s == 0.f;  // no label has a probability
    const float log_s = (float)log((double)st.s);
    const float2 norm = none ? make_float2(0.f, -INFINITY) : make_float2(st.m, log_s);
    sh_norm = norm;
    if (a.norm) *reinterpret_cast<float2*>(a.norm + 2 * row) = norm;
    if (kEntropy) a.entropy[row] = none ? 0.f : log_s - st.w / st.s;
    if (a.target) a.lp[row] = y >= 0 && y < a.v ? log_prob(xy, norm) : 0.f;
  }
  if constexpr (kTop) {
    __syncthreads();
    if (sh_norm.y == -INFINITY) {  // a row of nothing but -inf
      if ((int)threadIdx.x < a.top) {
        a.top_label[row * a.top + threadIdx.x] = threadIdx.x;
        a.top_lp[row * a.top + threadIdx.x] = -INFINITY;
      }
      return;
    }
    const int n = select<kThreads, kBf16>(best, r, a.top, key);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t c = best.cand[i];
      int above = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) above += best.cand[j] > c;
      if (above < a.top) {
        a.top_label[row * a.top + above] = label_of(c);
        a.top_lp[row * a.top + above] = log_prob(value_of(c), sh_norm);
      }
    }
  }
}

struct BackArgs {
  const void* x;
  int64_t pitch;
  const void* target;
  const float *norm, *entropy, *d_lp, *d_entropy, *d_top;
  int64_t d_lp_step, d_entropy_step, d_top_row, d_top_step;
  const int* top_label;
  void* dx;
  int target64, v, top;
  int part;  // labels of a CTA's share of a row, a multiple of 8
};

// kTop: the best labels have gradients too. kLastFirst: rows from the last one on. Block (row, share of its labels); share 0 has those outside the chunks too.
template <bool kBf16, bool kEntropy, bool kTop, bool kLastFirst>
__global__ void __launch_bounds__(kBack)
backward_kernel(const BackArgs a) {
  __shared__ int label[kMaxTop + 1];
  __shared__ float grad[kMaxTop + 1];
  const int64_t row = kLastFirst ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  rb_pdl_wait();
  rb_pdl_launch();
  const int64_t base = row * a.pitch, out = row * (int64_t)a.v;
  const float2 norm = *reinterpret_cast<const float2*>(a.norm + 2 * row);
  const bool none = norm.y == -INFINITY;
  long long y = -1;
  float all = 0.f;  // sum of the gradients of log probabilities
  if (a.target && a.d_lp) {
    y = a.target64 ? reinterpret_cast<const long long*>(a.target)[row] : reinterpret_cast<const int*>(a.target)[row];
    if (none || y < 0 || y >= a.v) y = -1;
    else all = a.d_lp[row * a.d_lp_step];
  }
  const float own = all;
  if (kTop) {
    if ((int)threadIdx.x <= a.top) {
      const int k = threadIdx.x - 1;
      label[threadIdx.x] = k < 0 ? (int)y : none ? -1 : a.top_label[row * a.top + k];
      grad[threadIdx.x] = k < 0 ? own : none ? 0.f : a.d_top[row * a.d_top_row + k * a.d_top_step];
    }
    __syncthreads();
    for (int i = 1; i <= a.top; ++i) all += grad[i];
  }
  const float ge = kEntropy && !none ? a.d_entropy[row * a.d_entropy_step] : 0.f;
  const float h = kEntropy ? a.entropy[row] : 0.f;
  auto of = [&](float x) {
    const float lp = (x - norm.x) - norm.y;
    const float p = none ? 0.f : exp2f(lp * kLog2e);
    return -p * (kEntropy ? all + ge * (fmaxf(lp, -1e4f) + h) : all);
  };
  const int head_in = row_head(a.x, base, a.v, kBf16 ? 2 : 4), head_out = row_head(a.dx, out, a.v, kBf16 ? 2 : 4);
  const int head = head_in == head_out ? head_in : a.v;  // (rows that are aligned differently: single elements)
  const int v8 = head + ((a.v - head) & ~7);
  const int lo = (int)min((int64_t)v8, head + (int64_t)blockIdx.y * a.part), hi = (int)min((int64_t)v8, (int64_t)lo + a.part);
  const bool outside = blockIdx.y == 0;
  auto mine = [&](int c) { return c >= head && c < v8 ? c >= lo && c < hi : outside; };
  auto put = [&](int64_t c, float d) {
    if (kBf16) reinterpret_cast<__nv_bfloat16*>(a.dx)[out + c] = __float2bfloat16(d);
    else reinterpret_cast<float*>(a.dx)[out + c] = d;
  };
  if (!none && !is_far(norm.x)) {
    const float least = floor_of(norm.x);
    const uint64_t minus_m = two(-norm.x, -norm.x), minus_s = two(-norm.y, -norm.y), l2 = two(kLog2e, kLog2e), slope = two(-ge, -ge);
    const float at0 = -(all + ge * h);
    const uint64_t offset = two(at0, at0);
#pragma unroll 4
    for (int64_t c = lo + (int)threadIdx.x * 8; c < hi; c += kBack * 8) {
      constexpr int kN = Chunk<kBf16>::kN;
      Chunk<kBf16> u[8 / kN];
#pragma unroll
      for (int i = 0; i < 8 / kN; ++i) u[i].load(a.x, base + c + i * kN);
      F8 d;
#pragma unroll
      for (int i = 0; i < 8 / kN; ++i) {
        uint64_t p[kN / 2];
        in_pairs<kEntropy>(u[i], least, p);
#pragma unroll
        for (int k = 0; k < kN / 2; ++k) {
          const uint64_t lp = add2(add2(p[k], minus_m), minus_s);
          float t0, t1;
          split(mul2(lp, l2), t0, t1);
          const uint64_t e = two(exp2f(t0), exp2f(t1));
          split(mul2(e, kEntropy ? fma2(lp, slope, offset) : offset), d.v[i * kN + 2 * k], d.v[i * kN + 2 * k + 1]);
        }
      }
      store8(a.dx, out + c, d, kBf16);
    }
  } else {
    for (int64_t c = lo + (int)threadIdx.x * 8; c < hi; c += kBack * 8)
      for (int k = 0; k < 8; ++k) put(c + k, of(ld(a.x, base + c + k, kBf16)));
  }
  for (int i = threadIdx.x; outside && i < a.v - (v8 - head); i += kBack) {
    const int c = i < head ? i : i + (v8 - head);
    put(c, of(ld(a.x, base + c, kBf16)));
  }
  if (!kTop) {
    // the target's entry again, by the thread that wrote it
    if (y >= 0 && mine((int)y)) {
      const int c = (int)y;
      const int who = c >= head && c < v8 ? (c - lo) / 8 % kBack : (c < head ? c : c - (v8 - head)) % kBack;
      if ((int)threadIdx.x == who) put(c, own + of(ld(a.x, base + c, kBf16)));
    }
  } else {
    __syncthreads();
    if ((int)threadIdx.x <= a.top && label[threadIdx.x] >= 0 && mine(label[threadIdx.x])) {
      const int c = label[threadIdx.x];
      float sum = 0.f;
      bool first = true;
      for (int i = 0; i <= a.top; ++i) {
        if (label[i] != c) continue;
        if (i < (int)threadIdx.x) first = false;
        sum += grad[i];
      }
      if (first) put(c, sum + of(ld(a.x, base + c, kBf16)));
    }
  }
}

}  // namespace

// x: rows of v logits, pitch apart. target [rows] (int32 or int64) or null; lp, entropy [rows]; norm [rows][2]; top_lp, top_label [rows][top]. entropy, norm null: not wanted
RB_EXPORT int rb200_token_log_probs_fwd(const void* x, long long pitch, const void* target, int target64, long long rows, int v, int top, int bf16, float* lp,
                                        float* norm, float* entropy, float* top_lp, int* top_label, cudaStream_t stream) {
  if (rows <= 0) return RB_OK;
  if (v < 1 || top < 0 || top > kMaxTop || top > v || rows > 0x7fffffffLL) {
    rb_set_error("token_log_probs: %lld rows of %d labels, %d best (at most %d and the labels)", rows, v, top, kMaxTop);
    return RB_ERR_UNSUPPORTED;
  }
  Args a = {};
  a.x = x; a.pitch = pitch; a.target = target; a.target64 = target64; a.v = v; a.top = top; a.lp = lp; a.norm = norm; a.entropy = entropy; a.top_lp = top_lp;
  a.top_label = top_label;
  // Threads of a row and 16-byte pieces that each has under way: 128 with four pieces (12 rows on an SM), 256 with four (six) or eight (four), 1024. Measured, us:
  // many rows, below 48 KB each: 128, where the latencies of one row's end are hidden best (1500 x 10001 fp32, 8 best: 15.9, with 256 18.3; 2740 x 1001, 20 best 12.5 and 23.5);
  // many longer rows: 256 (6001 x 32000 fp32, 32 best: with 128 222, 164), with eight pieces unless the ends of the rows are the longer (2000 x 128000 bf16, 8 best: with 128 132,
  // four pieces 106, eight 97; 6001 x 32000 bf16, 8 best: 89, 82, 86);
  // rows that are all on the SMs at once: as many pieces as that leaves room for (800 x 50001 fp32, 8 best: four 31, eight 36; 500 x 32000 bf16: 12.9 and 9.2);
  // two rows on an SM or fewer: 1024 for many labels (16 x 32000, 5 best: 6.8 with 256, 5.4; 4 x 128000 fp32, 8 best: 21.2 and 9.5; but 183 x 10001, 32 best, with
  // gradient 11.7 and 19.6).
  const long long bytes = (long long)v * (bf16 ? 2 : 4);
  const int way = rows <= 2 * 148   ? (v < 8192 ? 1 : v < 16384 ? 2 : 3)
                  : rows <= 4 * 148 ? (v < 8192 ? 1 : 2)
                  : rows <= 6 * 148 ? 1
                  : bytes >= (48 << 10) ? (top && bytes < (128 << 10) ? 1 : 2)
                                        : (rows >= 8 * 148 ? 0 : 1);
  auto pick = [&](auto threads, auto batch, auto b) {
    constexpr int kT = decltype(threads)::value, kP = decltype(batch)::value;
    constexpr bool kB = decltype(b)::value;
    return entropy ? (top ? forward_kernel<kT, kB, true, true, kP> : forward_kernel<kT, kB, true, false, kP>)
                   : (top ? forward_kernel<kT, kB, false, true, kP> : forward_kernel<kT, kB, false, false, kP>);
  };
  auto of_type = [&](auto b) {
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 8> eight;
    if (way == 0) return pick(std::integral_constant<int, 128>(), four, b);
    if (way == 1) return pick(std::integral_constant<int, 256>(), four, b);
    if (way == 2) return pick(std::integral_constant<int, 256>(), eight, b);
    return pick(std::integral_constant<int, 1024>(), four, b);
  };
  auto kernel = bf16 ? of_type(std::true_type()) : of_type(std::false_type());
  rb_launch_pdl(kernel, dim3((unsigned)rows), dim3(way == 0 ? 128 : way == 3 ? 1024 : 256), 0, stream, a);
  return rb_check_launch("token_log_probs_fwd");
}

// incoming gradients (null: none) with their strides: of the log probabilities, the entropy, the best; dx [rows][v] in the type of x
RB_EXPORT int rb200_token_log_probs_bwd(const void* x, long long pitch, const void* target, int target64, const float* norm, const float* entropy,
                                        const int* top_label, const float* d_lp, long long d_lp_step, const float* d_entropy, long long d_entropy_step,
                                        const float* d_top, long long d_top_row, long long d_top_step, void* dx, long long rows, int v, int top, int bf16,
                                        cudaStream_t stream) {
  if (rows <= 0) return RB_OK;
  if (v < 1 || top < 0 || top > kMaxTop || rows > 0x7fffffffLL) return RB_ERR_ARG;
  BackArgs a = {};
  a.x = x; a.pitch = pitch; a.target = target; a.target64 = target64; a.norm = norm; a.entropy = entropy; a.top_label = top_label; a.d_lp = d_lp;
  a.d_lp_step = d_lp_step; a.d_entropy = d_entropy; a.d_entropy_step = d_entropy_step; a.d_top = d_top; a.d_top_row = d_top_row; a.d_top_step = d_top_step;
  a.dx = dx; a.v = v; a.top = d_top ? top : 0;
  // the last rows first where logits and gradient do not fit the L2 together: what the forward pass read last is what it still holds
  const bool last_first = rows > 8 * 148 && rows * v * (bf16 ? 2 : 4) >= (64LL << 20);
  auto pick = [&](auto b) {
    constexpr bool kB = decltype(b)::value;
    return d_entropy ? (a.top ? (last_first ? backward_kernel<kB, true, true, true> : backward_kernel<kB, true, true, false>)
                              : (last_first ? backward_kernel<kB, true, false, true> : backward_kernel<kB, true, false, false>))
                     : (a.top ? (last_first ? backward_kernel<kB, false, true, true> : backward_kernel<kB, false, true, false>)
                              : (last_first ? backward_kernel<kB, false, false, true> : backward_kernel<kB, false, false, false>));
  };
  auto kernel = bf16 ? pick(std::true_type()) : pick(std::false_type());
  // few rows: shares of a row, as long as a thread has two chunks of 8 (25 x 128000 bf16, both passes: 28.1 us with whole rows, 13.9)
  const long long shares = std::max(1LL, std::min(4 * 148 / rows, (long long)v / (kBack * 16)));
  a.part = (int)(((v + shares - 1) / shares + 7) / 8 * 8);
  rb_launch_pdl(kernel, dim3((unsigned)rows, (unsigned)shares), dim3(kBack), 0, stream, a);
  return rb_check_launch("token_log_probs_bwd");
}
