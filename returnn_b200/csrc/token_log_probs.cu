// Log probabilities of given tokens over rows of logits, with the entropy of each row and its K best labels, and the gradient of all three.
//   with the maximum m: S = sum exp(x - m), lp = (x_y - m) - log S, H = log S - sum exp(x - m) (x - m) / S  (differences to the maximum: no cancellation)
//   best: the K largest logits, the lowest label first among equal ones (NaN counts as the largest), as log probabilities
//   dx_j = g (d_jy - p_j) + sum_k g_k (d_j,best_k - p_j) - g_H p_j (log p_j + H)
// A target outside 0 .. V - 1 has log probability 0 and no gradient of it. A label of logit -inf has probability 0; a row of nothing else has entropy 0,
// log probabilities -inf and no gradient.
//
// Forward: one CTA per row, one pass with a running maximum, sum and sum of exp(z) z; the logits are read once. The K best come without a sort and almost without
// a second read: the K-th largest of the threads' maxima bounds the K-th largest logit from below, so that only the threads whose maximum reaches the bound
// look their logits through again (K of 256, each warp one thread's logits at a time), and the few logits above it are ranked by counting.
// Backward: one pass, p from the maximum and the sum; the labels that have a gradient of their own are written once more at the end.
#include "class_rows.cuh"

namespace {

using rows::Chunk;
using rows::ld;
using rows::row_head;

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;
constexpr int kCand = 512;  // logits that are ranked
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
// The difference first: the exponent of the maximum is 0 whatever its size, up to the type's lowest value. (One fused multiply-add, x / ln 2 - m / ln 2, would round
// the second product by 2^-24 of the maximum and overflow at the end of the range.) A logit of -inf has e = 0, which must not meet an infinity.
__device__ __forceinline__ void add(float x, float m, float& s, float& w, bool entropy) {
  const float z = x - m;
  const float e = exp2f(z * kLog2e);
  s += e;
  if (entropy) w += e * fmaxf(z, -1e4f);
}

__device__ __forceinline__ void merge(Stat& a, Stat b) {
  const float nm = fmaxf(a.m, b.m);
  if (nm > a.m) a.to(nm);
  if (nm > b.m) b.to(nm);
  a.s += b.s;
  a.w += b.w;
}

// K-th largest of the CTA's 256 whole numbers in shared memory, by one warp, bit by bit (`bits` leading ones may differ)
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* key, int k, int bits) {
  const int lane = threadIdx.x & 31;
  uint32_t mine[kThreads / 32];
#pragma unroll
  for (int j = 0; j < kThreads / 32; ++j) mine[j] = key[j * 32 + lane];
  uint32_t found = 0;
  for (int b = 31; b >= 32 - bits; --b) {
    const uint32_t want = found | 1u << b;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kThreads / 32; ++j) n += mine[j] >= want;
    if ((int)__reduce_add_sync(0xffffffffu, n) >= k) found = want;
  }
  return found;
}

struct Row {
  const void* x;
  int64_t base;
  int head, v8, v;
};

struct Best {
  uint32_t key[kThreads];
  uint64_t cand[kCand];  // rank of the logit, and the label counted from above
  uint64_t last;
  uint32_t bound, limit;
  int count, above, equal;
};

__device__ __forceinline__ uint64_t composite(float x, int label) { return (uint64_t)rank_of(x) << 32 | (0xffffffffu - (uint32_t)label); }

template <bool kBf16>
__device__ __forceinline__ void consider(Best& b, float x, int label) {
  const uint32_t r = rank_of(x);
  if (r > b.bound || (r == b.bound && (uint32_t)label <= b.limit)) {
    const int at = atomicAdd(&b.count, 1);  // (the order does not matter: they are ranked)
    if (at < kCand) b.cand[at] = (uint64_t)r << 32 | (0xffffffffu - (uint32_t)label);
  }
}

// logits of the threads whose maximum reaches the bound, and those outside the chunks
template <bool kBf16>
__device__ __forceinline__ void collect(Best& b, const Row& r, uint32_t key) {
  constexpr int kN = Chunk<kBf16>::kN;
  const int lane = threadIdx.x & 31;
  uint32_t who = __ballot_sync(0xffffffffu, key >= b.bound);
  while (who) {
    const int t = (threadIdx.x & ~31) + __ffs(who) - 1;
    who &= who - 1;
    for (int c = r.head + (t + kThreads * lane) * kN; c < r.v8; c += 32 * kThreads * kN) {
      Chunk<kBf16> u;
      u.load(r.x, r.base + c);
#pragma unroll
      for (int k = 0; k < kN; ++k) consider<kBf16>(b, u.at(k), c + k);
    }
  }
  const int rest = r.v - (r.v8 - r.head);
  if ((int)threadIdx.x < rest) {
    const int c = (int)threadIdx.x < r.head ? threadIdx.x : threadIdx.x + (r.v8 - r.head);
    consider<kBf16>(b, ld(r.x, r.base + c, kBf16), c);
  }
}

// the first label of this thread's own logits (the chunks, and one outside) that has rank `want`
template <bool kBf16>
__device__ __forceinline__ uint32_t first_of(const Row& r, uint32_t want) {
  constexpr int kN = Chunk<kBf16>::kN;
  uint32_t at = 0xffffffffu;
  const int rest = r.v - (r.v8 - r.head);
  if ((int)threadIdx.x < rest) {
    const int c = (int)threadIdx.x < r.head ? threadIdx.x : threadIdx.x + (r.v8 - r.head);
    if (rank_of(ld(r.x, r.base + c, kBf16)) == want) at = c;
  }
  for (int c = r.head + (int)threadIdx.x * kN; c < r.v8 && (uint32_t)c < at; c += kThreads * kN) {
    Chunk<kBf16> u;
    u.load(r.x, r.base + c);
#pragma unroll
    for (int k = kN - 1; k >= 0; --k)
      if (rank_of(u.at(k)) == want) at = min(at, (uint32_t)(c + k));
  }
  return at;
}

// The K best labels of a row in b.cand, in no order; returns how many there are (at least K; all above the K-th, which is among them).
// `mx`: the maximum of this thread's chunks and of one logit outside them; `odd`: its sum is no number, the maximum may be one.
template <bool kBf16>
__device__ int select(Best& b, const Row& r, int top, float mx, bool odd) {
  uint32_t key = rank_of(mx);
  if (odd) {
    constexpr int kN = Chunk<kBf16>::kN;
    const int rest = r.v - (r.v8 - r.head);
    if ((int)threadIdx.x < rest) key = max(key, rank_of(ld(r.x, r.base + ((int)threadIdx.x < r.head ? threadIdx.x : threadIdx.x + (r.v8 - r.head)), kBf16)));
    for (int c = r.head + (int)threadIdx.x * kN; c < r.v8; c += kThreads * kN)
      for (int k = 0; k < kN; ++k) key = max(key, rank_of(ld(r.x, r.base + c + k, kBf16)));
  }
  b.key[threadIdx.x] = key;
  if (threadIdx.x == 0) b.count = b.above = b.equal = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    // (the lower half of a bf16 value's rank follows from the upper: zeros, ones where the value is negative or no number)
    uint32_t bound = kth_largest(b.key, top, kBf16 ? 16 : 32);
    if (kBf16 && (bound < 0x80000000u || bound == 0xffff0000u)) bound |= 0xffffu;
    if (threadIdx.x == 0) {
      b.bound = bound;
      b.limit = 0xffffffffu;
    }
  }
  __syncthreads();
  const unsigned above = __ballot_sync(0xffffffffu, key > b.bound), equal = __ballot_sync(0xffffffffu, key == b.bound);
  if ((threadIdx.x & 31) == 0) {
    if (above) atomicAdd(&b.above, __popc(above));
    if (equal) atomicAdd(&b.equal, __popc(equal));
  }
  __syncthreads();
  bool many = b.above + b.equal > 64;
  if (!many) {
    collect<kBf16>(b, r, key);
    __syncthreads();
    many = b.count > kCand;
  }
  if (many) {
    // many equal logits at the bound: of those, only the ones up to the label that the K best need. A thread's first one bounds it.
    __syncthreads();
    const uint32_t bound = b.bound, need = top - b.above;
    const uint32_t first = key == bound ? first_of<kBf16>(r, bound) : 0xffffffffu;
    b.key[threadIdx.x] = ~first;
    __syncthreads();
    if (threadIdx.x < 32) {
      const uint32_t limit = ~kth_largest(b.key, (int)need, 32);
      if (threadIdx.x == 0) {
        b.limit = limit;
        b.count = 0;
      }
    }
    __syncthreads();
    collect<kBf16>(b, r, key);
    __syncthreads();
    if (b.count > kCand) {
      // more logits above the bound than are ranked (all in few threads' share): the K best one after another
      __syncthreads();
      uint64_t before = ~0ull;
      for (int k = 0; k < top; ++k) {
        uint64_t best = 0;
        for (int c = threadIdx.x; c < r.v; c += kThreads) {
          const uint64_t q = composite(ld(r.x, r.base + c, kBf16), c);
          if (q < before && q > best) best = q;
        }
        if (threadIdx.x == 0) b.last = 0;
        __syncthreads();
        atomicMax(reinterpret_cast<unsigned long long*>(&b.last), (unsigned long long)best);
        __syncthreads();
        before = b.last;
        __syncthreads();
        if (threadIdx.x == 0) b.cand[k] = before;
      }
      if (threadIdx.x == 0) b.count = top;
      __syncthreads();
    }
  }
  return b.count;
}

__device__ __forceinline__ float value_of(uint64_t c) {
  const uint32_t r = (uint32_t)(c >> 32);
  return __uint_as_float(r & 0x80000000u ? r & 0x7fffffffu : ~r);  // (NaN: the largest rank is a NaN again)
}

__device__ __forceinline__ float log_prob(float x, float2 norm) {
  return x == -INFINITY && norm.y == norm.y ? -INFINITY : (x - norm.x) - norm.y;
}

// kBatch: chunks of 16 bytes that a thread has in flight
template <bool kBf16, bool kEntropy, bool kTop, int kBatch>
__global__ void __launch_bounds__(kThreads)
forward_kernel(const Args a) {
  constexpr int kN = Chunk<kBf16>::kN;
  __shared__ float sh_m[8], sh_s[8], sh_w[8];
  __shared__ float2 sh_norm;
  __shared__ Best best;
  const int64_t row = blockIdx.x;
  rb_pdl_wait();
  rb_pdl_launch();
  Row r;
  r.x = a.x;
  r.base = row * a.pitch;
  r.v = a.v;
  r.head = row_head(a.x, r.base, a.v, kBf16 ? 2 : 4);
  r.v8 = r.head + ((a.v - r.head) & ~7);
  Stat st{-INFINITY, 0.f, 0.f};
  for (int c0 = r.head + threadIdx.x * kN; c0 < r.v8; c0 += kBatch * kThreads * kN) {
    Chunk<kBf16> u[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int c = c0 + q * kThreads * kN;
      if (c < r.v8) u[q].load(a.x, r.base + c);
      else u[q].fill_neg_inf();
    }
    float lm = u[0].max();
#pragma unroll
    for (int q = 1; q < kBatch; ++q) lm = fmaxf(lm, u[q].max());
    if (lm > st.m) st.to(lm);
    const float m = st.m == -INFINITY ? 0.f : st.m;
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (q == 0 || c0 + q * kThreads * kN < r.v8)
#pragma unroll
        for (int k = 0; k < kN; ++k) add(u[q].at(k), m, s, w, kEntropy);
    st.s += s;
    st.w += w;
  }
  const int rest = a.v - (r.v8 - r.head);  // fewer than the threads
  if ((int)threadIdx.x < rest) {
    const int c = (int)threadIdx.x < r.head ? threadIdx.x : threadIdx.x + (r.v8 - r.head);
    const float x = ld(a.x, r.base + c, kBf16);
    if (x > st.m) st.to(x);
    add(x, st.m == -INFINITY ? 0.f : st.m, st.s, st.w, kEntropy);
  }
  const float mine = st.m;
  const bool odd = st.s != st.s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    merge(st, Stat{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.w, o)});
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    sh_m[warp] = st.m;
    sh_s[warp] = st.s;
    sh_w[warp] = st.w;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    st = Stat{sh_m[0], sh_s[0], sh_w[0]};
#pragma unroll
    for (int w = 1; w < 8; ++w) merge(st, Stat{sh_m[w], sh_s[w], sh_w[w]});
    const bool none = st.s == 0.f;  // no label has a probability
    const float log_s = (float)log((double)st.s);
    sh_norm = none ? make_float2(0.f, -INFINITY) : make_float2(st.m, log_s);
    if (a.norm) *reinterpret_cast<float2*>(a.norm + 2 * row) = sh_norm;
    if (kEntropy) a.entropy[row] = none ? 0.f : log_s - st.w / st.s;
    if (a.target) {
      const long long y = target_of(a, row);
      a.lp[row] = y >= 0 && y < a.v ? log_prob(ld(a.x, r.base + y, kBf16), sh_norm) : 0.f;
    }
  }
  if (kTop) {
    const int n = select<kBf16>(best, r, a.top, mine, odd);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t c = best.cand[i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += best.cand[j] > c;
      if (above < a.top) {
        a.top_label[row * a.top + above] = (int)(0xffffffffu - (uint32_t)c);
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
};

template <bool kBf16, bool kEntropy>
__global__ void __launch_bounds__(kThreads)
backward_kernel(const BackArgs a) {
  __shared__ int label[kMaxTop + 1];
  __shared__ float grad[kMaxTop + 1];
  const int64_t row = blockIdx.x;
  rb_pdl_wait();
  rb_pdl_launch();
  const int64_t base = row * a.pitch, out = row * (int64_t)a.v;
  const float2 norm = *reinterpret_cast<const float2*>(a.norm + 2 * row);
  const bool none = norm.y == -INFINITY;
  const int n = a.top + 1;
  if ((int)threadIdx.x < n) {
    const int k = threadIdx.x - 1;
    long long y = -1;
    float g = 0.f;
    if (k < 0) {
      if (a.target && a.d_lp) {
        y = a.target64 ? reinterpret_cast<const long long*>(a.target)[row] : reinterpret_cast<const int*>(a.target)[row];
        g = a.d_lp[row * a.d_lp_step];
      }
    } else if (a.d_top) {
      y = a.top_label[row * a.top + k];
      g = a.d_top[row * a.d_top_row + k * a.d_top_step];
    }
    const bool real = !none && y >= 0 && y < a.v;
    label[threadIdx.x] = real ? (int)y : -1;
    grad[threadIdx.x] = real ? g : 0.f;
  }
  __syncthreads();
  float all = 0.f;
  for (int i = 0; i < n; ++i) all += grad[i];
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
#pragma unroll 4
  for (int c = head + threadIdx.x * 8; c < v8; c += kThreads * 8) {
    F8 x = load8(a.x, base + c, kBf16);
#pragma unroll
    for (int k = 0; k < 8; ++k) x.v[k] = of(x.v[k]);
    store8(a.dx, out + c, x, kBf16);
  }
  auto put = [&](int c, float d) {
    if (kBf16) reinterpret_cast<__nv_bfloat16*>(a.dx)[out + c] = __float2bfloat16(d);
    else reinterpret_cast<float*>(a.dx)[out + c] = d;
  };
  for (int i = threadIdx.x; i < a.v - (v8 - head); i += kThreads) {
    const int c = i < head ? i : i + (v8 - head);
    put(c, of(ld(a.x, base + c, kBf16)));
  }
  __syncthreads();
  if ((int)threadIdx.x < n && label[threadIdx.x] >= 0) {
    const int c = label[threadIdx.x];
    float own = 0.f;
    bool first = true;
    for (int i = 0; i < n; ++i) {
      if (label[i] != c) continue;
      if (i < (int)threadIdx.x) first = false;
      own += grad[i];
    }
    if (first) put(c, own + of(ld(a.x, base + c, kBf16)));
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
  auto kernel = bf16 ? (entropy ? (top ? forward_kernel<true, true, true, 4> : forward_kernel<true, true, false, 4>)
                                : (top ? forward_kernel<true, false, true, 4> : forward_kernel<true, false, false, 4>))
                     : (entropy ? (top ? forward_kernel<false, true, true, 4> : forward_kernel<false, true, false, 4>)
                                : (top ? forward_kernel<false, false, true, 4> : forward_kernel<false, false, false, 4>));
  rb_launch_pdl(kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
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
  auto kernel = bf16 ? (d_entropy ? backward_kernel<true, true> : backward_kernel<true, false>)
                     : (d_entropy ? backward_kernel<false, true> : backward_kernel<false, false>);
  rb_launch_pdl(kernel, dim3((unsigned)rows), dim3(kThreads), 0, stream, a);
  return rb_check_launch("token_log_probs_bwd");
}
