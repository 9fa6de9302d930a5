// Block tables and slots of a paged key / value cache, kept on the GPU so that a decoding step needs no word from the host.
// A cache is pages of P tokens. Request i has len_i tokens in the pages table[i][0 .. ceil(len_i / P)). The pages that no request has lie in a ring:
// places head .. tail - 1 (modulo its size F) of `ring`.
//   append: request i gets new_i more tokens and needs ceil((len_i + new_i) / P) - ceil(len_i / P) pages. Requests are served in their order while the sum of
//           what they need is within tail - head; one that comes too late, or whose table row is too short, is left as it is. Token t of the call
//           (requests one after another) gets its request, its position and its slot = page * P + position % P.
//   release: the pages of the requests that are done go to the ring's tail, in the order of requests and blocks.
// Neither changes the lengths or the range that it is given: both are returned anew, so that a call can be repeated.
//
// All is a prefix sum over the requests and then independent entries, each found by a binary search in the sums. A kernel of its own for the sums
// would cost a launch, more than the sums: every CTA goes over all requests, 256 or 1024 at a time, and writes the entries that fall to it.
#include "common.cuh"
#include <algorithm>

namespace {

constexpr int kThreads = 256;

// Sums end at 2^32 - 1: more tokens than a list can have, more pages than there are
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < a ? 0xffffffffu : s;
}
struct Sums {
  uint32_t a, b;
};

// exclusive prefix sums over the threads of the CTA, and the totals
__device__ __forceinline__ Sums scan(Sums v, Sums* total) {
  __shared__ Sums warp_total[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, inc.a, o), b = __shfl_up_sync(0xffffffffu, inc.b, o);
    if (lane >= o) inc = {plus(inc.a, a), plus(inc.b, b)};
  }
  Sums before = {__shfl_up_sync(0xffffffffu, inc.a, 1), __shfl_up_sync(0xffffffffu, inc.b, 1)};
  if (lane == 0) before = {0, 0};
  if (lane == 31) warp_total[warp] = inc;
  __syncthreads();
  Sums base = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) base = all;
    all = {plus(all.a, warp_total[w].a), plus(all.b, warp_total[w].b)};
  }
  *total = all;
  return {plus(base.a, before.a), plus(base.b, before.b)};
}

// last i in [0, n) with first[i] <= x (first[0] <= x)
__device__ __forceinline__ int owner(const uint32_t* first, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Page size, with its logarithm where it is a power of two. Counts of tokens are below 2^32: 64-bit divisions, one per token and three per request, were most of the time.
struct Page {
  uint32_t size;
  int shift;
  __device__ __forceinline__ uint32_t of(uint32_t token) const { return shift >= 0 ? token >> shift : token / size; }
  __device__ __forceinline__ uint32_t count(uint32_t tokens) const {
    const uint32_t whole = of(tokens);
    return whole + (whole * size != tokens);
  }
};
__device__ __forceinline__ long long remainder_of(long long x, long long size) {  // x mod size, not negative
  if (((unsigned long long)x | (unsigned long long)size) >> 32 == 0) return (uint32_t)x % (uint32_t)size;
  const long long r = x % size;
  return r < 0 ? r + size : r;
}

struct Ring {
  int* pages;
  long long size;
  __device__ __forceinline__ int* at(long long place) const {  // place: from 0 to below 2 * size
    return pages + (place >= size ? place - size : place);
  }
};

// kEach: requests of a thread in a round; kTok: tokens of a thread, in a row (four have most often one request and one page, and one search)
template <int kEach, int kTok>
__global__ void __launch_bounds__(kThreads)
append_kernel(int* __restrict__ table, long long table_stride, int blocks, const int* __restrict__ lens, const int* __restrict__ add, int n, Ring ring,
              const long long* __restrict__ range, Page page, long long max_tokens, int* __restrict__ slots, int* __restrict__ positions,
              int* __restrict__ requests, int* __restrict__ offsets, int* __restrict__ new_lens, long long* __restrict__ new_range,
              uint8_t* __restrict__ granted) {
  constexpr int kChunk = kThreads * kEach;
  __shared__ uint32_t tok_first[kChunk], page_first[kChunk];  // of the requests of a round, from its own beginning
  __shared__ uint32_t len_of[kChunk];
  __shared__ uint8_t ok_of[kChunk];
  __shared__ uint32_t used_shared;
  rb_pdl_wait();
  rb_pdl_launch();
  const long long head = range[0], tail = range[1];
  const long long free_pages = min(max(tail - head, 0LL), ring.size);
  const long long start = remainder_of(head, ring.size);
  const bool writer = blockIdx.x == 0;
  // this CTA's tokens
  const long long per = ((max_tokens + gridDim.x - 1) / gridDim.x + 3) & ~3LL;  // (whole vectors)
  const bool vector = ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(requests)) & 15) == 0;
  const long long my0 = min(max_tokens, per * blockIdx.x), my1 = min(max_tokens, my0 + per);
  const long long room = (long long)blocks * page.size;
  long long tok_base = 0, page_base = 0, used = 0;
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    const int cn = min(kChunk, n - c0);
    uint32_t nw[kEach], need[kEach], len[kEach];
    int old[kEach];
    bool fit[kEach];
    Sums mine = {0, 0};
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = c0 + threadIdx.x * kEach + j;
      nw[j] = need[j] = len[j] = 0;
      old[j] = 0;
      fit[j] = false;
      if (i < n) {
        old[j] = lens[i];
        len[j] = (uint32_t)max(old[j], 0);
        nw[j] = (uint32_t)max(add[i], 0);
        fit[j] = len[j] + nw[j] <= room;
        if (fit[j]) need[j] = page.count(len[j] + nw[j]) - page.count(len[j]);
      }
      mine = {plus(mine.a, nw[j]), plus(mine.b, need[j])};
    }
    if (threadIdx.x == 0) used_shared = 0;
    Sums total;
    Sums at = scan(mine, &total);
    uint32_t most = 0;
    const long long left = free_pages - page_base;  // (negative: all pages are given)
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int k = threadIdx.x * kEach + j;
      const uint32_t next = plus(at.b, need[j]);
      const bool ok = fit[j] && (need[j] == 0 || next <= left);
      if (ok && need[j]) most = next;
      tok_first[k] = at.a;
      page_first[k] = at.b;
      len_of[k] = len[j];
      ok_of[k] = ok;
      if (writer && c0 + k < n) {
        offsets[c0 + k] = (int)(tok_base + at.a);
        new_lens[c0 + k] = ok ? (int)(len[j] + nw[j]) : old[j];
        granted[c0 + k] = ok;
      }
      at = {plus(at.a, nw[j]), next};
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0 && most) atomicMax(&used_shared, most);  // (a maximum of whole numbers: the same in any order)
    __syncthreads();
    const uint32_t taken = used_shared;
    if (taken) used = page_base + taken;
    // pages of this round: the first `taken` belong to requests that were served
    for (long long p = (long long)blockIdx.x * kThreads + threadIdx.x; p < taken; p += (long long)gridDim.x * kThreads) {
      const int k = owner(page_first, cn, (uint32_t)p);
      table[(long long)(c0 + k) * table_stride + page.count(len_of[k]) + (p - page_first[k])] = *ring.at(start + page_base + p);
    }
    // tokens of this round that are this CTA's
    const long long t_end = min(my1, tok_base + total.a), t_begin = max(my0, tok_base);
    for (long long q = (kTok > 1 ? t_begin & ~3LL : t_begin) + kTok * threadIdx.x; q < t_end; q += kTok * kThreads) {
      const long long t0 = max(q, t_begin), t1 = min(q + kTok, t_end);
      int k = owner(tok_first, cn, (uint32_t)(t0 - tok_base));
      uint32_t end = k + 1 < cn ? tok_first[k + 1] : 0xffffffffu;
      uint32_t block_at = 0xffffffffu;
      int pg = 0;
      int slot[kTok], place[kTok], who[kTok];
#pragma unroll
      for (int u = 0; u < kTok; ++u) {
        const long long t = q + u;
        slot[u] = place[u] = who[u] = 0;
        if (kTok > 1 && (t < t0 || t >= t1)) continue;
        const uint32_t x = (uint32_t)(t - tok_base);
        while (k + 1 < cn && end <= x) {
          ++k;
          end = k + 1 < cn ? tok_first[k + 1] : 0xffffffffu;
          block_at = 0xffffffffu;
        }
        const uint32_t pos = len_of[k] + (x - tok_first[k]), block = page.of(pos);
        if (ok_of[k] && block != block_at) {
          block_at = block;
          const uint32_t have = page.count(len_of[k]);
          pg = block < have ? table[(long long)(c0 + k) * table_stride + block] : *ring.at(start + page_base + page_first[k] + (block - have));
        }
        slot[u] = ok_of[k] ? pg * (int)page.size + (int)(pos - block * page.size) : -1;
        place[u] = (int)pos;
        who[u] = c0 + k;
      }
      if (kTok == 4 && vector && t0 == q && t1 == q + kTok) {
        *reinterpret_cast<int4*>(slots + q) = make_int4(slot[0], slot[kTok - 3], slot[kTok - 2], slot[kTok - 1]);
        *reinterpret_cast<int4*>(positions + q) = make_int4(place[0], place[kTok - 3], place[kTok - 2], place[kTok - 1]);
        *reinterpret_cast<int4*>(requests + q) = make_int4(who[0], who[kTok - 3], who[kTok - 2], who[kTok - 1]);
      } else {
#pragma unroll
        for (int u = 0; u < kTok; ++u) {
          if (kTok > 1 && (q + u < t0 || q + u >= t1)) continue;
          slots[q + u] = slot[u];
          positions[q + u] = place[u];
          requests[q + u] = who[u];
        }
      }
    }
    tok_base += total.a;
    page_base += total.b;
    if (c0 + kChunk < n) __syncthreads();
  }
  for (long long t = max(my0, tok_base) + threadIdx.x; t < my1; t += kThreads) {  // room without tokens
    slots[t] = -1;
    positions[t] = 0;
    requests[t] = -1;
  }
  if (writer && threadIdx.x == 0) {
    offsets[n] = (int)tok_base;
    new_range[0] = head + used;
    new_range[1] = tail;
  }
}

template <int kEach>
__global__ void __launch_bounds__(kThreads)
release_kernel(const int* __restrict__ table, long long table_stride, int blocks, const int* __restrict__ lens, const uint8_t* __restrict__ done, int n,
               Ring ring, const long long* __restrict__ range, Page page, int* __restrict__ new_lens, long long* __restrict__ new_range) {
  constexpr int kChunk = kThreads * kEach;
  __shared__ uint32_t first[kChunk];
  rb_pdl_wait();
  rb_pdl_launch();
  const long long head = range[0], tail = range[1];
  const long long room = max(ring.size - max(tail - head, 0LL), 0LL);  // more than this are not the ring's pages
  const long long start = remainder_of(tail, ring.size);
  long long base = 0;
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    const int cn = min(kChunk, n - c0);
    uint32_t count[kEach];
    Sums mine = {0, 0};
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = c0 + threadIdx.x * kEach + j;
      count[j] = 0;
      if (i < n) {
        const bool over = done[i] != 0;
        const int len = lens[i];
        if (over) count[j] = min(page.count((uint32_t)max(len, 0)), (uint32_t)blocks);
        if (blockIdx.x == 0) new_lens[i] = over ? 0 : len;
      }
      mine.a = plus(mine.a, count[j]);
    }
    Sums total;
    Sums at = scan(mine, &total);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      first[threadIdx.x * kEach + j] = at.a;
      at.a = plus(at.a, count[j]);
    }
    __syncthreads();
    const long long end = min((long long)total.a, room - base);
    for (long long p = (long long)blockIdx.x * kThreads + threadIdx.x; p < end; p += (long long)gridDim.x * kThreads) {
      const int k = owner(first, cn, (uint32_t)p);
      *ring.at(start + base + p) = table[(long long)(c0 + k) * table_stride + (p - first[k])];
    }
    base += total.a;
    if (c0 + kChunk < n) __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    new_range[0] = head;
    new_range[1] = tail + min(base, room);
  }
}

int bad(const char* what, int n, int blocks, long long ring_size, int page) {
  if (n >= 0 && blocks >= 0 && ring_size >= 1 && page >= 1) return 0;
  rb_set_error("%s: %d requests, %d blocks, %lld pages, page size %d", what, n, blocks, ring_size, page);
  return 1;
}

}  // namespace

static Page page_of(int size) {
  Page p{(uint32_t)size, -1};
  if ((size & (size - 1)) == 0) p.shift = __builtin_ctz((unsigned)size);
  return p;
}

// table [n][blocks] with rows table_stride apart, written in place; offsets [n + 1], new_range [2]
RB_EXPORT int rb200_paged_append(int* table, long long table_stride, int blocks, const int* lens, const int* add, int n, int* ring, long long ring_size,
                                 const long long* range, int page, long long max_tokens, int* slots, int* positions, int* requests, int* offsets, int* new_lens,
                                 long long* new_range, void* granted, cudaStream_t stream) {
  if (bad("paged_append", n, blocks, ring_size, page) || max_tokens < 0) return RB_ERR_ARG;
  // A token per thread where that is a wave of CTAs, four beyond; a request per thread where they fit one round. Device us, 64 requests of one token 3.4, with four
  // tokens a thread 5.0, with four requests a thread 4.1; 1M tokens of 256 requests (12 MB of lists, bound by the searches and the trip to the table) 9.0, with a token a
  // thread 14.7, of 500 requests 12.2 and 23.8. Eight CTAs to an
  // SM, or four where each goes over more requests than it has threads (the same 1M tokens with four and eight: 9.7 and 9.0, of 500 requests 12.2 and 16.1)
  const bool four = max_tokens > 148 * kThreads, many = n > kThreads;
  const long long of = (four ? 4 : 1) * kThreads, ctas = std::min<long long>(std::max<long long>((max_tokens + of - 1) / of, 1), 148 * (many ? 4 : 8));
  auto kernel = many ? (four ? append_kernel<4, 4> : append_kernel<4, 1>) : (four ? append_kernel<1, 4> : append_kernel<1, 1>);
  rb_launch_pdl(kernel, dim3((unsigned)ctas), dim3(kThreads), 0, stream, table, table_stride, blocks, lens, add, n, Ring{ring, ring_size}, range, page_of(page),
                max_tokens, slots, positions, requests, offsets, new_lens, new_range, reinterpret_cast<uint8_t*>(granted));
  return rb_check_launch("paged_append");
}

RB_EXPORT int rb200_paged_release(const int* table, long long table_stride, int blocks, const int* lens, const void* done, int n, int* ring, long long ring_size,
                                  const long long* range, int page, int* new_lens, long long* new_range, cudaStream_t stream) {
  if (bad("paged_release", n, blocks, ring_size, page)) return RB_ERR_ARG;
  const long long most = std::min<long long>((long long)n * blocks, ring_size);
  const long long ctas = std::min<long long>(std::max<long long>((most + 2 * kThreads - 1) / (2 * kThreads), 1), 148 * 4);
  rb_launch_pdl(n > kThreads ? release_kernel<4> : release_kernel<1>, dim3((unsigned)ctas), dim3(kThreads), 0, stream, table, table_stride, blocks, lens, reinterpret_cast<const uint8_t*>(done), n,
                Ring{ring, ring_size}, range, page_of(page), new_lens, new_range);
  return rb_check_launch("paged_release");
}
