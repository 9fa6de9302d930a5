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
// would cost a launch, more than the sums: every CTA goes over all requests (a thousand at a time, four per thread) and writes the entries that fall to it.
#include "common.cuh"
#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kEach = 4;                   // requests of a thread
constexpr int kChunk = kThreads * kEach;   // requests of a round

struct Sums {
  long long a, b;
};

// exclusive prefix sums over the threads of the CTA, and the totals
__device__ __forceinline__ Sums scan(Sums v, Sums* total) {
  __shared__ Sums warp_total[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, inc.a, o), b = __shfl_up_sync(0xffffffffu, inc.b, o);
    if (lane >= o) {
      inc.a += a;
      inc.b += b;
    }
  }
  __syncthreads();  // (the totals of the round before have been read)
  if (lane == 31) warp_total[warp] = inc;
  __syncthreads();
  Sums before = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) before = all;
    all.a += warp_total[w].a;
    all.b += warp_total[w].b;
  }
  *total = all;
  return {before.a + inc.a - v.a, before.b + inc.b - v.b};
}

// last i in [0, n) with first[i] <= x (first[0] <= x)
__device__ __forceinline__ int owner(const long long* first, int n, long long x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ long long pages_of(long long tokens, int page) { return (tokens + page - 1) / page; }

struct Ring {
  int* pages;
  long long size, head, tail;
  __device__ __forceinline__ int* at(long long place) const {  // place: from 0 to below 2 * size
    return pages + (place >= size ? place - size : place);
  }
};

__global__ void __launch_bounds__(kThreads)
append_kernel(int* __restrict__ table, long long table_stride, int blocks, const int* __restrict__ lens, const int* __restrict__ add, int n, Ring ring,
              const long long* __restrict__ range, int page, long long max_tokens, int* __restrict__ slots, int* __restrict__ positions,
              int* __restrict__ requests, int* __restrict__ offsets, int* __restrict__ new_lens, long long* __restrict__ new_range,
              uint8_t* __restrict__ granted) {
  __shared__ long long tok_first[kChunk], page_first[kChunk];
  __shared__ long long used_shared;
  rb_pdl_wait();
  rb_pdl_launch();
  const long long head = range[0], tail = range[1];
  const long long free_pages = min(max(tail - head, 0LL), ring.size);
  long long start = head % ring.size;
  if (start < 0) start += ring.size;
  const bool writer = blockIdx.x == 0;
  // this CTA's tokens
  const long long per = (max_tokens + gridDim.x - 1) / gridDim.x;
  const long long my0 = min(max_tokens, per * blockIdx.x), my1 = min(max_tokens, my0 + per);
  long long tok_base = 0, page_base = 0, used = 0;
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    const int cn = min(kChunk, n - c0);
    long long nw[kEach], need[kEach];
    bool fit[kEach];
    Sums mine = {0, 0};
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = c0 + threadIdx.x * kEach + j;
      nw[j] = need[j] = 0;
      fit[j] = false;
      if (i < n) {
        const long long len = max(lens[i], 0);
        nw[j] = max(add[i], 0);
        fit[j] = len + nw[j] <= (long long)blocks * page;
        need[j] = fit[j] ? pages_of(len + nw[j], page) - pages_of(len, page) : 0;
      }
      mine.a += nw[j];
      mine.b += need[j];
    }
    Sums total;
    Sums at = scan(mine, &total);
    at.a += tok_base;
    at.b += page_base;
    if (threadIdx.x == 0) used_shared = 0;
    __syncthreads();
    long long most = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int k = threadIdx.x * kEach + j;
      const bool ok = fit[j] && (need[j] == 0 || at.b + need[j] <= free_pages);
      if (ok && need[j]) most = at.b + need[j];
      tok_first[k] = at.a;
      page_first[k] = at.b;
      if (writer && c0 + k < n) {
        offsets[c0 + k] = (int)at.a;
        new_lens[c0 + k] = ok ? (int)(max(lens[c0 + k], 0) + nw[j]) : lens[c0 + k];
        granted[c0 + k] = ok;
      }
      at.a += nw[j];
      at.b += need[j];
    }
    if (most) atomicMax(&used_shared, most);  // (a maximum of whole numbers: the same in any order)
    __syncthreads();
    used = max(used, used_shared);
    // pages of this round: those up to `used` belong to requests that were served
    const long long page_end = min(page_base + total.b, used);
    for (long long p = page_base + (long long)blockIdx.x * kThreads + threadIdx.x; p < page_end; p += (long long)gridDim.x * kThreads) {
      const int k = owner(page_first, cn, p);
      const long long block = pages_of(max(lens[c0 + k], 0), page) + p - page_first[k];
      table[(long long)(c0 + k) * table_stride + block] = *ring.at(start + p);
    }
    // tokens of this round that are this CTA's
    const long long t1 = min(my1, tok_base + total.a);
    for (long long t = max(my0, tok_base) + threadIdx.x; t < t1; t += kThreads) {
      const int k = owner(tok_first, cn, t), i = c0 + k;
      const long long len = max(lens[i], 0), count = max(add[i], 0);
      const long long pos = len + t - tok_first[k];
      const long long have = pages_of(len, page);
      const bool fits = len + count <= (long long)blocks * page;
      const long long want = fits ? pages_of(len + count, page) - have : 0;
      int slot = -1;
      if (fits && (want == 0 || page_first[k] + want <= free_pages)) {
        const long long block = pos / page;
        const int pg = block < have ? table[(long long)i * table_stride + block] : *ring.at(start + page_first[k] + block - have);
        slot = (int)((long long)pg * page + pos - block * page);
      }
      slots[t] = slot;
      positions[t] = (int)pos;
      requests[t] = i;
    }
    tok_base += total.a;
    page_base += total.b;
    __syncthreads();
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

__global__ void __launch_bounds__(kThreads)
release_kernel(const int* __restrict__ table, long long table_stride, int blocks, const int* __restrict__ lens, const uint8_t* __restrict__ done, int n,
               Ring ring, const long long* __restrict__ range, int page, int* __restrict__ new_lens, long long* __restrict__ new_range) {
  __shared__ long long first[kChunk];
  rb_pdl_wait();
  rb_pdl_launch();
  const long long head = range[0], tail = range[1];
  const long long room = max(ring.size - max(tail - head, 0LL), 0LL);  // more than this are not the ring's pages
  long long start = tail % ring.size;
  if (start < 0) start += ring.size;
  long long base = 0;
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    const int cn = min(kChunk, n - c0);
    long long count[kEach];
    Sums mine = {0, 0};
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = c0 + threadIdx.x * kEach + j;
      count[j] = 0;
      if (i < n) {
        const bool over = done[i] != 0;
        if (over) count[j] = min(pages_of(max(lens[i], 0), page), (long long)blocks);
        if (blockIdx.x == 0) new_lens[i] = over ? 0 : lens[i];
      }
      mine.a += count[j];
    }
    Sums total;
    Sums at = scan(mine, &total);
    at.a += base;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      first[threadIdx.x * kEach + j] = at.a;
      at.a += count[j];
    }
    __syncthreads();
    const long long end = min(base + total.a, room);
    for (long long p = base + (long long)blockIdx.x * kThreads + threadIdx.x; p < end; p += (long long)gridDim.x * kThreads) {
      const int k = owner(first, cn, p);
      *ring.at(start + p) = table[(long long)(c0 + k) * table_stride + p - first[k]];
    }
    base += total.a;
    __syncthreads();
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

// table [n][blocks] with rows table_stride apart, written in place; offsets [n + 1], new_range [2]
RB_EXPORT int rb200_paged_append(int* table, long long table_stride, int blocks, const int* lens, const int* add, int n, int* ring, long long ring_size,
                                 const long long* range, int page, long long max_tokens, int* slots, int* positions, int* requests, int* offsets, int* new_lens,
                                 long long* new_range, void* granted, cudaStream_t stream) {
  if (bad("paged_append", n, blocks, ring_size, page) || max_tokens < 0) return RB_ERR_ARG;
  // a CTA per four tokens a thread: 64 requests of one token are one CTA
  const long long ctas = std::min<long long>(std::max<long long>((max_tokens + 4 * kThreads - 1) / (4 * kThreads), 1), 148 * 2);
  rb_launch_pdl(append_kernel, dim3((unsigned)ctas), dim3(kThreads), 0, stream, table, table_stride, blocks, lens, add, n, Ring{ring, ring_size, 0, 0}, range, page,
                max_tokens, slots, positions, requests, offsets, new_lens, new_range, reinterpret_cast<uint8_t*>(granted));
  return rb_check_launch("paged_append");
}

RB_EXPORT int rb200_paged_release(const int* table, long long table_stride, int blocks, const int* lens, const void* done, int n, int* ring, long long ring_size,
                                  const long long* range, int page, int* new_lens, long long* new_range, cudaStream_t stream) {
  if (bad("paged_release", n, blocks, ring_size, page)) return RB_ERR_ARG;
  const long long most = std::min<long long>((long long)n * blocks, ring_size);
  const long long ctas = std::min<long long>(std::max<long long>((most + 4 * kThreads - 1) / (4 * kThreads), 1), 148 * 2);
  rb_launch_pdl(release_kernel, dim3((unsigned)ctas), dim3(kThreads), 0, stream, table, table_stride, blocks, lens, reinterpret_cast<const uint8_t*>(done), n,
                Ring{ring, ring_size, 0, 0}, range, page, new_lens, new_range);
  return rb_check_launch("paged_release");
}
