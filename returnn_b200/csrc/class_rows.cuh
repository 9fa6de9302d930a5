// Rows of a matrix of classes, bf16 or fp32, that start anywhere: single elements up to a 16-byte boundary, 16-byte chunks from there on.
#pragma once
#include "common.cuh"

namespace rows {

__device__ __forceinline__ float ld(const void* x, int64_t i, int is_bf16) {
  return is_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[i]) : reinterpret_cast<const float*>(x)[i];
}

// A row of an odd vocabulary starts anywhere: single elements up to the first 16-byte boundary of the logits, 16-byte accesses from there
// on, single elements at the end. (With single elements for every such row, 6000 x 10025 took as long as 6000 x 32000.)
__device__ __forceinline__ int row_head(const void* x, int64_t base, int v, int elem) {
  const int off = (int)((reinterpret_cast<uintptr_t>(x) + (uint64_t)base * elem) & 15);
  return min(off ? (16 - off) / elem : 0, v);
}

// 16 bytes: 8 bf16 or 4 fp32 values
template <bool kBf16>
struct Chunk {
  static constexpr int kN = kBf16 ? 8 : 4;
  uint4 u;
  __device__ __forceinline__ void load(const void* x, int64_t at) {
    u = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(x) + at * (kBf16 ? 2 : 4));
  }
  __device__ __forceinline__ void fill_neg_inf() { u.x = u.y = u.z = u.w = kBf16 ? 0xff80ff80u : 0xff800000u; }
  __device__ __forceinline__ float at(int i) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
    if (kBf16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    return __uint_as_float(w[i]);
  }
  __device__ __forceinline__ float max() const {
    if (kBf16) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
      const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
      return fmaxf(m.x, m.y);
    }
    return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
  }
};

}  // namespace rows
