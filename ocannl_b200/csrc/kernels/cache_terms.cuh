// What the operators over a paged cache share: where a sequence's rows, pages and slots lie, and the 8-bit codes.
#ifndef B200_CACHE_TERMS_CUH
#define B200_CACHE_TERMS_CUH
#include "op_common.cuh"

namespace b200 {

struct CacheArgs {
  void *k, *v;                        // [pages, HK, page, D]
  float *k_scale, *v_scale;           // [pages, HK], with 8-bit codes
  const int *pages, *lengths, *starts;
  unsigned int n_pages, page, max_pages;
  int batch, tokens, each;            // each: rows of a sequence where there are no starts
  int HK, D;
  Divisor by_page;
};

// A sequence's new rows, and the position of the first (negative where the sequence has fewer tokens than new rows)
struct CacheSeq {
  int first, count, pos0;
};
__device__ __forceinline__ CacheSeq cache_seq(const CacheArgs& c, int b) {
  CacheSeq s;
  if (c.starts) {
    s.first = min(max(c.starts[b], 0), c.tokens);
    s.count = min(max(c.starts[b + 1], s.first), c.tokens) - s.first;
  } else {
    s.first = b * c.each;
    s.count = c.each;
  }
  s.pos0 = max(c.lengths[b], 0) - s.count;
  return s;
}
// the page that holds token j >= 0 of sequence b; -1: none
__device__ __forceinline__ int cache_page_at(const CacheArgs& c, int b, unsigned int index) {
  if (index >= c.max_pages) return -1;
  const int p = __ldg(c.pages + (long long)b * c.max_pages + index);
  return (unsigned int)p < c.n_pages ? p : -1;
}
// the first slot's element of a head in a page
__device__ __forceinline__ long long cache_at(const CacheArgs& c, int page, int hk) { return ((long long)page * c.HK + hk) * c.page * c.D; }

// ---- 8-bit codes
constexpr int kE4m3Least = -40, kE4m3Most = 40;                  // exponents of scales
constexpr float kE4m3Limit = 448.f * 1099511627776.f;            // 448 * 2^40: what is beyond has no code

__device__ __forceinline__ bool e4m3_has(float v) { return fabsf(v) <= kE4m3Limit; }
// The exponent of the least scale for values of up to `amax` (at most kE4m3Limit): 448 = 1.75 * 2^8
__device__ __forceinline__ int e4m3_exponent(float amax) {
  const unsigned int u = __float_as_uint(amax);
  return max((int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0), kE4m3Least);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned int)(e + 127) << 23); }    // -126 <= e <= 127
// two values, rounded to the nearest code; what is undefined keeps that
__device__ __forceinline__ unsigned int e4m3_pack2(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// the values of the two codes in the low half of w, as halves (exactly)
__device__ __forceinline__ unsigned int e4m3_halves(unsigned int w) {
  unsigned int r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)w));
  return r;
}
// the values of four codes, as two pairs of halves
__device__ __forceinline__ void e4m3_split(unsigned int w, unsigned int& lo, unsigned int& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float2 e4m3_unpack2(unsigned int w) {
  const unsigned int r = e4m3_halves(w);
  return __half22float2(*(const __half2*)&r);
}
__device__ __forceinline__ float e4m3_value(unsigned char w) { return e4m3_unpack2(w).x; }

// ---- blocks that share out a ragged batch: sequence b has units(b) of them, one behind the other.  The sequence of unit `target` and the unit's
// number in it; false for all threads if there is none.  Every thread of a block of NT calls it.
template <int NT, class F>
__device__ __forceinline__ bool find_unit(int batch, unsigned int target, F units, int& b, unsigned int& rest) {
  __shared__ unsigned int warps[NT / 32], found[2];
  const unsigned int lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  for (int b0 = 0; b0 < batch; b0 += NT) {
    const int i = b0 + (int)threadIdx.x;
    const unsigned int n = i < batch ? units(i) : 0u;
    unsigned int up_to = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int x = __shfl_up_sync(0xffffffffu, up_to, o);
      if (lane >= (unsigned int)o) up_to += x;
    }
    if (lane == 31) warps[warp] = up_to;
    if (threadIdx.x == 0) found[0] = 0xffffffffu;
    __syncthreads();
    unsigned int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      const unsigned int x = warps[w];
      if (w < (int)warp) before += x;
      all += x;
    }
    if (target < all) {
      if (before + up_to - n <= target && target < before + up_to) {
        found[0] = (unsigned int)i;
        found[1] = target - (before + up_to - n);
      }
      __syncthreads();
      b = (int)found[0];
      rest = found[1];
      __syncthreads();
      return b >= 0;                  // (sums that pass 32 bits, of starts that fall: nobody's)
    }
    target -= all;
    __syncthreads();                  // (the sums are written again)
  }
  return false;
}

}  // namespace b200
#endif
