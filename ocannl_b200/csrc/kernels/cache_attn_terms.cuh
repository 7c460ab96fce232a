// What the kernels of attention over a paged cache share: the arguments, which tokens a row sees, the score, and the plain row by row form.
//
// Row r of a sequence sees token j when j <= its position and, with a window, j >= first or j < sinks, where first is the position less the window
// plus one; tokens whose page is not there are seen by nobody.  Scores are kept in units of log 2, so that a weight is one exp2.
#ifndef B200_CACHE_ATTN_TERMS_CUH
#define B200_CACHE_ATTN_TERMS_CUH
#include "cache_terms.cuh"

namespace b200 {

struct CacheAttnArgs {
  CacheArgs c;
  const void* q;                       // [tokens, H, D]
  void* out;
  float* lse;                          // [tokens, H], or null
  const float* slopes;
  unsigned int* status;
  int H, group;                        // query heads, those that share a key head
  int window, sinks;                   // window 0: none
  float scale, cap, over;              // over: scale / cap
};

constexpr float kCacheLog2e = 1.4426950408889634f, kCacheLn2 = 0.6931471805599453f;

// the last token that a position sees, and the first of its window
__device__ __forceinline__ int cache_last(const CacheAttnArgs& a, int pos) {
  return (int)min((long long)pos, (long long)a.c.max_pages * a.c.page - 1);
}
// (positions ahead of the first token less a window of nearly 2^31 would pass 32 bits)
__device__ __forceinline__ int cache_first(const CacheAttnArgs& a, int pos) { return a.window ? max(max(pos, 0) - a.window + 1, 0) : 0; }

// a scale as the arithmetic takes it (what lies outside the range that codes are written with would not fit the weights)
__device__ __forceinline__ float cache_scale(float s) {
  return s != s ? s : fminf(fmaxf(s, 9.094947017729282e-13f), 1099511627776.f);        // 2^-40, 2^40
}

__device__ __forceinline__ float cache_score(const CacheAttnArgs& a, float qk, float slope2, int pos, int j) {
  const float s = a.cap > 0.f ? tanhf(qk * a.over) * (a.cap * kCacheLog2e) : qk * (a.scale * kCacheLog2e);
  return fmaf(-slope2, (float)(pos - j), s);
}

__device__ __forceinline__ float cache_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One row of a head by one warp: `row` of the packed nodes, at position `pos` of sequence b.  Only what the row sees is read: right whatever
// the rest holds, and the other kernels hand it the rows that come out infinite or undefined (0 times infinity from a token that is not seen).
// Elements lane, lane + 32, .. of a head, four at most.
template <class T, bool CODED>
__device__ __noinline__ void cache_attention_row(const CacheAttnArgs& a, int b, int h, int row, int pos, unsigned int lane) {
  const CacheArgs& c = a.c;
  const int hk = h / a.group;
  const long long at = ((long long)row * a.H + h) * c.D;
  const float slope2 = a.slopes ? a.slopes[h] * kCacheLog2e : 0.f;
  const int last = cache_last(a, pos), first = cache_first(a, pos);
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = (int)lane + 32 * i < c.D ? to_float(((const T*)a.q)[at + lane + 32 * i]) : 0.f;
  unsigned int index = 0xffffffffu;
  int page = -1;
  float ks = 1.f, vs = 1.f;
  for (int j = 0; j <= last; ++j) {
    if (j >= a.sinks && j < first) j = first;
    if (j > last) break;
    const unsigned int i = c.by_page.of((unsigned int)j);
    if (i != index) {
      index = i;
      page = cache_page_at(c, b, i);
      if (CODED && page >= 0) {
        ks = cache_scale(c.k_scale[(long long)page * c.HK + hk]);
        vs = cache_scale(c.v_scale[(long long)page * c.HK + hk]);
      }
    }
    if (page < 0) continue;
    const long long from = cache_at(c, page, hk) + (long long)((unsigned int)j - i * c.page) * c.D;
    float k[4], v[4], x = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool on = (int)lane + 32 * e < c.D;
      const long long p = from + lane + 32 * e;
      if constexpr (CODED) {
        k[e] = on ? e4m3_value(((const unsigned char*)c.k)[p]) : 0.f;
        v[e] = on ? e4m3_value(((const unsigned char*)c.v)[p]) * vs : 0.f;
      } else {
        k[e] = on ? to_float(((const T*)c.k)[p]) : 0.f;
        v[e] = on ? to_float(((const T*)c.v)[p]) : 0.f;
      }
      x = fmaf(q[e], k[e], x);
    }
    const float s = cache_score(a, cache_sum(x) * ks, slope2, pos, j);
    const float top = fmaxf(m, s);
    const float by = top == -INFINITY ? 1.f : exp2f(m - top), p = s == -INFINITY ? 0.f : exp2f(s - top);
    l = fmaf(l, by, p);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], by, p * v[e]);
    m = top;
  }
  const float by = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if ((int)lane + 32 * i < c.D) from_float(o[i] * by, ((T*)a.out)[at + lane + 32 * i]);
  if (a.lse && lane == 0) a.lse[(long long)row * a.H + h] = (m + log2f(l)) * kCacheLn2;
}

}  // namespace b200
#endif
