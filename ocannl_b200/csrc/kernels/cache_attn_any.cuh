// Attention of new tokens over a paged cache in single precision arithmetic: single heads, and 16-bit ones whose rows are no whole 16-byte pieces.
//
// A block takes 8 rows of a (sequence, key head) and a part of their tokens, as the tensor-core form for few rows does, 32 tokens at a time in
// shared memory as floats.  A warp has two rows: a lane a token for the scores, four elements for the output.  Bound by shared memory: a warp reads a
// tile's keys and values once for two rows, some 350 accesses of 128 bytes each for heads of 128 elements, so four warps take 32 KB of cache in 1400 cycles,
// which is the rate at which an SM gets them from memory; warps without rows read nothing.  Scores keep their own unit until the maximum is taken off: rounded
// in units of log 2 first, scores of 50 would cost weights 2^-18.
#ifndef B200_CACHE_ATTN_ANY_CUH
#define B200_CACHE_ATTN_ANY_CUH
#include "cache_attn_few_sm100.cuh"

namespace b200 {

constexpr int kAnyRows = 8, kAnyTokens = 32, kAnyWidth = 132;
// floats from one row to the next in shared memory: an odd number of 16 bytes, so that eight lanes' 16 bytes lie in banks of their own
__host__ __device__ constexpr int any_pitch(int d) { return (d + 7) / 8 * 8 + 4; }
inline size_t any_smem(int d) { return (size_t)(kAnyRows + 2 * kAnyTokens) * any_pitch(d) * 4; }

template <class T, bool CODED>
__global__ void __launch_bounds__(kCacheFewThreads) cache_attention_any(const __grid_constant__ CacheAttnArgs a, const __grid_constant__ CacheFewArgs f, const int vec) {
  extern __shared__ __align__(16) float any_shared[];
  __shared__ long long places[kAnyTokens];          // elements of the cache ahead of a token's row, -1: not there
  __shared__ float scale_of[2][kAnyTokens];
  __shared__ float weight_of[kCacheFewWarps][2][kAnyTokens];
  __shared__ float weigh[kCacheFewWarps][kFewMost];
  __shared__ unsigned int last_block;
  const CacheArgs& c = a.c;
  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  grid_begin();
  CachePart part;
  if (!cache_part<kCacheFewThreads, kAnyRows>(a, f, part)) return;
  const int pitch = any_pitch(c.D);
  CachePiece plan;
  for (; cache_piece<kAnyRows>(a, f, part, plan); cache_advance<kAnyRows>(a, part)) {
  const int rows = plan.rows;
  float *const q = any_shared, *const keys = q + kAnyRows * pitch, *const values = keys + kAnyTokens * pitch;
  auto query_of = [&](int i) { return (int)f.by_group.of((unsigned int)(plan.first_row + i)); };
  auto head_of = [&](int i) { return plan.hk * a.group + plan.first_row + i - query_of(i) * a.group; };
  for (int i = (int)threadIdx.x; i < kAnyRows * pitch; i += kCacheFewThreads) {
    const int r = i / pitch, e = i - r * pitch;
    q[i] = r < rows && e < c.D ? to_float(((const T*)a.q)[((long long)(part.s.first + query_of(r)) * a.H + head_of(r)) * c.D + e]) : 0.f;
  }
  const int r0 = 2 * (int)warp;                     // this warp's rows are r0 and r0 + 1
  const bool mine = r0 < rows;
  int pos[2];
  float slope[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = min(r0 + k, rows - 1);
    pos[k] = part.s.pos0 + query_of(r);
    slope[k] = a.slopes ? a.slopes[head_of(r)] : 0.f;
  }
  float o[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  for (unsigned int v0 = (unsigned int)plan.begin; v0 < (unsigned int)plan.stop; v0 += kAnyTokens) {      // (of up to 2^31 - 1 tokens: signed numbers would not end)
    __syncthreads();
    if (threadIdx.x < kAnyTokens) {
      const unsigned int v = v0 + threadIdx.x;
      const int j = v < (unsigned int)plan.stop ? plan.token_of((int)v) : plan.end;
      long long place = -1;
      float ks = 0.f, vs = 0.f;
      if (j < plan.end) {
        const unsigned int index = c.by_page.of((unsigned int)j);
        const int page = cache_page_at(c, part.b, index);
        if (page >= 0) {
          place = cache_at(c, page, plan.hk) + (long long)((unsigned int)j - index * c.page) * c.D;
          if (CODED) {
            ks = cache_scale(c.k_scale[(long long)page * c.HK + plan.hk]);
            vs = cache_scale(c.v_scale[(long long)page * c.HK + plan.hk]);
          }
        }
      }
      places[threadIdx.x] = place;
      scale_of[0][threadIdx.x] = ks;
      scale_of[1][threadIdx.x] = vs;
    }
    __syncthreads();
    // keys and values as floats; zeros where there are none, and behind a row's end
    if (vec) {
      constexpr int V = CODED ? 4 : 16 / (int)sizeof(T);
      const int pieces = pitch / 4 - 1, each = CODED || V == 4 ? pieces : (pieces + 1) / 2;     // (whole pieces of V elements: D is a multiple of V)
      for (int i = (int)threadIdx.x; i < 2 * kAnyTokens * each; i += kCacheFewThreads) {
        const int row = i / each, e = (i - row * each) * V, token = row & (kAnyTokens - 1), which = row >= kAnyTokens;
        float x[V];
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = 0.f;
        const long long place = places[token];
        if (place >= 0 && e < c.D) {
          if constexpr (CODED) {
            const unsigned int w = *(const unsigned int*)((const unsigned char*)(which ? c.v : c.k) + place + e);
            const float2 lo = e4m3_unpack2(w & 0xffffu), hi = e4m3_unpack2(w >> 16);
            const float by = scale_of[which][token];
            x[0] = lo.x * by; x[1] = lo.y * by; x[2] = hi.x * by; x[3] = hi.y * by;
          } else {
            Vec<T, V>::load((const T*)(which ? c.v : c.k) + place + e, x);
          }
        }
        float* to = (which ? values : keys) + token * pitch + e;
#pragma unroll
        for (int k = 0; k < V; k += 4) *(float4*)(to + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
      }
    } else {
      for (int i = (int)threadIdx.x; i < 2 * kAnyTokens * pitch; i += kCacheFewThreads) {
        const int row = i / pitch, e = i - row * pitch, token = row & (kAnyTokens - 1), which = row >= kAnyTokens;
        const long long place = places[token];
        float x = 0.f;
        if (place >= 0 && e < c.D) {
          if constexpr (CODED) x = e4m3_value(((const unsigned char*)(which ? c.v : c.k))[place + e]) * scale_of[which][token];
          else x = to_float(((const T*)(which ? c.v : c.k))[place + e]);
        }
        (which ? values : keys)[token * pitch + e] = x;
      }
    }
    __syncthreads();
    if (!mine) continue;
    // scores: a lane a token; four sums a row
    float s[2];
    {
      float4 sum[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
      const float *key = keys + lane * pitch, *q0 = q + r0 * pitch;
#pragma unroll 4
      for (int e = 0; e < pitch - 4; e += 4) {
        const float4 k = *(const float4*)(key + e);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 x = *(const float4*)(q0 + i * pitch + e);
          sum[i] = make_float4(fmaf(x.x, k.x, sum[i].x), fmaf(x.y, k.y, sum[i].y), fmaf(x.z, k.z, sum[i].z), fmaf(x.w, k.w, sum[i].w));
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i] = (sum[i].x + sum[i].y) + (sum[i].z + sum[i].w);
    }
    const int j = places[lane] >= 0 ? plan.token_of((int)(v0 + lane)) : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = a.cap > 0.f ? tanhf(s[i] * a.over) * a.cap : s[i] * a.scale;
      s[i] = fmaf(-slope[i], (float)(pos[i] - j), s[i]);
      if (places[lane] < 0 || j > cache_last(a, pos[i]) || (j < cache_first(a, pos[i]) && j >= a.sinks)) s[i] = -INFINITY;
      float top = s[i];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float next = fmaxf(m[i], top);
      if (next != m[i]) {
        const float by = m[i] == -INFINITY ? 0.f : exp2f((m[i] - next) * kCacheLog2e);
        m[i] = next;
        l[i] *= by;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] *= by;
      }
      const float w = s[i] == -INFINITY ? 0.f : exp2f((s[i] - (next == -INFINITY ? 0.f : next)) * kCacheLog2e);
      l[i] += w;
      weight_of[warp][i][lane] = w;
    }
    __syncwarp();
    if (4 * (int)lane < c.D) {
      float4 sum[2][2];                             // of even and odd tokens, so that rounding does not add up in one
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i >> 1][i & 1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int t = 0; t < kAnyTokens; t += 2)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 v = *(const float4*)(values + (t + k) * pitch + 4 * lane);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float w = weight_of[warp][i][t + k];
            float4& u = sum[i][k];
            u = make_float4(fmaf(w, v.x, u.x), fmaf(w, v.y, u.y), fmaf(w, v.z, u.z), fmaf(w, v.w, u.w));
          }
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        o[i][0] += sum[i][0].x + sum[i][1].x;
        o[i][1] += sum[i][0].y + sum[i][1].y;
        o[i][2] += sum[i][0].z + sum[i][1].z;
        o[i][3] += sum[i][0].w + sum[i][1].w;
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) l[i] = cache_sum(l[i]);
  auto finish = [&](int i, const float4& v, float top, float sum) {
    const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const float y[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
    const int row = part.s.first + query_of(i), h = head_of(i);
    const long long at = (long long)row * a.H + h;
    bool fine = true;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (4 * (int)lane + k < c.D) {
        from_float(y[k], ((T*)a.out)[at * c.D + 4 * lane + k]);
        fine = fine && y[k] * 0.f == 0.f;
      }
    if (lane == 0 && a.lse) a.lse[at] = by != 0.f ? top + logf(sum) : -INFINITY;
    if (attn_again(fine)) cache_attention_row<T, CODED>(a, part.b, h, row, part.s.pos0 + query_of(i), lane);
  };
  if (plan.parts == 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (r0 + i < rows) finish(r0 + i, make_float4(o[i][0], o[i][1], o[i][2], o[i][3]), m[i], l[i]);
  } else {
    float* parts = f.parts + cache_part_at(plan.first_block, plan.part) * kAnyRows * kAnyWidth;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (r0 + i < rows) {
        float* row = parts + (r0 + i) * kAnyWidth;
        *(float4*)(row + 4 * lane) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
        if (lane == 0) {
          row[128] = m[i];
          row[129] = l[i];
        }
      }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      last_block = plan.meets && atomicAdd(&f.tickets[plan.first_block], 1u) == plan.parts - 1u;
      if (last_block) f.tickets[plan.first_block] = 0u;        // for the next run
    }
    __syncthreads();
    if (last_block) {
      __threadfence();
      const int n = (int)plan.parts;
      for (int i = (int)warp; i < rows; i += kCacheFewWarps) {
        // (the maxima are in the scores' unit; a part without visible tokens has a sum of exactly 0 and counts nothing)
        const float* from = f.parts + cache_part_at(plan.first_block, 0) * kAnyRows * kAnyWidth + i * kAnyWidth;
        float top, sum;
        const float4 v = cache_join<128, kAnyRows>([](float x) { return exp2f(x * kCacheLog2e); }, from, n, weigh[warp], true, 4 * (int)lane, top, sum);
        finish(i, v, top, sum);
      }
    }
  }
  __syncthreads();                                  // (what is shared is written again)
  }
}

}  // namespace b200
#endif
