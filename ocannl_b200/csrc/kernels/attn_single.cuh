// Attention and its gradients in single precision: products by fused multiply-adds (the tensor cores would read tf32), tiles of 64 x 64
// in shared memory, 256 threads, a thread 4 rows x 4 columns of a tile.  Bound by the multiply-adds and the shared-memory
// reads that feed them: four rows of one operand and four of the other are read 16 bytes at a time, 8 reads for 64 of them.
// Rows lie 4 floats more than their length apart, so that 8 neighbouring rows fill the banks.
#ifndef B200_ATTN_SINGLE_CUH
#define B200_ATTN_SINGLE_CUH
#include "attn_terms.cuh"

namespace b200 {

constexpr int kSide = 64, kSmall = kSide + 4;

// rows of a tile: what the queries are
struct SingleRows {
  int pos[kSide], last[kSide], doc[kSide], kdoc[kSide];
  float lse2[kSide], delta[kSide];
  unsigned int bad[kSide];
};

struct SingleShape {
  static __host__ __device__ int ld(int d) { return (d + 3) / 4 * 4 + 4; }
  static size_t smem(int d, int tiles) { return sizeof(SingleRows) + (size_t)tiles * kSide * ld(d) * 4 + kSide * kSmall * 4 * 2; }
};

// 64 rows from row `first` of [.., n, heads, d] into shared memory; zeros behind the last row and the last element.  A warp takes 8 rows.
__device__ __forceinline__ void single_load(float* to, const void* from, long long at, long long stride, int first, int n, int d, int ld, bool vec) {
  const int lane = (int)threadIdx.x & 31, w = (int)threadIdx.x >> 5, quads = (d + 3) / 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = w * 8 + i;
    if (lane >= quads) continue;
    const float* src = (const float*)from + at + (long long)(first + r) * stride + lane * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (first + r < n) {
      if (vec) {
        v = *(const float4*)src;
      } else {
        v.x = src[0];
        if (lane * 4 + 1 < d) v.y = src[1];
        if (lane * 4 + 2 < d) v.z = src[2];
        if (lane * 4 + 3 < d) v.w = src[3];
      }
    }
    *(float4*)(to + r * ld + lane * 4) = v;
  }
}
// acc[i][c] = <row 4 ty + i of x, row tx + 16 c of y>
__device__ __forceinline__ void single_dots(float (&acc)[4][4], const float* x, const float* y, int ld, int quads, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
  for (int e = 0; e < quads; ++e) {
    float4 u[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = *(const float4*)(x + (4 * ty + i) * ld + 4 * e);
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = *(const float4*)(y + (tx + 16 * c) * ld + 4 * e);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][c] = fmaf(u[i].x, w[c].x, fmaf(u[i].y, w[c].y, fmaf(u[i].z, w[c].z, fmaf(u[i].w, w[c].w, acc[i][c]))));
  }
}
// acc[i][4 q + k] += sum_j p[4 ty + i][j] y[j][4 tx + 64 q + k]
template <int Q>
__device__ __forceinline__ void single_add(float (&acc)[4][4 * Q], const float* p, const float* y, int ld, int d, int ty, int tx) {
  for (int j = 0; j < kSide; j += 4) {
    float4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = *(const float4*)(p + (4 * ty + i) * kSmall + j);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int e = 4 * tx + 64 * q;
      if (e >= d) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 w = *(const float4*)(y + (j + k) * ld + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float t = k == 0 ? u[i].x : k == 1 ? u[i].y : k == 2 ? u[i].z : u[i].w;
          acc[i][4 * q] = fmaf(t, w.x, acc[i][4 * q]);
          acc[i][4 * q + 1] = fmaf(t, w.y, acc[i][4 * q + 1]);
          acc[i][4 * q + 2] = fmaf(t, w.z, acc[i][4 * q + 2]);
          acc[i][4 * q + 3] = fmaf(t, w.w, acc[i][4 * q + 3]);
        }
      }
    }
  }
}
// rows of the result; false where a value is infinite or undefined
template <int Q>
__device__ __forceinline__ bool single_store(const float (&v)[4 * Q], float by, void* to, long long at, int d, int tx) {
  bool fine = true;
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = 4 * tx + 64 * q + k;
      const float y = by == 0.f ? 0.f : v[4 * q + k] * by;
      if (e < d) {
        ((float*)to)[at + e] = y;
        fine = fine && y * 0.f == 0.f;
      }
    }
  return fine;
}

__device__ __forceinline__ void single_queries(SingleRows* s, const AttnArgs& a, int b, int h, int r0) {
  const int i = (int)threadIdx.x;
  if (i < kSide) {
    AttnRow w;
    w.pos = 0; w.last = -1; w.doc = -1;
    if (r0 + i < a.S) w = attn_row(a, b, r0 + i);
    s->pos[i] = w.pos;
    s->last[i] = w.last;
    s->doc[i] = w.doc;
    if (a.stat && r0 + i < a.S) {
      const long long at = attn_stat_at(a, b, h, r0 + i);
      s->lse2[i] = a.stat[at];
      s->delta[i] = a.stat[at + 128];
    }
  }
}
__device__ __forceinline__ void single_keys(SingleRows* s, const AttnArgs& a, int b, int j0) {
  const int i = (int)threadIdx.x - kSide;
  if (a.kdoc && i >= 0 && i < kSide) s->kdoc[i] = j0 + i < a.T ? a.kdoc[(long long)b * a.T + j0 + i] : -1;
}
__device__ __forceinline__ bool single_sees(const SingleRows* s, const AttnArgs& a, int i, int j0, int c) {
  return j0 + c <= s->last[i] && (!a.kdoc || s->kdoc[c] == s->doc[i]);
}

template <int Q>
__global__ void __launch_bounds__(256) attn_forward_single(const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ __align__(128) unsigned char dyn[];
  grid_begin();
  SingleRows* s = (SingleRows*)dyn;
  const int ld = SingleShape::ld(a.D), quads = (a.D + 3) / 4, tile = kSide * ld;
  float *q = (float*)(dyn + sizeof(SingleRows)), *k = q + tile, *v = k + tile, *p = v + tile;
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.H;
  const int tiles_q = (a.S + kSide - 1) / kSide, r0 = (tiles_q - 1 - (int)(blockIdx.x / heads)) * kSide;
  const int b = (int)(blockIdx.x % heads) / a.H, h = (int)(blockIdx.x % heads) % a.H, hk = h / a.group;
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  single_queries(s, a, b, h, r0);
  single_load(q, a.q, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
  __syncthreads();
  int end = 0;
  for (int i = 0; i < kSide; ++i) end = max(end, s->last[i] + 1);
  float o[4][4 * Q], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) o[i][e] = 0.f;
  }
  for (int j0 = 0; j0 < end; j0 += kSide) {
    single_keys(s, a, b, j0);
    __syncthreads();
    bool on[4][4], any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) any |= on[i][c] = single_sees(s, a, 4 * ty + i, j0, tx + 16 * c);
    if (!__syncthreads_or(any)) continue;
    single_load(k, a.k, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
    single_load(v, a.v, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
    __syncthreads();
    float x[4][4], th;
    single_dots(x, q, k, ld, quads, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[i][c] = on[i][c] ? attn_score(a, x[i][c], slope2, s->pos[4 * ty + i], j0 + tx + 16 * c, th) : -INFINITY;
        top = fmaxf(top, x[i][c]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float next = fmaxf(m[i], top), by = m[i] == next ? 1.f : m[i] == -INFINITY ? 0.f : exp2f(m[i] - next);
      m[i] = next;
      l[i] *= by;
#pragma unroll
      for (int e = 0; e < 4 * Q; ++e) o[i][e] *= by;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float w = next == -INFINITY ? 0.f : exp2f(x[i][c] - next);
        l[i] += w;
        p[(4 * ty + i) * kSmall + tx + 16 * c] = w;
      }
    }
    __syncwarp();       // (a row of weights is written and read by one half warp)
    single_add<Q>(o, p, v, ld, a.D, ty, tx);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    const int r = r0 + 4 * ty + i;
    bool fine = true;
    if (r < a.S) {
      const bool on = l[i] > 0.f || l[i] != l[i];
      fine = single_store<Q>(o[i], on ? 1.f / l[i] : 0.f, a.out, attn_q_at(a, b, r, h), a.D, tx);
      if (tx == 0 && a.lse) a.lse[((long long)b * a.H + h) * a.S + r] = on ? (m[i] + log2f(l[i])) * kLn2 : -INFINITY;
    }
    const unsigned int bad = __ballot_sync(0xffffffffu, !fine);
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if ((bad >> (16 * w)) & 0xffffu) attn_forward_row<float>(a, b, h, r0 + (int)(threadIdx.x >> 5) * 8 + 4 * w + i, threadIdx.x & 31u);
  }
}

template <int Q>
__global__ void __launch_bounds__(256) attn_grad_queries_single(const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ __align__(128) unsigned char dyn[];
  grid_begin();
  SingleRows* s = (SingleRows*)dyn;
  const int ld = SingleShape::ld(a.D), quads = (a.D + 3) / 4, tile = kSide * ld;
  float *q = (float*)(dyn + sizeof(SingleRows)), *go = q + tile, *k = go + tile, *v = k + tile, *p = v + tile;
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.H;
  const int tiles_q = (a.S + kSide - 1) / kSide, r0 = (tiles_q - 1 - (int)(blockIdx.x / heads)) * kSide;
  const int b = (int)(blockIdx.x % heads) / a.H, h = (int)(blockIdx.x % heads) % a.H, hk = h / a.group;
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  single_queries(s, a, b, h, r0);
  single_load(q, a.q, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
  single_load(go, a.d_out, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
  __syncthreads();
  int end = 0;
  for (int i = 0; i < kSide; ++i) end = max(end, s->last[i] + 1);
  float g[4][4 * Q];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) g[i][e] = 0.f;
  for (int j0 = 0; j0 < end; j0 += kSide) {
    single_keys(s, a, b, j0);
    __syncthreads();
    bool on[4][4], any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) any |= on[i][c] = single_sees(s, a, 4 * ty + i, j0, tx + 16 * c);
    if (!__syncthreads_or(any)) continue;
    single_load(k, a.k, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
    single_load(v, a.v, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
    __syncthreads();
    float x[4][4], y[4][4], w, dx;
    single_dots(x, q, k, ld, quads, ty, tx);
    single_dots(y, go, v, ld, quads, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int r = 4 * ty + i;
        attn_pair(a, x[i][c], y[i][c], slope2, s->pos[r], j0 + tx + 16 * c, s->lse2[r], s->delta[r], w, dx);
        p[r * kSmall + tx + 16 * c] = on[i][c] ? dx : 0.f;
      }
    __syncwarp();
    single_add<Q>(g, p, k, ld, a.D, ty, tx);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * ty + i;
    const bool fine = r >= a.S || single_store<Q>(g[i], 1.f, a.dq, attn_q_at(a, b, r, h), a.D, tx);
    const unsigned int bad = __ballot_sync(0xffffffffu, !fine);
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if ((bad >> (16 * w)) & 0xffffu) attn_dq_row<float>(a, b, h, r0 + (int)(threadIdx.x >> 5) * 8 + 4 * w + i, threadIdx.x & 31u);
  }
}

template <int Q>
__global__ void __launch_bounds__(256) attn_grad_keys_single(const __grid_constant__ AttnArgs a, int vec) {
  extern __shared__ __align__(128) unsigned char dyn[];
  grid_begin();
  SingleRows* s = (SingleRows*)dyn;
  const int ld = SingleShape::ld(a.D), quads = (a.D + 3) / 4, tile = kSide * ld;
  float *q = (float*)(dyn + sizeof(SingleRows)), *go = q + tile, *k = go + tile, *v = k + tile, *p = v + tile, *ds = p + kSide * kSmall;
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.HK;
  const int j0 = (int)(blockIdx.x / heads) * kSide;
  const int b = (int)(blockIdx.x % heads) / a.HK, hk = (int)(blockIdx.x % heads) % a.HK;
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  single_keys(s, a, b, j0);
  single_load(k, a.k, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
  single_load(v, a.v, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
  float gk[4][4 * Q], gv[4][4 * Q];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) gk[i][e] = gv[i][e] = 0.f;
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    for (int r0 = 0; r0 < a.S; r0 += kSide) {
      __syncthreads();
      single_queries(s, a, b, h, r0);
      __syncthreads();
      bool on[4][4], any = false;       // of the thread's four keys and four queries
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) any |= on[i][c] = single_sees(s, a, tx + 16 * c, j0, 4 * ty + i);
      if (!__syncthreads_or(any)) continue;
      single_load(q, a.q, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
      single_load(go, a.d_out, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
      __syncthreads();
      float x[4][4], y[4][4], w, dx;
      single_dots(x, k, q, ld, quads, ty, tx);
      single_dots(y, v, go, ld, quads, ty, tx);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = tx + 16 * c;
          attn_pair(a, x[i][c], y[i][c], slope2, s->pos[r], j0 + 4 * ty + i, s->lse2[r], s->delta[r], w, dx);
          p[(4 * ty + i) * kSmall + r] = on[i][c] ? w : 0.f;
          ds[(4 * ty + i) * kSmall + r] = on[i][c] ? dx : 0.f;
        }
      __syncwarp();
      single_add<Q>(gv, p, go, ld, a.D, ty, tx);
      single_add<Q>(gk, ds, q, ld, a.D, ty, tx);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = j0 + 4 * ty + i;
    const bool fine_k = j >= a.T || single_store<Q>(gk[i], 1.f, a.dk, attn_k_at(a, b, j, hk), a.D, tx);
    const bool fine_v = j >= a.T || single_store<Q>(gv[i], 1.f, a.dv, attn_k_at(a, b, j, hk), a.D, tx);
    const unsigned int bad_k = __ballot_sync(0xffffffffu, !fine_k), bad_v = __ballot_sync(0xffffffffu, !fine_v);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int which = ((bad_k >> (16 * w)) & 0xffffu ? 1 : 0) | ((bad_v >> (16 * w)) & 0xffffu ? 2 : 0);
      if (which) attn_dkv_row<float>(a, b, hk, j0 + (int)(threadIdx.x >> 5) * 8 + 4 * w + i, threadIdx.x & 31u, which);
    }
  }
}

}  // namespace b200
#endif
