// Attention and its gradients in single precision: products by fused multiply-adds (the tensor cores would read tf32), tiles of 64 or 32
// rows of the block's own and 64 of the others in shared memory, 256 threads, a thread R = 4 or 2 rows x 4 columns.  Bound by the
// multiply-adds and the shared-memory reads that feed them (16 bytes each, 8 for 64 multiply-adds, which go two to an instruction where
// both operands lie in pairs).  Rows lie 4 floats more than their length apart, so that 8 neighbouring rows fill the banks.
#ifndef B200_ATTN_SINGLE_CUH
#define B200_ATTN_SINGLE_CUH
#include "attn_fwd_sm100.cuh"
#include "attn_terms.cuh"

namespace b200 {

constexpr int kSide = 64, kSmall = kSide + 4;

// rows of a tile: what the queries are
struct SingleRows {
  int pos[kSide], last[kSide], doc[kSide], kdoc[kSide];
  float lse2[kSide], delta[kSide];
};

struct SingleShape {
  static __host__ __device__ int ld(int d) { return (d + 3) / 4 * 4 + 4; }
  // tiles of the block's own rows, of weights, of the others (two each for one tile's place)
  static size_t smem(int d, int r, int own, int weights, int places) { return sizeof(SingleRows) + (size_t)(own * 16 * r + places * 2 * kSide) * ld(d) * 4 + (size_t)weights * 16 * r * kSmall * 4; }
};

// 8 W rows (W a warp) from row `first` of [.., n, heads, d] on their way into shared memory (cp.async); zeros behind the last row and the last element.
// Rows that are no multiple of 16 bytes come element by element.
template <int W>
__device__ __forceinline__ void single_load(float* to, const void* from, long long at, long long stride, int first, int n, int d, int ld, bool vec) {
  const int lane = (int)threadIdx.x & 31, w = (int)threadIdx.x >> 5, quads = (d + 3) / 4;
  if (lane < quads) {
    const float* src = (const float*)from + at + (long long)(first + w * W) * stride + lane * 4;
    const unsigned int dst = (unsigned int)__cvta_generic_to_shared(to + w * W * ld + lane * 4);
#pragma unroll
    for (int i = 0; i < W; ++i, src += stride) {
      const bool on = first + w * W + i < n;
      if (vec) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * ld * 4), "l"(on ? src : (const float*)from), "r"(on ? 16 : 0) : "memory");
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool in = on && lane * 4 + k < d;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + i * ld * 4 + 4 * k), "l"(in ? src + k : (const float*)from), "r"(in ? 4 : 0) : "memory");
        }
      }
    }
  }
}
__device__ __forceinline__ void single_sent() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all groups but the last, or all
__device__ __forceinline__ void single_arrived(bool but_last) {
  if (but_last) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
// acc[i][c] = <row R ty + i of x, row tx + 16 c of y>
template <int R>
__device__ __forceinline__ void single_dots(float (&acc)[R][4], const float* x, const float* y, int ld, int quads, int ty, int tx) {
  Pair sum[R][4];                   // even elements, odd elements
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[i][c] = Pair(0.f, 0.f);
  for (int e = 0; e < quads; ++e) {
    float4 u[R], w[4];
#pragma unroll
    for (int i = 0; i < R; ++i) u[i] = *(const float4*)(x + (R * ty + i) * ld + 4 * e);
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = *(const float4*)(y + (tx + 16 * c) * ld + 4 * e);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[i][c] = fma2(Pair(u[i].z, u[i].w), Pair(w[c].z, w[c].w), fma2(Pair(u[i].x, u[i].y), Pair(w[c].x, w[c].y), sum[i][c]));
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float even, odd;
      sum[i][c].get(even, odd);
      acc[i][c] = even + odd;
    }
}
// acc[i][4 q + k] += sum_j p[R ty + i][j] y[j][4 tx + 64 q + k]
template <int R, int Q>
__device__ __forceinline__ void single_add(float (&acc)[R][4 * Q], const float* p, const float* y, int ld, int d, int ty, int tx) {
  for (int j = 0; j < kSide; j += 4) {
    float4 u[R];
#pragma unroll
    for (int i = 0; i < R; ++i) u[i] = *(const float4*)(p + (R * ty + i) * kSmall + j);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int e = 4 * tx + 64 * q;
      if (e >= d) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 w = *(const float4*)(y + (j + k) * ld + e);
#pragma unroll
        for (int i = 0; i < R; ++i) {
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

// A thread's query of a tile, fetched ahead of its use
struct SingleQuery {
  int last, doc;
  float lse2, delta;
  __device__ __forceinline__ void fetch(const AttnArgs& a, const AttnSeq& q, int b, int h, int r) {
    last = doc = -1;
    if (threadIdx.x < kSide && r < a.S) {
      last = attn_last(a, q, r);
      doc = 0;
      if (a.qdoc) {
        doc = a.qdoc[(long long)b * a.S + r];
        if (doc < 0) last = -1;
      }
      if (a.stat) {
        const long long at = attn_stat_at(a, b, h, r);
        lse2 = a.stat[at];
        delta = a.stat[at + 128];
      }
    }
  }
  __device__ __forceinline__ void put(SingleRows* s, const AttnArgs& a, const AttnSeq& q, int r) const {
    const int i = (int)threadIdx.x;
    if (i < kSide) {
      s->pos[i] = q.len - a.S + r;
      s->last[i] = last;
      s->doc[i] = doc;
      s->lse2[i] = lse2;
      s->delta[i] = delta;
    }
  }
};
__device__ __forceinline__ void single_keys(SingleRows* s, const AttnArgs& a, int b, int j0) {
  const int i = (int)threadIdx.x - kSide;
  if (a.kdoc && i >= 0 && i < kSide) s->kdoc[i] = j0 + i < a.T ? a.kdoc[(long long)b * a.T + j0 + i] : -1;
}
__device__ __forceinline__ bool single_sees(const SingleRows* s, const AttnArgs& a, int i, int j0, int c) {
  return j0 + c <= s->last[i] && (!a.kdoc || s->kdoc[c] == s->doc[i]);
}

template <int Q, int R>
__global__ void __launch_bounds__(256, R == 2 ? 2 : 1) attn_forward_single(const __grid_constant__ AttnArgs a, int vec, int places) {
  extern __shared__ __align__(128) unsigned char dyn[];
  grid_begin();
  SingleRows* s = (SingleRows*)dyn;
  const int ld = SingleShape::ld(a.D), quads = (a.D + 3) / 4, tile = kSide * ld, own = 16 * R * ld;
  float *q = (float*)(dyn + sizeof(SingleRows)), *p = q + own, *k = p + 16 * R * kSmall;
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.H;
  const int tiles_q = (a.S + 16 * R - 1) / (16 * R), r0 = (tiles_q - 1 - (int)(blockIdx.x / heads)) * 16 * R;
  const int b = (int)(blockIdx.x % heads) / a.H, h = (int)(blockIdx.x % heads) % a.H, hk = h / a.group;
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  const AttnSeq seq = attn_seq(a, b);
  SingleQuery mine;
  mine.fetch(a, seq, b, h, r0 + (int)threadIdx.x);
  mine.put(s, a, seq, r0 + (int)threadIdx.x);
  single_load<2 * R>(q, a.q, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
  __syncthreads();
  int end = 0;
  for (int i = 0; i < 16 * R; ++i) end = max(end, s->last[i] + 1);
  float o[R][4 * Q], m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) o[i][e] = 0.f;
  }
  // The next tile of keys is on its way while this one is worked on, where there is room for two (`places`).  A warp of its own decides
  // whether its rows see anything of a tile.
  const long long k_at = attn_k_at(a, b, 0, hk), k_step = (long long)a.HK * a.ld;
  auto load = [&](int j0, int n) {
    float* to = k + (n & (places - 1)) * 2 * tile;
    single_load<8>(to, a.k, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_load<8>(to + tile, a.v, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_sent();
  };
  if (places == 2 && end > 0) load(0, 0);
  for (int j0 = 0, n = 0; j0 < end; j0 += kSide, ++n) {
    __syncthreads();
    const bool more = places == 2 && j0 + kSide < end;
    if (places == 1) load(j0, n);
    else if (more) load(j0 + kSide, n + 1);
    single_keys(s, a, b, j0);
    single_arrived(more);
    __syncthreads();
    const float *kt = k + (n & (places - 1)) * 2 * tile, *vt = kt + tile;
    bool on[R][4], any = false;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) any |= on[i][c] = single_sees(s, a, R * ty + i, j0, tx + 16 * c);
    if (!__any_sync(0xffffffffu, any)) continue;
    float x[R][4], th;
    single_dots<R>(x, q, kt, ld, quads, ty, tx);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[i][c] = on[i][c] ? attn_score(a, x[i][c], slope2, s->pos[R * ty + i], j0 + tx + 16 * c, th) : -INFINITY;
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
        p[(R * ty + i) * kSmall + tx + 16 * c] = w;
      }
    }
    __syncwarp();       // (a row of weights is written and read by one half warp)
    single_add<R, Q>(o, p, vt, ld, a.D, ty, tx);
    __syncwarp();
  }
  single_sent();
  single_arrived(false);
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    const int r = r0 + R * ty + i;
    bool fine = true;
    if (r < a.S) {
      const bool on = l[i] > 0.f || l[i] != l[i];
      fine = single_store<Q>(o[i], on ? 1.f / l[i] : 0.f, a.out, attn_q_at(a, b, r, h), a.D, tx);
      if (tx == 0 && a.lse) a.lse[((long long)b * a.H + h) * a.S + r] = on ? (m[i] + log2f(l[i])) * kLn2 : -INFINITY;
    }
    const unsigned int bad = __ballot_sync(0xffffffffu, !fine);
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if ((bad >> (16 * w)) & 0xffffu) attn_forward_row<float>(a, b, h, r0 + (int)(threadIdx.x >> 5) * 2 * R + R * w + i, threadIdx.x & 31u);
  }
}

template <int Q, int R>
__global__ void __launch_bounds__(256, R == 2 ? 2 : 1) attn_grad_queries_single(const __grid_constant__ AttnArgs a, int vec, int places) {
  extern __shared__ __align__(128) unsigned char dyn[];
  grid_begin();
  SingleRows* s = (SingleRows*)dyn;
  const int ld = SingleShape::ld(a.D), quads = (a.D + 3) / 4, tile = kSide * ld, own = 16 * R * ld;
  float *q = (float*)(dyn + sizeof(SingleRows)), *go = q + own, *p = go + own, *k = p + 16 * R * kSmall;
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.H;
  const int tiles_q = (a.S + 16 * R - 1) / (16 * R), r0 = (tiles_q - 1 - (int)(blockIdx.x / heads)) * 16 * R;
  const int b = (int)(blockIdx.x % heads) / a.H, h = (int)(blockIdx.x % heads) % a.H, hk = h / a.group;
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  const AttnSeq seq = attn_seq(a, b);
  SingleQuery mine;
  mine.fetch(a, seq, b, h, r0 + (int)threadIdx.x);
  mine.put(s, a, seq, r0 + (int)threadIdx.x);
  single_load<2 * R>(q, a.q, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
  single_load<2 * R>(go, a.d_out, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
  __syncthreads();
  int end = 0;
  for (int i = 0; i < 16 * R; ++i) end = max(end, s->last[i] + 1);
  float g[R][4 * Q];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) g[i][e] = 0.f;
  const long long k_at = attn_k_at(a, b, 0, hk), k_step = (long long)a.HK * a.ld;
  auto load = [&](int j0, int n) {
    float* to = k + (n & (places - 1)) * 2 * tile;
    single_load<8>(to, a.k, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_load<8>(to + tile, a.v, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_sent();
  };
  if (places == 2 && end > 0) load(0, 0);
  for (int j0 = 0, n = 0; j0 < end; j0 += kSide, ++n) {
    __syncthreads();
    const bool more = places == 2 && j0 + kSide < end;
    if (places == 1) load(j0, n);
    else if (more) load(j0 + kSide, n + 1);
    single_keys(s, a, b, j0);
    single_arrived(more);
    __syncthreads();
    const float *kt = k + (n & (places - 1)) * 2 * tile, *vt = kt + tile;
    bool on[R][4], any = false;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) any |= on[i][c] = single_sees(s, a, R * ty + i, j0, tx + 16 * c);
    if (!__any_sync(0xffffffffu, any)) continue;
    float x[R][4], y[R][4], w, dx;
    single_dots<R>(x, q, kt, ld, quads, ty, tx);
    single_dots<R>(y, go, vt, ld, quads, ty, tx);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int r = R * ty + i;
        attn_pair(a, x[i][c], y[i][c], slope2, s->pos[r], j0 + tx + 16 * c, s->lse2[r], s->delta[r], w, dx);
        p[r * kSmall + tx + 16 * c] = on[i][c] ? dx : 0.f;
      }
    __syncwarp();
    single_add<R, Q>(g, p, kt, ld, a.D, ty, tx);
    __syncwarp();
  }
  single_sent();
  single_arrived(false);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + R * ty + i;
    const bool fine = r >= a.S || single_store<Q>(g[i], 1.f, a.dq, attn_q_at(a, b, r, h), a.D, tx);
    const unsigned int bad = __ballot_sync(0xffffffffu, !fine);
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if ((bad >> (16 * w)) & 0xffffu) attn_dq_row<float>(a, b, h, r0 + (int)(threadIdx.x >> 5) * 2 * R + R * w + i, threadIdx.x & 31u);
  }
}

template <int Q, int R>
__global__ void __launch_bounds__(256, R == 2 ? 2 : 1) attn_grad_keys_single(const __grid_constant__ AttnArgs a, int vec, int places) {
  extern __shared__ __align__(128) unsigned char dyn[];
  grid_begin();
  SingleRows* s = (SingleRows*)dyn;
  const int ld = SingleShape::ld(a.D), quads = (a.D + 3) / 4, tile = kSide * ld, own = 16 * R * ld;
  float *k = (float*)(dyn + sizeof(SingleRows)), *v = k + own, *p = v + own, *ds = p + 16 * R * kSmall, *q = ds + 16 * R * kSmall;
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.HK;
  const int j0 = (int)(blockIdx.x / heads) * 16 * R;
  const int b = (int)(blockIdx.x % heads) / a.HK, hk = (int)(blockIdx.x % heads) % a.HK;
  const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
  single_keys(s, a, b, j0);
  single_load<2 * R>(k, a.k, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
  single_load<2 * R>(v, a.v, attn_k_at(a, b, 0, hk), (long long)a.HK * a.ld, j0, a.T, a.D, ld, vec);
  float gk[R][4 * Q], gv[R][4 * Q];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) gk[i][e] = gv[i][e] = 0.f;
  single_sent();
  const AttnSeq seq = attn_seq(a, b);
  // the first tile of queries that see a key of the block's (later ones see no fewer)
  int begin = 0;
  while (begin < a.S && attn_last(a, seq, min(begin + kSide, a.S) - 1) < j0) begin += kSide;
  auto load = [&](int h, int r0, int n) {
    float* to = q + (n & (places - 1)) * 2 * tile;
    const long long at = attn_q_at(a, b, 0, h), step = (long long)a.H * a.ld;
    single_load<8>(to, a.q, at, step, r0, a.S, a.D, ld, vec);
    single_load<8>(to + tile, a.d_out, at, step, r0, a.S, a.D, ld, vec);
    single_sent();
  };
  const int last_head = (hk + 1) * a.group - 1;
  SingleQuery next;
  if (begin < a.S) {
    next.fetch(a, seq, b, hk * a.group, begin + (int)threadIdx.x);
    if (places == 2) load(hk * a.group, begin, 0);
  }
  int n = 0;
  for (int h = hk * a.group; h <= last_head; ++h) {
    const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    for (int r0 = begin; r0 < a.S; r0 += kSide, ++n) {
      __syncthreads();
      const bool more = r0 + kSide < a.S || h < last_head;
      const int next_h = r0 + kSide < a.S ? h : h + 1, next_r = r0 + kSide < a.S ? r0 + kSide : begin;
      if (places == 1) load(h, r0, n);
      else if (more) load(next_h, next_r, n + 1);
      next.put(s, a, seq, r0 + (int)threadIdx.x);
      if (more) next.fetch(a, seq, b, next_h, next_r + (int)threadIdx.x);
      single_arrived(places == 2 && more);
      __syncthreads();
      const float *qt = q + (n & (places - 1)) * 2 * tile, *gt = qt + tile;
      bool on[R][4], any = false;       // of the thread's keys and four queries
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) any |= on[i][c] = single_sees(s, a, tx + 16 * c, j0, R * ty + i);
      if (!__any_sync(0xffffffffu, any)) continue;
      float x[R][4], y[R][4], w, dx;
      single_dots<R>(x, k, qt, ld, quads, ty, tx);
      single_dots<R>(y, v, gt, ld, quads, ty, tx);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = tx + 16 * c;
          attn_pair(a, x[i][c], y[i][c], slope2, s->pos[r], j0 + R * ty + i, s->lse2[r], s->delta[r], w, dx);
          p[(R * ty + i) * kSmall + r] = on[i][c] ? w : 0.f;
          ds[(R * ty + i) * kSmall + r] = on[i][c] ? dx : 0.f;
        }
      __syncwarp();
      single_add<R, Q>(gv, p, gt, ld, a.D, ty, tx);
      single_add<R, Q>(gk, ds, qt, ld, a.D, ty, tx);
      __syncwarp();
    }
  }
  single_arrived(false);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int j = j0 + R * ty + i;
    const bool fine_k = j >= a.T || single_store<Q>(gk[i], 1.f, a.dk, attn_k_at(a, b, j, hk), a.D, tx);
    const bool fine_v = j >= a.T || single_store<Q>(gv[i], 1.f, a.dv, attn_k_at(a, b, j, hk), a.D, tx);
    const unsigned int bad_k = __ballot_sync(0xffffffffu, !fine_k), bad_v = __ballot_sync(0xffffffffu, !fine_v);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int which = ((bad_k >> (16 * w)) & 0xffffu ? 1 : 0) | ((bad_v >> (16 * w)) & 0xffffu ? 2 : 0);
      if (which) attn_dkv_row<float>(a, b, hk, j0 + (int)(threadIdx.x >> 5) * 2 * R + R * w + i, threadIdx.x & 31u, which);
    }
  }
}

}  // namespace b200
#endif
