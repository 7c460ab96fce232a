// Attention and its gradients in single precision on mma.sync.m16n8k8 with tf32 operands in two parts each.
//
// The multiply-add units make 73 TFLOP/s, these instructions 276 (both measured): x = hi + lo with 11 bits each, and
// hi hi + hi lo + lo hi keeps 2^-21 of a product at a third of their rate.  The tensor cores cut sums off instead of rounding them, so at
// most six products in a row are summed there, from zero; the results are added to the accumulators by ordinary additions.
//
// A warp has 16 rows of its own (queries, or keys for the keys' gradients) and walks the others 32 at a time; two or four warps share
// the rows and take the steps in turn (one warp an SM quarter left the products waiting for one another: tensor pipe 27 % busy), their
// parts meet in shared memory at the end, in order.  The others' tiles lie in shared memory, the next ones on their way (cp.async) where
// there is room for two places; scores and weights stay in registers, where the accumulator layout of the first product is the operand
// layout of the second up to the order of its terms.  Rows lie 8 floats more than a
// multiple of 32 apart.  Rows that come out infinite or undefined (0 times infinity at a place that is not seen, values next to the
// largest float) are done again one by one.
#ifndef B200_ATTN_SINGLE_CUH
#define B200_ATTN_SINGLE_CUH
#include "attn_fwd_sm100.cuh"
#include "attn_terms.cuh"

namespace b200 {

constexpr int kOthers = 32, kOtherTiles = kOthers / 8;    // rows of a step, columns of a warp's scores in eights
constexpr int kMostShares = 4;                            // warps that share their rows

struct SingleShape {
  static __host__ __device__ int ld(int d) { return (d + 31) / 32 * 32 + 8; }
  // own rows of `own` tensors, `places` times the others' two tiles of a step of every share, their descriptions
  static size_t smem(int d, int groups, int shares, int own, int places) {
    return (size_t)(own * 16 * groups + places * 2 * kOthers * shares) * ld(d) * 4 + 5 * kOthers * kMostShares * 4;
  }
  // ... of which the others' tiles take the parts of the warps that are not the first of their rows (`own` sums of DT eights, four more values)
  static bool room_to_meet(int d, int groups, int shares, int own, int places, int dt) {
    return (size_t)(shares - 1) * groups * (own * dt * 4 + 4) * 32 <= (size_t)places * 2 * kOthers * shares * ld(d);
  }
};

// `rows` rows from row `first` of [.., n, heads, d] on their way into shared memory; zeros behind the last row and up to a multiple of 8
// elements.  Rows that are no multiple of 16 bytes come element by element.
__device__ __forceinline__ void single_load(float* to, int rows, const void* from, long long at, long long stride, int first, int n, int d, int ld, int vec) {
  const int lane = (int)threadIdx.x & 31, warps = (int)blockDim.x >> 5;
  if (lane >= (d + 7) / 8 * 2) return;
  for (int r = (int)threadIdx.x >> 5; r < rows; r += warps) {
    const float* src = (const float*)from + at + (long long)(first + r) * stride + lane * 4;
    const unsigned int dst = (unsigned int)__cvta_generic_to_shared(to + r * ld + lane * 4);
    const bool on = first + r < n;
    if (vec) {
      const bool in = on && lane * 4 < d;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(in ? src : (const float*)from), "r"(in ? 16 : 0) : "memory");
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = on && lane * 4 + k < d;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * k), "l"(in ? src + k : (const float*)from), "r"(in ? 4 : 0) : "memory");
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

// x in two parts of 11 bits, the first rounded
__device__ __forceinline__ void tf32_parts(float x, unsigned int& hi, unsigned int& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const unsigned int (&x)[4], unsigned int y0, unsigned int y1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(y0), "r"(y1));
}
struct PartsA {
  unsigned int hi[4], lo[4];
};
// d[i] += x y_i for N operands side by side, in three products, the small ones first.  (One operand after the other would be a chain of
// three dependent instructions each: gradients of 2 x 1024 positions took 340 us.)
template <int N>
__device__ __forceinline__ void mma_parts(float (&d)[N][4], const PartsA& x, const float (&y)[N][2]) {
  unsigned int h[N][2], l[N][2];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    tf32_parts(y[i][0], h[i][0], l[i][0]);
    tf32_parts(y[i][1], h[i][1], l[i][1]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) mma_tf32(d[i], x.lo, h[i][0], h[i][1]);
#pragma unroll
  for (int i = 0; i < N; ++i) mma_tf32(d[i], x.hi, l[i][0], l[i][1]);
#pragma unroll
  for (int i = 0; i < N; ++i) mma_tf32(d[i], x.hi, h[i][0], h[i][1]);
}

// acc[n] = (16 rows of x from its first) . (rows 8 n .. of y): elements 2 t and 2 t + 1 of each eight are k index t and t + 4.
// steps: eights of elements
__device__ __forceinline__ void single_dots(float (&acc)[kOtherTiles][4], const float* x, const float* y, int ld, int steps) {
  const int g = ((int)threadIdx.x & 31) >> 2, t = (int)threadIdx.x & 3;
#pragma unroll
  for (int n = 0; n < kOtherTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  const float *x0 = x + g * ld + 2 * t, *x1 = x0 + 8 * ld, *y0 = y + g * ld + 2 * t;
  for (int s = 0; s < steps; s += 2) {
    float part[kOtherTiles][4];
#pragma unroll
    for (int n = 0; n < kOtherTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[n][i] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (s + k >= steps) continue;
      const float2 u = *(const float2*)(x0 + 8 * (s + k)), v = *(const float2*)(x1 + 8 * (s + k));
      PartsA a;
      tf32_parts(u.x, a.hi[0], a.lo[0]);
      tf32_parts(v.x, a.hi[1], a.lo[1]);
      tf32_parts(u.y, a.hi[2], a.lo[2]);
      tf32_parts(v.y, a.hi[3], a.lo[3]);
      float w[kOtherTiles][2];
#pragma unroll
      for (int n = 0; n < kOtherTiles; ++n) {
        const float2 z = *(const float2*)(y0 + 8 * n * ld + 8 * (s + k));
        w[n][0] = z.x;
        w[n][1] = z.y;
      }
      mma_parts(part, a, w);
    }
#pragma unroll
    for (int n = 0; n < kOtherTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] += part[n][i];
  }
}
// acc[e] += p (rows of y), elements 8 e .. of y's rows: the columns 2 t and 2 t + 1 that a lane has of each eight are k index t and t + 4
template <int DT>
__device__ __forceinline__ void single_add(float (&acc)[DT][4], const float (&p)[kOtherTiles][4], const float* y, int ld, int steps) {
  const int g = ((int)threadIdx.x & 31) >> 2, t = (int)threadIdx.x & 3;
#pragma unroll
  for (int n = 0; n < kOtherTiles; n += 2) {
    PartsA a[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      tf32_parts(p[n + k][0], a[k].hi[0], a[k].lo[0]);
      tf32_parts(p[n + k][2], a[k].hi[1], a[k].lo[1]);
      tf32_parts(p[n + k][1], a[k].hi[2], a[k].lo[2]);
      tf32_parts(p[n + k][3], a[k].hi[3], a[k].lo[3]);
    }
    const float* y0 = y + (8 * n + 2 * t) * ld + g;
    constexpr int N = 4;
#pragma unroll
    for (int e = 0; e < DT; e += N) {
      if (e >= steps) continue;          // (of the last N some may be zeros)
      float part[N][4];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) part[i][c] = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float w[N][2];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool in = e + i < steps;
          w[i][0] = in ? y0[8 * k * ld + 8 * (e + i)] : 0.f;
          w[i][1] = in ? y0[(8 * k + 1) * ld + 8 * (e + i)] : 0.f;
        }
        mma_parts(part, a[k], w);
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[e + i][c] += part[i][c];
    }
  }
}
// One of a lane's two rows of the result; false (in all lanes of the row) where a value is infinite or undefined
template <int DT>
__device__ __forceinline__ bool single_store(const float (&v)[DT][4], int second, float by, void* to, long long at, int d) {
  const int t = (int)threadIdx.x & 3;
  bool fine = true;
#pragma unroll
  for (int e = 0; e < DT; ++e)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = 8 * e + 2 * t + i;
      const float y = by == 0.f ? 0.f : v[e][2 * second + i] * by;
      if (c < d) {
        ((float*)to)[at + c] = y;
        fine = fine && y * 0.f == 0.f;
      }
    }
  return fine;
}
// lanes 4 g .. 4 g + 3 have rows g and g + 8: the rows, a bit each, of which some lane says no.  What the lanes have written of them lies
// behind (a vote alone orders no memory): the rows are written again by other lanes.
__device__ __forceinline__ unsigned int rows_not(bool fine) {
  unsigned int b = __ballot_sync(0xffffffffu, !fine), rows = 0u;
  __syncwarp();
#pragma unroll
  for (int g = 0; g < 8; ++g) rows |= (b >> (4 * g) & 15u ? 1u : 0u) << g;
  return rows;
}

// What describes the other rows of a step: keys' documents, or the queries
struct SingleOthers {
  int last[kOthers * kMostShares], doc[kOthers * kMostShares], pos[kOthers * kMostShares];
  float lse[kOthers * kMostShares], delta[kOthers * kMostShares];
};

// The warps' part in the block: which 16 of its rows, which of the steps
struct SingleWarp {
  int group, groups, share, shares;
  __device__ __forceinline__ explicit SingleWarp(int n) {
    groups = n;
    shares = (int)(blockDim.x >> 5) / n;
    group = (int)(threadIdx.x >> 5) % n;
    share = (int)(threadIdx.x >> 5) / n;
  }
  // where a lane's i-th value goes when the shares meet
  __device__ __forceinline__ float* slot(float* at, int which, int values, int i) const { return at + (((which - 1) * groups + group) * values + i) * 32 + (threadIdx.x & 31u); }
};

// own rows as queries
struct SingleOwn {
  AttnRow row[2];
  int end;                  // behind the last key that a row of the warp sees
  __device__ __forceinline__ void fetch(const AttnArgs& a, int b, int first) {
    const int g = ((int)threadIdx.x & 31) >> 2;
    end = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = first + g + 8 * i;
      row[i].pos = 0; row[i].last = -1; row[i].doc = -1;
      if (r < a.S) row[i] = attn_row(a, b, r);
      end = max(end, row[i].last + 1);
    }
    end = __reduce_max_sync(0xffffffffu, end);
  }
};

template <int DT>
__global__ void __launch_bounds__(256, DT == 8 ? 2 : 1) attn_forward_single(const __grid_constant__ AttnArgs a, int vec, int places, int groups) {
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ int block_end;
  grid_begin();
  const SingleWarp me(groups);
  const int lane = (int)threadIdx.x & 31, g = lane >> 2, t = lane & 3, span = kOthers * me.shares;       // (rows of the others a round)
  const int ld = SingleShape::ld(a.D), steps = (a.D + 7) / 8, tile = span * ld, mine = me.share * kOthers;
  float *q = (float*)dyn, *k = q + 16 * groups * ld;
  SingleOthers* o_ = (SingleOthers*)(k + places * 2 * tile);
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.H;
  const int tiles_q = (a.S + 16 * groups - 1) / (16 * groups), r0 = (tiles_q - 1 - (int)(blockIdx.x / heads)) * 16 * groups;
  const int b = (int)(blockIdx.x % heads) / a.H, h = (int)(blockIdx.x % heads) % a.H, hk = h / a.group;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  if (threadIdx.x == 0) block_end = 0;
  single_load(q, 16 * groups, a.q, attn_q_at(a, b, 0, h), (long long)a.H * a.ld, r0, a.S, a.D, ld, vec);
  SingleOwn own;
  own.fetch(a, b, r0 + 16 * me.group);
  __syncthreads();
  if (lane == 0) atomicMax(&block_end, own.end);
  __syncthreads();
  const int end = block_end;
  const long long k_at = attn_k_at(a, b, 0, hk), k_step = (long long)a.HK * a.ld;
  auto load = [&](int j0, int n) {
    float* to = k + (n & (places - 1)) * 2 * tile;
    single_load(to, span, a.k, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_load(to + tile, span, a.v, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_sent();
  };
  float o[DT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int e = 0; e < DT; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[e][i] = 0.f;
  if (places == 2 && end > 0) load(0, 0);
  for (int j0 = 0, n = 0; j0 < end; j0 += span, ++n) {
    __syncthreads();
    const bool more = places == 2 && j0 + span < end;
    if (places == 1) load(j0, n);
    else if (more) load(j0 + span, n + 1);
    if (a.kdoc && (int)threadIdx.x < span) o_->doc[threadIdx.x] = j0 + (int)threadIdx.x < a.T ? a.kdoc[(long long)b * a.T + j0 + threadIdx.x] : -1;
    single_arrived(more);
    __syncthreads();
    // a warp whose rows see nothing of the step leaves it out
    if (j0 + mine >= own.end) continue;
    const float *kt = k + (n & (places - 1)) * 2 * tile + mine * ld, *vt = kt + tile;
    float x[kOtherTiles][4], th, top[2] = {-INFINITY, -INFINITY};
    single_dots(x, q + 16 * me.group * ld, kt, ld, steps);
#pragma unroll
    for (int c = 0; c < kOtherTiles; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const AttnRow& w = own.row[i >> 1];
        const int at = mine + 8 * c + 2 * t + (i & 1), j = j0 + at;
        const bool on = j <= w.last && (!a.kdoc || o_->doc[at] == w.doc);
        x[c][i] = on ? attn_score(a, x[c][i], slope2, w.pos, j, th) : -INFINITY;
        top[i >> 1] = fmaxf(top[i >> 1], x[c][i]);
      }
    float by[2], off[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 1));
      top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 2));
      const float next = fmaxf(m[w], top[w]);
      by[w] = m[w] == next ? 1.f : m[w] == -INFINITY ? 0.f : exp2f(m[w] - next);
      m[w] = next;
      off[w] = next == -INFINITY ? 0.f : next;
      l[w] *= by[w];
    }
    if (__any_sync(0xffffffffu, by[0] != 1.f || by[1] != 1.f)) {
#pragma unroll
      for (int e = 0; e < DT; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[e][i] *= by[i >> 1];
    }
#pragma unroll
    for (int c = 0; c < kOtherTiles; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[c][i] = exp2f(x[c][i] - off[i >> 1]);
        l[i >> 1] += x[c][i];
      }
    single_add<DT>(o, x, vt, ld, steps);
  }
  single_sent();
  single_arrived(false);
  __syncthreads();
  constexpr int kValues = DT * 4 + 4;
  if (me.share) {
#pragma unroll
    for (int e = 0; e < DT; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) *me.slot(k, me.share, kValues, 4 * e + i) = o[e][i];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      *me.slot(k, me.share, kValues, DT * 4 + w) = m[w];
      *me.slot(k, me.share, kValues, DT * 4 + 2 + w) = l[w];
    }
  }
  __syncthreads();
  if (me.share) return;
  for (int other = 1; other < me.shares; ++other) {
    float c[2], d[2];          // what the sums so far and the other's are multiplied by
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float theirs = *me.slot(k, other, kValues, DT * 4 + w), next = fmaxf(m[w], theirs);
      c[w] = m[w] == next ? 1.f : m[w] == -INFINITY ? 0.f : exp2f(m[w] - next);
      d[w] = theirs == next ? 1.f : theirs == -INFINITY ? 0.f : exp2f(theirs - next);
      l[w] = l[w] * c[w] + *me.slot(k, other, kValues, DT * 4 + 2 + w) * d[w];
      m[w] = next;
    }
#pragma unroll
    for (int e = 0; e < DT; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[e][i] = o[e][i] * c[i >> 1] + *me.slot(k, other, kValues, 4 * e + i) * d[i >> 1];
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
    const int r = r0 + 16 * me.group + g + 8 * w;
    bool fine = true;
    if (r < a.S) {
      const bool on = l[w] > 0.f || l[w] != l[w];
      fine = single_store<DT>(o, w, on ? 1.f / l[w] : 0.f, a.out, attn_q_at(a, b, r, h), a.D);
      if (t == 0 && a.lse) a.lse[((long long)b * a.H + h) * a.S + r] = on ? (m[w] + log2f(l[w])) * kLn2 : -INFINITY;
    }
    for (unsigned int todo = rows_not(fine); todo; todo &= todo - 1) attn_forward_row<float>(a, b, h, r0 + 16 * me.group + 8 * w + __ffs(todo) - 1, lane);
  }
}

// The sums of the warps that share their rows, added in order by the first; false in the others, which are done.
template <int DT>
__device__ __forceinline__ bool single_meet(const SingleWarp& me, float* at, float (&x)[DT][4], float (*y)[4]) {
  const int values = (y ? 2 : 1) * DT * 4;
  __syncthreads();
  if (me.share) {
#pragma unroll
    for (int e = 0; e < DT; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *me.slot(at, me.share, values, 4 * e + i) = x[e][i];
        if (y) *me.slot(at, me.share, values, DT * 4 + 4 * e + i) = y[e][i];
      }
  }
  __syncthreads();
  if (me.share) return false;
  for (int other = 1; other < me.shares; ++other)
#pragma unroll
    for (int e = 0; e < DT; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[e][i] += *me.slot(at, other, values, 4 * e + i);
        if (y) y[e][i] += *me.slot(at, other, values, DT * 4 + 4 * e + i);
      }
  return true;
}

// ------------------------------------------------------------------ gradients: of the queries ...
template <int DT>
__device__ __forceinline__ void single_grad_queries(const AttnArgs& a, int vec, int places, int groups, unsigned int block, unsigned char* dyn, int* block_end) {
  const SingleWarp me(groups);
  const int lane = (int)threadIdx.x & 31, g = lane >> 2, t = lane & 3, span = kOthers * me.shares;       // (rows of the others a round)
  const int ld = SingleShape::ld(a.D), steps = (a.D + 7) / 8, tile = span * ld, mine = me.share * kOthers;
  float *q = (float*)dyn, *go = q + 16 * groups * ld, *k = go + 16 * groups * ld;
  SingleOthers* o_ = (SingleOthers*)(k + places * 2 * tile);
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.H;
  const int tiles_q = (a.S + 16 * groups - 1) / (16 * groups), r0 = (tiles_q - 1 - (int)(block / heads)) * 16 * groups;
  const int b = (int)(block % heads) / a.H, h = (int)(block % heads) % a.H, hk = h / a.group;
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  if (threadIdx.x == 0) *block_end = 0;
  const long long q_at = attn_q_at(a, b, 0, h), q_step = (long long)a.H * a.ld;
  single_load(q, 16 * groups, a.q, q_at, q_step, r0, a.S, a.D, ld, vec);
  single_load(go, 16 * groups, a.d_out, q_at, q_step, r0, a.S, a.D, ld, vec);
  SingleOwn own;
  own.fetch(a, b, r0 + 16 * me.group);
  float lse[2], delta[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int r = r0 + 16 * me.group + g + 8 * w;
    lse[w] = INFINITY;
    delta[w] = 0.f;
    if (r < a.S) {
      lse[w] = a.stat[attn_stat_at(a, b, h, r)];
      delta[w] = a.stat[attn_stat_at(a, b, h, r) + 128];
    }
  }
  __syncthreads();
  if (lane == 0) atomicMax(block_end, own.end);
  __syncthreads();
  const int end = *block_end;
  const long long k_at = attn_k_at(a, b, 0, hk), k_step = (long long)a.HK * a.ld;
  auto load = [&](int j0, int n) {
    float* to = k + (n & (places - 1)) * 2 * tile;
    single_load(to, span, a.k, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_load(to + tile, span, a.v, k_at, k_step, j0, a.T, a.D, ld, vec);
    single_sent();
  };
  float acc[DT][4];
#pragma unroll
  for (int e = 0; e < DT; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[e][i] = 0.f;
  if (places == 2 && end > 0) load(0, 0);
  for (int j0 = 0, n = 0; j0 < end; j0 += span, ++n) {
    __syncthreads();
    const bool more = places == 2 && j0 + span < end;
    if (places == 1) load(j0, n);
    else if (more) load(j0 + span, n + 1);
    if (a.kdoc && (int)threadIdx.x < span) o_->doc[threadIdx.x] = j0 + (int)threadIdx.x < a.T ? a.kdoc[(long long)b * a.T + j0 + threadIdx.x] : -1;
    single_arrived(more);
    __syncthreads();
    if (j0 + mine >= own.end) continue;
    const float *kt = k + (n & (places - 1)) * 2 * tile + mine * ld, *vt = kt + tile;
    float x[kOtherTiles][4], y[kOtherTiles][4], p, dx;
    single_dots(x, q + 16 * me.group * ld, kt, ld, steps);
    single_dots(y, go + 16 * me.group * ld, vt, ld, steps);
#pragma unroll
    for (int c = 0; c < kOtherTiles; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const AttnRow& w = own.row[i >> 1];
        const int at = mine + 8 * c + 2 * t + (i & 1), j = j0 + at;
        const bool on = j <= w.last && (!a.kdoc || o_->doc[at] == w.doc);
        attn_pair(a, x[c][i], y[c][i], slope, w.pos, j, lse[i >> 1], delta[i >> 1], p, dx);
        x[c][i] = on ? dx : 0.f;
      }
    single_add<DT>(acc, x, kt, ld, steps);
  }
  single_sent();
  single_arrived(false);
  if (!single_meet<DT>(me, k, acc, nullptr)) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int r = r0 + 16 * me.group + g + 8 * w;
    const bool fine = r >= a.S || single_store<DT>(acc, w, 1.f, a.dq, attn_q_at(a, b, r, h), a.D);
    for (unsigned int todo = rows_not(fine); todo; todo &= todo - 1) attn_dq_row<float>(a, b, h, r0 + 16 * me.group + 8 * w + __ffs(todo) - 1, lane);
  }
}

// ... and of the keys
template <int DT>
__device__ __forceinline__ void single_grad_keys(const AttnArgs& a, int vec, int places, int groups, unsigned int block, unsigned char* dyn) {
  const SingleWarp me(groups);
  const int lane = (int)threadIdx.x & 31, g = lane >> 2, t = lane & 3, span = kOthers * me.shares;       // (rows of the others a round)
  const int ld = SingleShape::ld(a.D), steps = (a.D + 7) / 8, tile = span * ld, mine = me.share * kOthers;
  float *k = (float*)dyn, *v = k + 16 * groups * ld, *q = v + 16 * groups * ld;
  SingleOthers* o_ = (SingleOthers*)(q + places * 2 * tile);
  const unsigned int heads = (unsigned int)a.B * (unsigned int)a.HK;
  const int j0 = (int)(block / heads) * 16 * groups;
  const int b = (int)(block % heads) / a.HK, hk = (int)(block % heads) % a.HK;
  const long long k_at = attn_k_at(a, b, 0, hk), k_step = (long long)a.HK * a.ld;
  single_load(k, 16 * groups, a.k, k_at, k_step, j0, a.T, a.D, ld, vec);
  single_load(v, 16 * groups, a.v, k_at, k_step, j0, a.T, a.D, ld, vec);
  single_sent();
  const AttnSeq seq = attn_seq(a, b);
  const int key[2] = {j0 + 16 * me.group + g, j0 + 16 * me.group + g + 8};
  int doc[2] = {0, 0};
  if (a.kdoc)
#pragma unroll
    for (int w = 0; w < 2; ++w) doc[w] = key[w] < a.T ? a.kdoc[(long long)b * a.T + key[w]] : -1;
  // the first step of queries that see a key of the block's (later ones see no fewer)
  int begin = 0;
  if (a.mask != B200_MASK_NONE) {
    // (position >= j0, or a prefix that reaches a key)
    begin = j0 < seq.prefix ? 0 : max(0, j0 - (seq.len - a.S)) / span * span;
  }
  if (j0 >= seq.len) begin = a.S;
  auto load = [&](int h, int r0, int n) {
    float* to = q + (n & (places - 1)) * 2 * tile;
    const long long at = attn_q_at(a, b, 0, h), step = (long long)a.H * a.ld;
    single_load(to, span, a.q, at, step, r0, a.S, a.D, ld, vec);
    single_load(to + tile, span, a.d_out, at, step, r0, a.S, a.D, ld, vec);
    single_sent();
  };
  const int last_head = (hk + 1) * a.group - 1;
  float gk[DT][4], gv[DT][4];
#pragma unroll
  for (int e = 0; e < DT; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) gk[e][i] = gv[e][i] = 0.f;
  // a thread's query of the next step, fetched ahead
  int next_last = -1, next_doc = -1;
  float next_lse = INFINITY, next_delta = 0.f;
  auto fetch = [&](int h, int r0) {
    const int r = r0 + (int)threadIdx.x;
    next_last = next_doc = -1;
    if ((int)threadIdx.x < span && r < a.S) {
      next_last = attn_last(a, seq, r);
      next_doc = a.kdoc ? AttnQueryDocs(a, seq, b).of(r) : 0;
      if (next_doc < 0) next_last = -1;
      next_lse = a.stat[attn_stat_at(a, b, h, r)];
      next_delta = a.stat[attn_stat_at(a, b, h, r) + 128];
    }
  };
  if (begin < a.S) {
    fetch(hk * a.group, begin);
    if (places == 2) load(hk * a.group, begin, 0);
  }
  int n = 0;
  for (int h = hk * a.group; h <= last_head; ++h) {
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    for (int r0 = begin; r0 < a.S; r0 += span, ++n) {
      __syncthreads();
      const bool more = r0 + span < a.S || h < last_head;
      const int next_h = r0 + span < a.S ? h : h + 1, next_r = r0 + span < a.S ? r0 + span : begin;
      if (places == 1) load(h, r0, n);
      else if (more) load(next_h, next_r, n + 1);
      if ((int)threadIdx.x < span) {
        o_->last[threadIdx.x] = next_last;
        o_->doc[threadIdx.x] = next_doc;
        o_->pos[threadIdx.x] = seq.len - a.S + r0 + (int)threadIdx.x;
        o_->lse[threadIdx.x] = next_lse;
        o_->delta[threadIdx.x] = next_delta;
      }
      if (more) fetch(next_h, next_r);
      single_arrived(places == 2 && more);
      __syncthreads();
      // a step without a visible pair for the warp is left out
      bool any = false;
#pragma unroll
      for (int c = 0; c < kOtherTiles; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = mine + 8 * c + 2 * t + (i & 1);
          any |= key[i >> 1] <= o_->last[at] && (!a.kdoc || o_->doc[at] == doc[i >> 1]);
        }
      if (!__any_sync(0xffffffffu, any)) continue;
      const float *qt = q + (n & (places - 1)) * 2 * tile + mine * ld, *gt = qt + tile;
      float x[kOtherTiles][4], y[kOtherTiles][4], p, dx;
      single_dots(x, k + 16 * me.group * ld, qt, ld, steps);
      single_dots(y, v + 16 * me.group * ld, gt, ld, steps);
#pragma unroll
      for (int c = 0; c < kOtherTiles; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = mine + 8 * c + 2 * t + (i & 1);
          const bool on = key[i >> 1] <= o_->last[at] && (!a.kdoc || o_->doc[at] == doc[i >> 1]);
          attn_pair(a, x[c][i], y[c][i], slope, o_->pos[at], key[i >> 1], o_->lse[at], o_->delta[at], p, dx);
          x[c][i] = on ? p : 0.f;
          y[c][i] = on ? dx : 0.f;
        }
      single_add<DT>(gv, x, gt, ld, steps);
      single_add<DT>(gk, y, qt, ld, steps);
    }
  }
  single_arrived(false);
  if (!single_meet<DT>(me, q, gk, gv)) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const bool in = key[w] < a.T;
    const long long at = attn_k_at(a, b, key[w], hk);
    const bool fine_k = !in || single_store<DT>(gk, w, 1.f, a.dk, at, a.D), fine_v = !in || single_store<DT>(gv, w, 1.f, a.dv, at, a.D);
    const unsigned int not_k = rows_not(fine_k), not_v = rows_not(fine_v);
    for (unsigned int todo = not_k | not_v; todo; todo &= todo - 1) {
      const int i = __ffs(todo) - 1;
      attn_dkv_row<float>(a, b, hk, j0 + 16 * me.group + 8 * w + i, lane, (int)(not_k >> i & 1u) | (int)(not_v >> i & 1u) << 1);
    }
  }
}

// both in one launch: the keys' blocks first, theirs are the longer walks
template <int DT>
__global__ void __launch_bounds__(256) attn_grad_single(const __grid_constant__ AttnArgs a, int vec, int places, int groups, unsigned int keys_grid) {
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ int block_end;
  grid_begin();
  if (blockIdx.x < keys_grid) single_grad_keys<DT>(a, vec, places, groups, blockIdx.x, dyn);
  else single_grad_queries<DT>(a, vec, places, groups, blockIdx.x - keys_grid, dyn, &block_end);
}

}  // namespace b200
#endif
