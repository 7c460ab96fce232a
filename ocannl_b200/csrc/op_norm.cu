// Layer norm of the rows of a [rows, n] node, and its gradients.
//
//   forward    h = x + r;  mean = sum(h) / n;  rstd = 1 / sqrt(sum((h - mean)^2) / n + eps)
//              y = (h - mean) * rstd * gamma + beta
//   gradients  u = (h - mean) * rstd;  g = dy * gamma
//              dx = rstd * (g - sum(g) / n - u * sum(g * u) / n) (+ dh);  dgamma = sum_rows(dy * u);  dbeta = sum_rows(dy)
//
// Both move every plane of the rows once.  A group of 8, 32, 128, 512 or (forward) 1024 threads keeps its row in
// registers, at most 16 elements a thread, so that the squares of the distances from the mean are summed in a second pass over
// registers (no difference of large sums).  The groups stride over the rows, the next row's loads under way while one is worked
// on; the scale and the shift stay in shared memory.  In the gradient a thread keeps its sums over the rows of its columns in
// registers; they meet in shared memory once per block and then in a second kernel that adds the blocks' partial sums in their order: the
// same bits every time.  Sums of a thread's own rows are in single precision, those over threads and blocks in double.
// Longer rows (of more than 8192 elements; forward and on 16 bytes, of more than 16384) are read again for each pass, by 1024 threads (they come
// from L2 then), their column sums kept in shared memory.
#include "kernels/op_common.cuh"
#include "operators.hpp"

using namespace b200;

namespace {

struct NormArgs {
  const void *x, *r, *gamma, *beta, *dy, *dh;
  void *y, *h, *dx;
  float *mean, *rstd;              // written by the forward pass, read by the gradient
  float *partial;                  // gradient: [2][blocks][n]
  unsigned long long rows;
  unsigned int n;
  int own_columns;                 // wide gradient: the column sums are made along with dx
  int weight_f32;                  // gamma and beta in single precision, or in the rows' type
  float eps, inv_n;
};

template <class T>
__device__ __forceinline__ float weight_at(const void* p, int f32, unsigned int i, float otherwise) {
  if (!p) return otherwise;
  return f32 ? ((const float*)p)[i] : to_float(((const T*)p)[i]);
}

// Sums of K values over the TPR threads of a row.  `sh`: [2][K][threads / 32], the halves used in turn, so that one barrier a
// sum is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* sh, int half) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TPR > 32) {
    const unsigned int warps = blockDim.x / 32, warp = threadIdx.x / 32, first = threadIdx.x / TPR * (TPR / 32);
    float* s = sh + half * K * 32;
    if ((threadIdx.x & 31u) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k * 32 + warp] = v[k];
    __syncthreads();
    (void)warps;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 32; ++w) t += s[k * 32 + first + w];
      v[k] = t;
    }
  }
}

template <class T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256, TPR > 256 ? 1 : 3) norm_rows(const NormArgs a) {
  constexpr int E = NV * VEC;
  __shared__ float sh[2 * 32];
  extern __shared__ __align__(16) float weights[];      // scale and shift
  grid_begin();
  const unsigned int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, per_block = blockDim.x / TPR;
  constexpr unsigned int kSpan = TPR * E;
  for (unsigned int e = threadIdx.x; e < kSpan; e += blockDim.x) {
    weights[e] = e < a.n ? weight_at<T>(a.gamma, a.weight_f32, e, 1.f) : 0.f;
    weights[kSpan + e] = e < a.n ? weight_at<T>(a.beta, a.weight_f32, e, 0.f) : 0.f;
  }
  // the next row is on its way while this one is worked on
  Raw<T, VEC> rx[NV], rr[NV];
  const unsigned long long step = (unsigned long long)gridDim.x * per_block;
  auto fetch = [&](unsigned long long row) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const unsigned int e = (c * TPR + t) * VEC;
      if (row < a.rows && e < a.n) {
        rx[c].load((const T*)a.x + row * a.n + e);
        if (a.r) rr[c].load((const T*)a.r + row * a.n + e);
      }
    }
  };
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    rx[c].clear();
    rr[c].clear();
  }
  fetch((unsigned long long)blockIdx.x * per_block + sub);
  __syncthreads();
  for (unsigned long long first = (unsigned long long)blockIdx.x * per_block; first < a.rows; first += step) {
    const unsigned long long row = first + sub;
    const bool on = row < a.rows;
    const unsigned long long at = row * a.n;
    float h[E];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float w[VEC];
      rx[c].values(h + c * VEC);
      rr[c].values(w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[c * VEC + i] += w[i];
    }
    fetch(row + step);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) s[0] += h[i];
    row_sum<TPR>(s, sh, 0);
    const float mean = s[0] * a.inv_n;
    float q[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = (c * TPR + t) * VEC + i < a.n ? h[c * VEC + i] - mean : 0.f;
        q[0] = fmaf(d, d, q[0]);
      }
    row_sum<TPR>(q, sh, 1);
    const float rstd = 1.f / sqrtf(fmaf(q[0], a.inv_n, a.eps));
    if (!on) continue;
    if (t == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const unsigned int e = (c * TPR + t) * VEC;
      if (e >= a.n) continue;
      float v[VEC];
      if (a.h) Vec<T, VEC>::store((T*)a.h + at + e, h + c * VEC);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = fmaf((h[c * VEC + i] - mean) * rstd, weights[e + i], weights[kSpan + e + i]);
      Vec<T, VEC>::store((T*)a.y + at + e, v);
    }
  }
}

template <class T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(512, 1) norm_grad_rows(const NormArgs a) {
  constexpr int E = NV * VEC;
  __shared__ float sh[2 * 2 * 32];
  extern __shared__ __align__(16) float weights[];      // the scale; at the end [2][rows of the block at a time][n] sums
  float* columns = weights;
  grid_begin();
  const unsigned int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, per_block = blockDim.x / TPR;
  constexpr unsigned int kSpan = TPR * E;
  for (unsigned int e = threadIdx.x; e < kSpan; e += blockDim.x) weights[e] = e < a.n ? weight_at<T>(a.gamma, a.weight_f32, e, 1.f) : 0.f;
  [[maybe_unused]] float dg[E], db[E];
  [[maybe_unused]] Pair dg2[E / 2 + 1], db2[E / 2 + 1];
#pragma unroll
  for (int i = 0; i < E; ++i) dg[i] = db[i] = 0.f;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) dg2[i] = db2[i] = Pair(0.f, 0.f);
  // the next row is on its way while this one is worked on; a row's values are taken from its bits twice, before and after the sums
  struct Row {
    Raw<T, VEC> x[NV], dy[NV], dh[NV];
    float mean, rstd;
  } next, now;
  const unsigned long long step = (unsigned long long)gridDim.x * per_block;
  auto fetch = [&](unsigned long long row) {
    const bool on = row < a.rows;
    next.mean = on ? a.mean[row] : 0.f;
    next.rstd = on ? a.rstd[row] : 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const unsigned int e = (c * TPR + t) * VEC;
      next.x[c].clear();
      next.dy[c].clear();
      next.dh[c].clear();
      if (on && e < a.n) {
        next.x[c].load((const T*)a.x + row * a.n + e);
        next.dy[c].load((const T*)a.dy + row * a.n + e);
        if (a.dh) next.dh[c].load((const T*)a.dh + row * a.n + e);
      }
    }
  };
  int half = 0;
  fetch((unsigned long long)blockIdx.x * per_block + sub);
  __syncthreads();
  for (unsigned long long first = (unsigned long long)blockIdx.x * per_block; first < a.rows; first += step) {
    const unsigned long long row = first + sub;
    const bool on = row < a.rows;
    now = next;
    fetch(row + step);
    float s[2] = {0.f, 0.f};
    // (behind the row's end dy and gamma are zero)
    if constexpr (VEC == 1) {
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float u, dy;
        now.x[c].values(&u);
        now.dy[c].values(&dy);
        u = (u - now.mean) * now.rstd;
        const float g = dy * weights[c * TPR + t];
        s[0] += g;
        s[1] = fmaf(g, u, s[1]);
        dg[c] = fmaf(dy, u, dg[c]);
        db[c] += dy;
      }
    } else {
      // two elements to an instruction (16384 x 512 bf16: 19.4 us, 20.7 with one; what bounds it is latency, with 16 warps an SM and a row
      // of each under way, 41 % of the issue slots are used)
      const Pair shift(-now.mean, -now.mean), rstd2(now.rstd, now.rstd);
      Pair s0(0.f, 0.f), s1(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float x[VEC], dy[VEC];
        now.x[c].values(x);
        now.dy[c].values(dy);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const int k = (c * VEC + i) / 2;
          const float2 w = *(const float2*)(weights + (c * TPR + t) * VEC + i);
          const Pair d(dy[i], dy[i + 1]), u = mul2(add2(Pair(x[i], x[i + 1]), shift), rstd2), g = mul2(d, Pair(w.x, w.y));
          s0 = add2(s0, g);
          s1 = fma2(g, u, s1);
          dg2[k] = fma2(d, u, dg2[k]);
          db2[k] = add2(db2[k], d);
        }
      }
      float even, odd;
      s0.get(even, odd);
      s[0] = even + odd;
      s1.get(even, odd);
      s[1] = even + odd;
    }
    row_sum<TPR>(s, sh, half);
    half ^= 1;
    if (!on) continue;
    const float m0 = s[0] * a.inv_n, m1 = s[1] * a.inv_n;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const unsigned int e = (c * TPR + t) * VEC;
      if (e >= a.n) continue;
      float v[VEC], dy[VEC], w[VEC];
      now.x[c].values(v);
      now.dy[c].values(dy);
      now.dh[c].values(w);
      if constexpr (VEC == 1) {
        v[0] = fmaf(now.rstd, dy[0] * weights[e] - m0 - (v[0] - now.mean) * now.rstd * m1, w[0]);
      } else {
        const Pair shift(-now.mean, -now.mean), rstd2(now.rstd, now.rstd), less0(-m0, -m0), less1(-m1, -m1);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const float2 ga = *(const float2*)(weights + e + i);
          const Pair u = mul2(add2(Pair(v[i], v[i + 1]), shift), rstd2), g = fma2(Pair(dy[i], dy[i + 1]), Pair(ga.x, ga.y), less0);
          fma2(rstd2, fma2(u, less1, g), Pair(w[i], w[i + 1])).get(v[i], v[i + 1]);
        }
      }
      Vec<T, VEC>::store((T*)a.dx + row * a.n + e, v);
    }
  }
  if (!a.partial) return;
  if constexpr (VEC > 1) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      dg2[i].get(dg[2 * i], dg[2 * i + 1]);
      db2[i].get(db[2 * i], db[2 * i + 1]);
    }
  }
  // the block's groups of threads meet: columns[which][group][column]
  const unsigned int plane = per_block * a.n;
  if (per_block > 1) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const unsigned int e = (c * TPR + t) * VEC + i;
        if (e >= a.n) continue;
        columns[sub * a.n + e] = dg[c * VEC + i];
        columns[plane + sub * a.n + e] = db[c * VEC + i];
      }
    __syncthreads();
    for (unsigned int e = threadIdx.x; e < 2 * a.n; e += blockDim.x) {
      const unsigned int which = e >= a.n, col = e - which * a.n;
      double v = 0.;
      for (unsigned int g = 0; g < per_block; ++g) v += (double)columns[which * plane + g * a.n + col];
      a.partial[((unsigned long long)which * gridDim.x + blockIdx.x) * a.n + col] = (float)v;
    }
  } else {
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const unsigned int e = (c * TPR + t) * VEC + i;
        if (e >= a.n) continue;
        a.partial[(unsigned long long)blockIdx.x * a.n + e] = dg[c * VEC + i];
        a.partial[((unsigned long long)gridDim.x + blockIdx.x) * a.n + e] = db[c * VEC + i];
      }
  }
}

// ---- rows that do not fit the registers: a block of 1024 threads each, read again for every pass
template <class T, int VEC>
__global__ void __launch_bounds__(1024) norm_wide(const NormArgs a) {
  __shared__ float sh[2 * 32];
  grid_begin();
  for (unsigned long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = (const T*)a.x + row * a.n, *r = a.r ? (const T*)a.r + row * a.n : nullptr;
    auto load = [&](unsigned int e, float* v) {
      Vec<T, VEC>::load(x + e, v);
      if (r) {
        float w[VEC];
        Vec<T, VEC>::load(r + e, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += w[i];
      }
    };
    float s[1] = {0.f}, q[1] = {0.f};
    for (unsigned int e = threadIdx.x * VEC; e < a.n; e += 1024 * VEC) {
      float v[VEC];
      load(e, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[0] += v[i];
    }
    row_sum<1024>(s, sh, 0);
    const float mean = s[0] * a.inv_n;
    for (unsigned int e = threadIdx.x * VEC; e < a.n; e += 1024 * VEC) {
      float v[VEC];
      load(e, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) q[0] = fmaf(v[i] - mean, v[i] - mean, q[0]);
    }
    row_sum<1024>(q, sh, 1);
    const float rstd = 1.f / sqrtf(fmaf(q[0], a.inv_n, a.eps));
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    for (unsigned int e = threadIdx.x * VEC; e < a.n; e += 1024 * VEC) {
      float v[VEC];
      load(e, v);
      if (a.h) Vec<T, VEC>::store((T*)a.h + row * a.n + e, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        v[i] = fmaf((v[i] - mean) * rstd, weight_at<T>(a.gamma, a.weight_f32, e + i, 1.f), weight_at<T>(a.beta, a.weight_f32, e + i, 0.f));
      Vec<T, VEC>::store((T*)a.y + row * a.n + e, v);
    }
  }
}

// `own_columns`: the block's column sums lie in shared memory, where a thread adds to those of its elements alone
template <class T, int VEC>
__global__ void __launch_bounds__(1024) norm_grad_wide(const NormArgs a) {
  __shared__ float sh[2 * 2 * 32];
  extern __shared__ __align__(16) float columns[];
  grid_begin();
  if (a.own_columns)
    for (unsigned int e = threadIdx.x * VEC; e < a.n; e += 1024 * VEC)
#pragma unroll
      for (int i = 0; i < VEC; ++i) columns[e + i] = columns[a.n + e + i] = 0.f;
  int half = 0;
  for (unsigned long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const unsigned long long at = row * a.n;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (unsigned int e = threadIdx.x * VEC; e < a.n; e += 1024 * VEC) {
      float v[VEC], w[VEC];
      Vec<T, VEC>::load((const T*)a.x + at + e, v);
      Vec<T, VEC>::load((const T*)a.dy + at + e, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float g = w[i] * weight_at<T>(a.gamma, a.weight_f32, e + i, 1.f);
        s[0] += g;
        s[1] = fmaf(g, (v[i] - mean) * rstd, s[1]);
      }
    }
    row_sum<1024>(s, sh, half);
    half ^= 1;
    const float m0 = s[0] * a.inv_n, m1 = s[1] * a.inv_n;
    for (unsigned int e = threadIdx.x * VEC; e < a.n; e += 1024 * VEC) {
      float v[VEC], w[VEC], d[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[i] = 0.f;
      Vec<T, VEC>::load((const T*)a.x + at + e, v);
      Vec<T, VEC>::load((const T*)a.dy + at + e, w);
      if (a.dh) Vec<T, VEC>::load((const T*)a.dh + at + e, d);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float g = w[i] * weight_at<T>(a.gamma, a.weight_f32, e + i, 1.f), u = (v[i] - mean) * rstd;
        if (a.own_columns) {
          columns[e + i] = fmaf(w[i], u, columns[e + i]);
          columns[a.n + e + i] += w[i];
        }
        v[i] = fmaf(rstd, g - m0 - u * m1, d[i]);
      }
      Vec<T, VEC>::store((T*)a.dx + at + e, v);
    }
  }
  if (a.own_columns && a.partial)
    for (unsigned int e = threadIdx.x * VEC; e < a.n; e += 1024 * VEC)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        a.partial[(unsigned long long)blockIdx.x * a.n + e + i] = columns[e + i];
        a.partial[((unsigned long long)gridDim.x + blockIdx.x) * a.n + e + i] = columns[a.n + e + i];
      }
}

// column sums of wide rows: a thread per column, a slice of the rows per block, which may be long: in double; partial sums as above
template <class T>
__global__ void __launch_bounds__(256) norm_grad_columns(const NormArgs a, unsigned int slices) {
  grid_begin();
  const unsigned int col = blockIdx.x * 256 + threadIdx.x, slice = blockIdx.y;
  if (col >= a.n) return;
  const unsigned long long first = a.rows * slice / slices, last = a.rows * (slice + 1) / slices;
  double dg = 0., db = 0.;
#pragma unroll 4
  for (unsigned long long row = first; row < last; ++row) {
    const float dy = to_float(((const T*)a.dy)[row * a.n + col]);
    const float u = (to_float(((const T*)a.x)[row * a.n + col]) - a.mean[row]) * a.rstd[row];
    dg = fma((double)dy, (double)u, dg);
    db += (double)dy;
  }
  a.partial[(unsigned long long)slice * a.n + col] = (float)dg;
  a.partial[((unsigned long long)slices + slice) * a.n + col] = (float)db;
}

// Partial sums of `blocks` blocks, added in their order: 32 columns x 32 runs of blocks, then the runs.
__global__ void __launch_bounds__(1024) norm_grad_join(const float* partial, unsigned int blocks, unsigned int n, float* dgamma, float* dbeta) {
  __shared__ double sh[32][33];
  grid_begin();
  const unsigned int col = blockIdx.x * 32 + threadIdx.x, which = blockIdx.y;
  float* out = which ? dbeta : dgamma;
  double v = 0.;
  if (out && col < n) {
    const float* p = partial + (unsigned long long)which * blocks * n + col;
#pragma unroll 4
    for (unsigned int b = threadIdx.y; b < blocks; b += 32) v += (double)p[(unsigned long long)b * n];
  }
  sh[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && out && col < n) {
    double s = 0.;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sh[i][threadIdx.x];
    out[col] = (float)s;
  }
}

typedef void (*NormKernel)(const NormArgs);

struct NormPlan {
  NormKernel kernel = nullptr;
  unsigned int block = 0, tpr = 0, elements = 0;       // elements a thread
};

template <class T, int VEC, int NV>
NormPlan rows_of(bool grad, unsigned int n) {
  const unsigned int e = VEC * NV;
  // (a gradient's blocks are larger: each leaves a row of partial sums)
  const unsigned int block = grad ? 512 : 256;
  if (n <= 8 * e) return {grad ? norm_grad_rows<T, VEC, NV, 8> : norm_rows<T, VEC, NV, 8>, block, 8, e};
  if (n <= 32 * e) return {grad ? norm_grad_rows<T, VEC, NV, 32> : norm_rows<T, VEC, NV, 32>, block, 32, e};
  if (n <= 128 * e) return {grad ? norm_grad_rows<T, VEC, NV, 128> : norm_rows<T, VEC, NV, 128>, block, 128, e};
  return {grad ? norm_grad_rows<T, VEC, NV, 512> : norm_rows<T, VEC, NV, 512>, 512, 512, e};
}

// The group of threads is the smallest that holds a row at 16 elements a thread; rows of at most half of what it holds
// take 8 a thread.
template <class T>
NormPlan plan_of(bool grad, unsigned int n, bool vec) {
  constexpr int V = 16 / (int)sizeof(T);
  // (forward rows of up to 16384 elements still fit the registers of 1024 threads)
  if (!grad && vec && n > 8192 && n <= 16384) return {norm_rows<T, V, 16 / V, 1024>, 1024, 1024, 16};
  if (n > 8192) {
    if (vec) return {grad ? norm_grad_wide<T, V> : norm_wide<T, V>, 1024, 1024, 0};
    return {grad ? norm_grad_wide<T, 1> : norm_wide<T, 1>, 1024, 1024, 0};
  }
  // 16 single elements a thread, or the gradient's 16 of single precision, twice for the next row, would not fit its registers (1999
  // rows of 777 single elements: 19.5 us, 8.8 with 8 of them); between 4096 and 8192 they have to.
  constexpr unsigned int kMost = 512;
  if (!vec) return n <= kMost * 8 ? rows_of<T, 1, 8>(grad, n) : NormPlan{grad ? norm_grad_rows<T, 1, 16, kMost> : norm_rows<T, 1, 16, kMost>, kMost, kMost, 16};
  if (sizeof(T) == 4 && grad)
    return n <= kMost * 8 ? NormPlan(rows_of<T, V, 8 / V>(true, n)) : NormPlan{norm_grad_rows<T, V, 16 / V, kMost>, kMost, kMost, 16};
  const unsigned int g = n <= 128 ? 8 : n <= 512 ? 32 : n <= 2048 ? 128 : 512;
  return n <= g * 8 ? rows_of<T, V, 8 / V>(grad, n) : rows_of<T, V, 16 / V>(grad, n);
}

struct NormOperator : b200_operator {
  NormArgs a = {};
  NormPlan plan;
  int dtype = 0;
  bool grad = false;
  size_t smem = 0;
  unsigned int grid = 0, slices = 0;
  float *dgamma = nullptr, *dbeta = nullptr;

  void choose() {
    const size_t size = dtype_bytes(dtype);
    bool vec = (size_t)a.n * size % 16 == 0;
    for (const void* p : {a.x, a.r, a.dy, a.dh, (const void*)a.y, (const void*)a.h, (const void*)a.dx}) vec &= ((size_t)p & 15) == 0;
    plan = dtype == B200_F32 ? plan_of<float>(grad, a.n, vec) : dtype == B200_BF16 ? plan_of<__nv_bfloat16>(grad, a.n, vec) : plan_of<__half>(grad, a.n, vec);
    const unsigned int per_block = plan.block / plan.tpr;
    const bool wide = plan.elements == 0;
    smem = wide ? 0 : (size_t)plan.tpr * plan.elements * 4 * (grad ? 1 : 2);
    if (grad && per_block > 1 && !wide) smem = std::max(smem, 2 * (size_t)per_block * a.n * 4);
    // (up to 28000 elements; wider rows' column sums take a pass of their own)
    if (wide && grad && (dgamma || dbeta) && (size_t)a.n * 8 <= 224 * 1024) {
      a.own_columns = 1;
      smem = (size_t)a.n * 8;
    }
    ready(plan.kernel, smem);
    int resident = 0;
    rt_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, plan.kernel, (int)plan.block, smem), "occupancy");
    const unsigned long long blocks = (a.rows + per_block - 1) / per_block;
    grid = (unsigned int)std::min<unsigned long long>(blocks, (unsigned long long)std::max(1, resident) * (unsigned)dev->sm_count);
    if (grad && (dgamma || dbeta)) {
      ready(norm_grad_join);
      unsigned int partials = grid;
      if (wide && !a.own_columns) {
        // enough blocks for the machine, at least 32 rows each
        const unsigned int across = (a.n + 255) / 256;
        slices = (unsigned int)std::max<unsigned long long>(1, std::min<unsigned long long>(a.rows / 32, (8u * dev->sm_count + across - 1) / across));
        partials = slices;
        if (dtype == B200_F32) ready(norm_grad_columns<float>);
        else if (dtype == B200_BF16) ready(norm_grad_columns<__nv_bfloat16>);
        else ready(norm_grad_columns<__half>);
      }
      take_workspace((size_t)2 * std::max(1u, partials) * a.n * 4);
      a.partial = (float*)workspace;
    }
  }

  void run(cudaStream_t s) override {
    if (grid) launch(plan.kernel, grid, plan.block, smem, s, a);
    if (!a.partial) return;
    unsigned int partials = grid;
    if (slices && a.rows) {
      const dim3 g((a.n + 255) / 256, slices);
      if (dtype == B200_F32) launch(norm_grad_columns<float>, g, 256, 0, s, a, slices);
      else if (dtype == B200_BF16) launch(norm_grad_columns<__nv_bfloat16>, g, 256, 0, s, a, slices);
      else launch(norm_grad_columns<__half>, g, 256, 0, s, a, slices);
      partials = slices;
    }
    // (no rows: no partial sums, zeros)
    launch(norm_grad_join, dim3((a.n + 31) / 32, 2), dim3(32, 32), 0, s, (const float*)workspace, a.rows ? partials : 0u, a.n, dgamma, dbeta);
  }
};

void check_norm(const b200_layer_norm& p, const Operands& ops) {
  ops.dtype(p.dtype);
  if (p.weight_dtype != B200_F32 && p.weight_dtype != p.dtype) ops.refuse("gamma and beta are single precision or of the rows' type");
  if (p.rows < 0 || p.n < 1 || p.n > (1ll << 30)) ops.refuse("rows must not be negative, n between 1 and 2^30");
  if (!(p.eps >= 0.f)) ops.refuse("eps must not be negative");
}

}  // namespace

extern "C" int b200_layer_norm_link(b200_dev* dev, const b200_layer_norm* p, b200_operator** out) {
  return link_operator<NormOperator>(dev, p, out, [&](NormOperator* op) {
    Operands ops(op, "layer_norm");
    check_norm(*p, ops);
    const unsigned long long count = extent_product({p->rows, p->n}, "layer_norm");
    const size_t size = dtype_bytes(p->dtype), wsize = dtype_bytes(p->weight_dtype);
    op->dtype = p->dtype;
    NormArgs& a = op->a;
    a.x = (const void*)ops.in(p->x, "x", count, size);
    a.r = (const void*)ops.in(p->residual, "residual", count, size, false);
    a.gamma = (const void*)ops.in(p->gamma, "gamma", p->n, wsize, false);
    a.beta = (const void*)ops.in(p->beta, "beta", p->n, wsize, false);
    a.y = (void*)ops.out(p->y, "y", count, size);
    a.h = (void*)ops.out(p->total, "total", count, size, false);
    a.mean = (float*)ops.out(p->mean, "mean", p->rows, 4, false);
    a.rstd = (float*)ops.out(p->rstd, "rstd", p->rows, 4, false);
    if (a.h && !a.r) ops.refuse("'total' is the sum with a residual, which is not given");
    ops.check_overlaps();
    a.rows = (unsigned long long)p->rows;
    a.n = (unsigned int)p->n;
    a.weight_f32 = p->weight_dtype == B200_F32;
    a.eps = p->eps;
    a.inv_n = 1.f / (float)p->n;
    op->choose();
  });
}

extern "C" int b200_layer_norm_grad_link(b200_dev* dev, const b200_layer_norm* p, b200_operator** out) {
  return link_operator<NormOperator>(dev, p, out, [&](NormOperator* op) {
    Operands ops(op, "layer_norm_grad");
    check_norm(*p, ops);
    const unsigned long long count = extent_product({p->rows, p->n}, "layer_norm_grad");
    const size_t size = dtype_bytes(p->dtype), wsize = dtype_bytes(p->weight_dtype);
    op->dtype = p->dtype;
    op->grad = true;
    NormArgs& a = op->a;
    a.x = (const void*)ops.in(p->x, "x", count, size);
    a.gamma = (const void*)ops.in(p->gamma, "gamma", p->n, wsize, false);
    a.mean = (float*)ops.in(p->mean, "mean", p->rows, 4);
    a.rstd = (float*)ops.in(p->rstd, "rstd", p->rows, 4);
    a.dy = (const void*)ops.in(p->dy, "dy", count, size);
    a.dh = (const void*)ops.in(p->d_total, "d_total", count, size, false);
    a.dx = (void*)ops.out(p->dx, "dx", count, size);
    op->dgamma = (float*)ops.out(p->dgamma, "dgamma", p->n, 4, false);
    op->dbeta = (float*)ops.out(p->dbeta, "dbeta", p->n, 4, false);
    ops.check_overlaps();
    a.rows = (unsigned long long)p->rows;
    a.n = (unsigned int)p->n;
    a.weight_f32 = p->weight_dtype == B200_F32;
    a.inv_n = 1.f / (float)p->n;
    op->choose();
  });
}
