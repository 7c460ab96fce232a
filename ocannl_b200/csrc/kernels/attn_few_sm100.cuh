// Attention of a few new rows over many keys, 16-bit heads: the next tokens of sequences over their caches.
//
// The keys and values are read once and bound it.  The query heads that share a key head, and their few rows, are the 16 rows of a
// tile of mma.m16n8k16 (tcgen05 has no tile of 16 rows); up to 16 of them ride on one pass over the keys.  The keys of a (sequence, key
// head) are cut into `splits` ranges, one a block, so that a few sequences fill the machine; a block's four warps take
// every fourth step of 16 keys, each with a ring of its own that cp.async fills two steps ahead, and its own running maximum, sum and
// output.  The warps meet in shared memory, the blocks in the workspace: the block that comes last joins the ranges in their
// order (the same bits whoever comes last).  Keys behind the last visible one are not read but zeroed in shared memory.
#ifndef B200_ATTN_FEW_SM100_CUH
#define B200_ATTN_FEW_SM100_CUH
#include "attn_fwd_sm100.cuh"

namespace b200 {

constexpr int kFewRows = 16, kFewStep = 16, kFewStages = 3, kFewWarps = 4, kFewMost = 256;   // (most ranges)

struct FewArgs {
  float* parts;            // [pair][split][16][DP + 4]: output (not divided), maximum, sum, and two floats that keep rows on 16 bytes
  unsigned int* tickets;   // [pair], zero between runs
  int splits, per_split;   // keys of a range, a multiple of 16 * 4
};

template <int DP>
struct FewShape {
  static constexpr int kRow = DP + 8;                                  // elements of a staged row: no bank is met twice by ldmatrix
  static constexpr int kStage = 2 * kFewStep * kRow * 2;               // bytes: keys, then values
  static constexpr int kRing = kFewStages * kStage;                    // of a warp
  static constexpr int kWidth = DP + 4;
  static constexpr int kJoin = kFewWarps * kFewRows * kWidth * 4;
  static constexpr int smem() { return kFewWarps * kRing > kJoin ? kFewWarps * kRing : kJoin; }
};

template <class T>
__device__ __forceinline__ void mma16(float (&d)[4], const unsigned int (&x)[4], unsigned int y0, unsigned int y1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(y0), "r"(y1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(y0), "r"(y1));
}
__device__ __forceinline__ void ldmatrix4(unsigned int (&r)[4], unsigned int at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(unsigned int (&r)[4], unsigned int at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// 16 bytes, zeros where not `on`
__device__ __forceinline__ void copy16(unsigned int dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// blockIdx.x: (sequence, key head, sixteen of the rows that share it); blockIdx.y: range of keys
template <class T, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kFewWarps * 32) attn_forward_few(const __grid_constant__ AttnArgs a, const FewArgs f) {
  typedef FewShape<DP> Sh;
  constexpr int KS = DP / 16;
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ unsigned int last_block;
  asm volatile("griddepcontrol.launch_dependents;");
  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const int shared_rows = a.group * a.S, sixteens = (shared_rows + kFewRows - 1) / kFewRows;
  const int pair = (int)blockIdx.x, unit = pair / sixteens, first_row = pair % sixteens * kFewRows;
  const int b = unit / a.HK, hk = unit % a.HK;
  const int split = (int)blockIdx.y;
  // row i of the tile: query head and position
  auto head_of = [&](int i) { return hk * a.group + (first_row + i) / a.S; };
  auto query_of = [&](int i) { return (first_row + i) % a.S; };
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // this thread's two accumulator rows
  const int ra = (int)lane / 4, rb = ra + 8;
  AttnRow row[2];
  float slope2[2] = {0.f, 0.f};
  int last = -1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int k = i ? rb : ra;
    row[i].pos = 0; row[i].last = -1; row[i].doc = 0;
    if (first_row + k < shared_rows) {
      row[i] = attn_row(a, b, query_of(k));
      if (BIAS) slope2[i] = a.slopes[head_of(k)] * kLog2e;
    }
    last = max(last, row[i].last);
  }
  last = __reduce_max_sync(0xffffffffu, last);
  const int j_begin = split * f.per_split, j_end = min(j_begin + f.per_split, last + 1);

  // the queries as the A operand, straight from memory: rows ra and rb, elements 2 (lane % 4) .. of each eight
  unsigned int q[KS][4];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = i & 1 ? rb : ra, e = ks * 16 + (i >> 1) * 8 + (int)(lane & 3u) * 2;
      q[ks][i] = 0u;
      if (first_row + k < shared_rows && e < a.D) {
        const unsigned short* p = (const unsigned short*)a.q + attn_q_at(a, b, query_of(k), head_of(k)) + e;
        q[ks][i] = (unsigned int)p[0] | (e + 1 < a.D ? (unsigned int)p[1] << 16 : 0u);
      }
    }

  float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
  const float c = CAP ? a.cap * kLog2e : a.scale * kLog2e, to_tanh = CAP ? 2.f * kLog2e * a.scale / a.cap : 0.f;
  const unsigned int ring = b200_smem_addr(dyn) + warp * Sh::kRing;
  const int steps = j_end > j_begin ? (j_end - j_begin + kFewStep - 1) / kFewStep : 0;
  const int mine = steps > (int)warp ? (steps - (int)warp + kFewWarps - 1) / kFewWarps : 0;     // this warp's steps

  auto fetch = [&](int n) {
    if (n < mine) {
      const int j0 = j_begin + ((int)warp + n * kFewWarps) * kFewStep;
      const unsigned int at = ring + (n % kFewStages) * Sh::kStage;
      constexpr int pieces = DP / 8;
#pragma unroll
      for (int i = (int)lane; i < kFewStep * pieces; i += 32) {
        const int r = i / pieces, p = i % pieces;
        const bool on = j0 + r < j_end && p * 8 < a.D;
        const long long src = on ? attn_k_at(a, b, j0 + r, hk) + p * 8 : 0;
        const unsigned int dst = at + (r * Sh::kRow + p * 8) * 2;
        copy16(dst, (const unsigned short*)a.k + src, on);
        copy16(dst + kFewStep * Sh::kRow * 2, (const unsigned short*)a.v + src, on);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kFewStages - 1; ++i) fetch(i);
  for (int n = 0; n < mine; ++n) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
    __syncwarp();
    fetch(n + kFewStages - 1);        // into the slot of the step before, which the whole warp has left
    const int j0 = j_begin + ((int)warp + n * kFewWarps) * kFewStep;
    const unsigned int k_at = ring + (n % kFewStages) * Sh::kStage, v_at = k_at + kFewStep * Sh::kRow * 2;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    // keys 0-7 and 8-15, elements 0-7 and 8-15 of each sixteen: four 8 x 8 blocks
    const unsigned int k_row = k_at + (((lane & 7u) + (lane >> 4) * 8) * Sh::kRow + ((lane >> 3) & 1u) * 8) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      unsigned int y[4];
      ldmatrix4(y, k_row + ks * 32);
      mma16<T>(s[0], q[ks], y[0], y[1]);
      mma16<T>(s[1], q[ks], y[2], y[3]);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int w = i >> 1, j = j0 + h * 8 + (int)(lane & 3u) * 2 + (i & 1);
        float x = s[h][i];
        if constexpr (CAP) x = tanh_of(x * to_tanh);
        x *= c;
        if constexpr (BIAS) x = fmaf(-slope2[w], fabsf((float)(row[w].pos - j)), x);
        bool on = j <= row[w].last;
        if (a.kdoc) on = on && a.kdoc[(long long)b * a.T + j] == row[w].doc;
        s[h][i] = on ? x : -INFINITY;
        top[w] = fmaxf(top[w], s[h][i]);
      }
    float by[2], off[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 1));
      top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 2));
      const float next = fmaxf(m[w], top[w]);
      by[w] = m[w] == next ? 1.f : m[w] == -INFINITY ? 0.f : ex2(m[w] - next);
      m[w] = next;
      off[w] = next == -INFINITY ? 0.f : next;
      l[w] *= by[w];
    }
    // weights as the A operand: rows ra, rb, keys 0-7 and 8-15
    unsigned int p[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float p0 = ex2(s[h][0] - off[0]), p1 = ex2(s[h][1] - off[0]), p2 = ex2(s[h][2] - off[1]), p3 = ex2(s[h][3] - off[1]);
      l[0] += p0 + p1;
      l[1] += p2 + p3;
      p[2 * h] = pack2(p0, p1, T());
      p[2 * h + 1] = pack2(p2, p3, T());
    }
    if (__any_sync(0xffffffffu, by[0] != 1.f || by[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        o[i][0] *= by[0]; o[i][1] *= by[0];
        o[i][2] *= by[1]; o[i][3] *= by[1];
      }
    }
    // values: keys 0-7 and 8-15 of elements 0-7, then of elements 8-15, of each sixteen
    const unsigned int v_row = v_at + (((lane & 7u) + ((lane >> 3) & 1u) * 8) * Sh::kRow + (lane >> 4) * 8) * 2;
#pragma unroll
    for (int e = 0; e < KS; ++e) {
      unsigned int y[4];
      ldmatrix4_t(y, v_row + e * 32);
      mma16<T>(o[2 * e], p, y[0], y[1]);
      mma16<T>(o[2 * e + 1], p, y[2], y[3]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
  }
  __syncthreads();                  // the rings become the place where the warps meet
  constexpr int W = Sh::kWidth;
  float* join = (float*)dyn;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float* to = join + (warp * kFewRows + (w ? rb : ra)) * W;
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
      to[i * 8 + (lane & 3u) * 2] = o[i][2 * w];
      to[i * 8 + (lane & 3u) * 2 + 1] = o[i][2 * w + 1];
    }
    if ((lane & 3u) == 0) {
      to[DP] = m[w];
      to[DP + 1] = l[w];
    }
  }
  __syncthreads();
  const int rows = min(kFewRows, shared_rows - first_row);
  // The maximum and the sum of `n` partial rows `step` apart, and in `weight` (n of them) what each is multiplied by: a warp.
  // (a part without visible keys counts nothing, whatever it holds)
  auto weigh = [&](const float* from, int n, long long step, float* weight, float& top, float& sum) {
    top = -INFINITY;
    for (int i = (int)lane; i < n; i += 32) top = fmaxf(top, from[i * step + DP]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    sum = 0.f;
    for (int i = (int)lane; i < n; i += 32) {
      const float t = from[i * step + DP], w = t == -INFINITY ? 0.f : ex2(t - top);
      weight[i] = w;
      if (w != 0.f) sum = fmaf(w, from[i * step + DP + 1], sum);
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    __syncwarp();
  };
  // four elements of the sum of the weighed parts
  auto gather = [&](const float* from, int n, long long step, const float* weight, int e) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float w = weight[i];
      const float4 x = *(const float4*)(from + i * step + e);
      if (w != 0.f) v = make_float4(fmaf(w, x.x, v.x), fmaf(w, x.y, v.y), fmaf(w, x.z, v.z), fmaf(w, x.w, v.w));
    }
    return v;
  };
  bool fine = true;
  auto finish = [&](int i, int e, const float4& v, float top, float sum) {
    const int h = head_of(i), r = query_of(i);
    const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const float y[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
    T* to = (T*)a.out + attn_q_at(a, b, r, h) + e;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (e + k < a.D) {
        from_float(y[k], to[k]);
        fine = fine && y[k] * 0.f == 0.f;
      }
    if (e == 0 && a.lse) a.lse[((long long)b * a.H + h) * a.S + r] = by != 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
  };
  __shared__ float weights[kFewWarps][kFewMost];
  float* parts = f.parts + ((long long)pair * f.splits + split) * kFewRows * W;
  // a warp takes every fourth row; rows with a value that is infinite or undefined are mended (0 times infinity from a hidden key
  // among visible ones)
  if (f.splits > 1) {
    for (int i = (int)warp; i < rows; i += kFewWarps) {
      float top, sum;
      weigh(join + i * W, kFewWarps, kFewRows * W, weights[warp], top, sum);
      if ((int)lane < DP / 4) *(float4*)(parts + i * W + 4 * lane) = gather(join + i * W, kFewWarps, kFewRows * W, weights[warp], 4 * (int)lane);
      if (lane == 0) {
        parts[i * W + DP] = top;
        parts[i * W + DP + 1] = sum;
      }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last_block = atomicAdd(&f.tickets[pair], 1u) == (unsigned int)f.splits - 1u;
    __syncthreads();
    if (!last_block) return;
    if (threadIdx.x == 0) f.tickets[pair] = 0u;      // for the next run
    __threadfence();
  }
  const float* all = f.splits > 1 ? f.parts + (long long)pair * f.splits * kFewRows * W : join;
  const int n_parts = f.splits > 1 ? f.splits : kFewWarps;
  for (int i = (int)warp; i < rows; i += kFewWarps) {
    float top, sum;
    weigh(all + i * W, n_parts, kFewRows * W, weights[warp], top, sum);
    fine = true;
    if ((int)lane < DP / 4) finish(i, 4 * (int)lane, gather(all + i * W, n_parts, kFewRows * W, weights[warp], 4 * (int)lane), top, sum);
    if (__any_sync(0xffffffffu, !fine)) attn_forward_row<T>(a, b, head_of(i), query_of(i), lane);
  }
}

}  // namespace b200
#endif
