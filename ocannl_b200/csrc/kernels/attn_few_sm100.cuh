// Attention of a few new rows over many keys, 16-bit heads: the next tokens of sequences over their caches.
//
// The keys and values are read once and bound it.  The query heads that share a key head, and their few rows, are the 16 rows of a
// tile of mma.m16n8k16 (tcgen05 has no tile of 16 rows); up to 16 of them ride on one pass over the keys.  The keys of a (sequence, key
// head) are cut into `splits` ranges, one a block, so that a few sequences fill the machine; a block's four warps take
// every fourth step of 16 keys, each with a ring of its own that cp.async fills two steps ahead, and its own running maximum, sum and
// output.  The warps meet in shared memory, the blocks in the workspace: the block that comes last joins the ranges in their
// order (the same bits whoever comes last), or, where a warp of it would have several rows to join, a second launch with a block a row.  Keys behind the last visible one are not read but zeroed in shared memory.
#ifndef B200_ATTN_FEW_SM100_CUH
#define B200_ATTN_FEW_SM100_CUH
#include "attn_fwd_sm100.cuh"

namespace b200 {

constexpr int kFewRows = 16, kFewStep = 16, kFewStages = 3, kFewWarps = 4, kFewMost = 256;   // (most ranges)

struct FewArgs {
  float* parts;            // [pair][split][16][DP + 4]: output (not divided), maximum, sum (half weights times 2^7), and two floats that
                           // keep rows on 16 bytes
  unsigned int* tickets;   // [pair], zero between runs
  int splits, per_split;   // keys of a range, a multiple of 16 * 4
  int join_later;          // the ranges are joined by a launch of its own
};

template <int DP>
struct FewShape {
  static constexpr int kRow = DP + 8;                                  // elements of a staged row: no bank is met twice by ldmatrix
  static constexpr int kStage = 2 * kFewStep * kRow * 2;               // bytes: keys, then values
  static constexpr int kRing = kFewStages * kStage;                    // of a warp
  static constexpr int kWidth = DP + 4;
  static constexpr int kJoin = kFewWarps * kFewRows * kWidth * 4;
  static constexpr int smem() { return kFewWarps * kRing; }
  static_assert(kJoin + kFewWarps * DP * 4 <= kFewWarps * kRing, "the warps meet where the rings were");
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

// The maximum and the sum of `n` partial rows `step` apart, and in `weight` (n of them) what each is multiplied by: a warp.
// (a part without visible keys has a sum of exactly 0 and counts nothing, whatever else it holds; one whose visible scores are all
// undefined has no maximum either, but an undefined sum, which has to reach the result)
template <int DP>
__device__ __forceinline__ void few_weigh(const float* from, int n, long long step, float* weight, float& top, float& sum) {
  const unsigned int lane = threadIdx.x & 31u;
  float t[kFewMost / 32], u[kFewMost / 32];
  top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kFewMost / 32; ++k) {
    const int i = (int)lane + 32 * k;
    t[k] = i < n ? from[i * step + DP] : -INFINITY;
    u[k] = i < n ? from[i * step + DP + 1] : 0.f;
    top = fmaxf(top, t[k]);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  sum = 0.f;
  __syncwarp();                     // (all lanes have read the weights of the row before)
#pragma unroll
  for (int k = 0; k < kFewMost / 32; ++k) {
    const float w = u[k] == 0.f ? 0.f : t[k] == -INFINITY ? 1.f : ex2(t[k] - top);
    if ((int)lane + 32 * k < n) weight[lane + 32 * k] = w;
    if (w != 0.f) sum = fmaf(w, u[k], sum);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  __syncwarp();
}
// four elements of the sum of every `each`-th weighed part from `i0` on; eight loads under way together
__device__ __forceinline__ float4 few_gather(const float* from, int n, long long step, const float* weight, int e, int i0, int each) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = i0; i < n; i += 8 * each) {
    float4 x[8];
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int at = i + k * each;
      w[k] = at < n ? weight[at] : 0.f;
      x[k] = *(const float4*)(from + (at < n ? at : i) * step + e);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (w[k] != 0.f) v = make_float4(fmaf(w[k], x[k].x, v.x), fmaf(w[k], x[k].y, v.y), fmaf(w[k], x[k].z, v.z), fmaf(w[k], x[k].w, v.w));
  }
  return v;
}
// Writes four elements of a row and, with the first, its lse.  False: one is infinite or undefined, and the row has to be mended (0 times
// infinity from a hidden key among visible ones)
template <class T>
__device__ __forceinline__ bool few_finish(const AttnArgs& a, int b, int h, int r, int e, const float4& v, float top, float sum) {
  const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const float y[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
  T* to = (T*)a.out + attn_q_at(a, b, r, h) + e;
  bool fine = true;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (e + k < a.D) {
      from_float(y[k], to[k]);
      fine = fine && y[k] * 0.f == 0.f;
    }
  if (e == 0 && a.lse) a.lse[((long long)b * a.H + h) * a.S + r] = by != 0.f ? (top - kLift<T> + log2f(sum)) * kLn2 : -INFINITY;
  return fine;
}
// One row by a block: each of the four warps adds every fourth part, the first adds the four sums.
template <class T, int DP>
__device__ __forceinline__ void few_row_of_block(const AttnArgs& a, int b, int h, int r, const float* from, int n, float* weight, float4* meet) {
  constexpr int step = kFewRows * FewShape<DP>::kWidth;
  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  float top, sum;
  few_weigh<DP>(from, n, step, weight, top, sum);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (lane < DP / 4) v = few_gather(from, n, step, weight, 4 * (int)lane, (int)warp, kFewWarps);
  __syncthreads();
  if (lane < DP / 4) meet[warp * (DP / 4) + lane] = v;
  __syncthreads();
  if (warp) return;
  bool fine = true;
  if (lane < DP / 4) {
    for (int w = 1; w < kFewWarps; ++w) {
      const float4 x = meet[w * (DP / 4) + lane];
      v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
    }
    fine = few_finish<T>(a, b, h, r, 4 * (int)lane, v, top, sum);
  }
  if (attn_again(fine)) attn_forward_row<T>(a, b, h, r, lane);
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
  for (int w = 0; w < 2; ++w) {
    const bool on = first_row + (w ? rb : ra) < shared_rows;
    const unsigned short* p = (const unsigned short*)a.q + (on ? attn_q_at(a, b, query_of(w ? rb : ra), head_of(w ? rb : ra)) : 0) + (lane & 3u) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = ks * 16 + i * 8;
        // (rows lie on 16 bytes, zeros behind their end)
        q[ks][2 * i + w] = on && e + (int)(lane & 3u) * 2 < a.D ? *(const unsigned int*)(p + e) : 0u;
      }
  }

  float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
  const float c = CAP ? a.cap * kLog2e : a.scale * kLog2e, to_tanh = CAP ? a.over : 0.f;
  const unsigned int ring = b200_smem_addr(dyn) + warp * Sh::kRing;
  const int steps = j_end > j_begin ? (j_end - j_begin + kFewStep - 1) / kFewStep : 0;
  const int mine = steps > (int)warp ? (steps - (int)warp + kFewWarps - 1) / kFewWarps : 0;     // this warp's steps

  // a lane copies the same 16 bytes of every kRowsApart-th row of a step, from pointers that move on with the steps
  constexpr int kPieces = DP / 8, kRowsApart = 32 / kPieces;
  const int my_row = (int)lane / kPieces, my_piece = (int)lane % kPieces;
  const bool in_head = my_piece * 8 < a.D;
  const long long stride = (long long)a.HK * a.ld;
  int next_j = j_begin + (int)warp * kFewStep + my_row;
  const unsigned short *next_k = (const unsigned short*)a.k + attn_k_at(a, b, 0, hk) + (long long)next_j * stride + my_piece * 8,
                       *next_v = (const unsigned short*)a.v + attn_k_at(a, b, 0, hk) + (long long)next_j * stride + my_piece * 8;
  const unsigned int my_slot = ring + (my_row * Sh::kRow + my_piece * 8) * 2;
  unsigned int to = 0;               // the slot that is filled next
  auto fetch = [&](int n) {
    if (n < mine) {
      const unsigned int at = my_slot + to * Sh::kStage;
#pragma unroll
      for (int i = 0; i < kFewStep / kRowsApart; ++i) {
        const bool on = in_head && next_j + i * kRowsApart < j_end;
        copy16(at + i * kRowsApart * Sh::kRow * 2, on ? next_k + i * kRowsApart * stride : (const unsigned short*)a.k, on);
        copy16(at + (i * kRowsApart + kFewStep) * Sh::kRow * 2, on ? next_v + i * kRowsApart * stride : (const unsigned short*)a.v, on);
      }
      next_j += kFewWarps * kFewStep;
      next_k += kFewWarps * kFewStep * stride;
      next_v += kFewWarps * kFewStep * stride;
      to = to + 1 == kFewStages ? 0 : to + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kFewStages - 1; ++i) fetch(i);
  const int all_see = __reduce_min_sync(0xffffffffu, min(first_row + ra < shared_rows ? row[0].last : 0x7fffffff, first_row + rb < shared_rows ? row[1].last : 0x7fffffff));
  unsigned int slot = 0;
  for (int n = 0; n < mine; ++n) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
    __syncwarp();
    fetch(n + kFewStages - 1);        // into the slot of the step before, which the whole warp has left
    const int j0 = j_begin + ((int)warp + n * kFewWarps) * kFewStep;
    const unsigned int k_at = ring + slot * Sh::kStage, v_at = k_at + kFewStep * Sh::kRow * 2;
    slot = slot + 1 == kFewStages ? 0 : slot + 1;
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
    if constexpr (CAP) {
      tanh_chunk(s[0], to_tanh);
      tanh_chunk(s[1], to_tanh);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[h][i] *= c;
        if constexpr (BIAS) s[h][i] = fmaf(-slope2[i >> 1], fabsf((float)(row[i >> 1].pos - j0 - h * 8 - (int)(lane & 3u) * 2 - (i & 1))), s[h][i]);
      }
    if (a.kdoc || j0 + kFewStep - 1 > all_see) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int w = i >> 1, j = j0 + h * 8 + (int)(lane & 3u) * 2 + (i & 1);
          bool on = j <= row[w].last;
          if (a.kdoc) on = on && a.kdoc[(long long)b * a.T + j] == row[w].doc;
          s[h][i] = on ? s[h][i] : -INFINITY;
        }
    }
    // the maximum in use moves when a row has outgrown it by 2^8 (or has had none): hardly ever after the first steps
    float top[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) top[w] = fmaxf(fmaxf(s[0][2 * w], s[0][2 * w + 1]), fmaxf(s[1][2 * w], s[1][2 * w + 1]));
    if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 1));
        top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 2));
        const float next = fmaxf(m[w], top[w]);
        const float by = m[w] == next ? 1.f : m[w] == -INFINITY ? 0.f : ex2(m[w] - next);
        m[w] = next;
        l[w] *= by;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][2 * w] *= by;
          o[i][2 * w + 1] *= by;
        }
      }
    }
    const float off[2] = {m[0] == -INFINITY ? 0.f : m[0] - kLift<T>, m[1] == -INFINITY ? 0.f : m[1] - kLift<T>};
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
  const int lane_e = 4 * (int)lane;
  __shared__ float weights[kFewWarps][kFewMost];
  float* parts = f.parts + ((long long)pair * f.splits + split) * kFewRows * W;
  // a warp takes every fourth row
  if (f.splits > 1) {
    for (int i = (int)warp; i < rows; i += kFewWarps) {
      float top, sum;
      few_weigh<DP>(join + i * W, kFewWarps, kFewRows * W, weights[warp], top, sum);
      if (lane_e < DP) *(float4*)(parts + i * W + lane_e) = few_gather(join + i * W, kFewWarps, kFewRows * W, weights[warp], lane_e, 0, 1);
      if (lane == 0) {
        parts[i * W + DP] = top;
        parts[i * W + DP + 1] = sum;
      }
    }
    if (f.join_later) return;
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
  if (rows == 1) {
    few_row_of_block<T, DP>(a, b, head_of(0), query_of(0), all, n_parts, weights[warp], (float4*)(dyn + sizeof(float) * kFewWarps * kFewRows * W));   // (behind `join`)
    return;
  }
  for (int i = (int)warp; i < rows; i += kFewWarps) {
    float top, sum;
    few_weigh<DP>(all + i * W, n_parts, kFewRows * W, weights[warp], top, sum);
    bool fine = true;
    if (lane_e < DP) fine = few_finish<T>(a, b, head_of(i), query_of(i), lane_e, few_gather(all + i * W, n_parts, kFewRows * W, weights[warp], lane_e, 0, 1), top, sum);
    if (attn_again(fine)) attn_forward_row<T>(a, b, head_of(i), query_of(i), lane);
  }
}

// The join of the ranges of one row, a block; blockIdx.x as above, blockIdx.y: the row of its sixteen
template <class T, int DP>
__global__ void __launch_bounds__(kFewWarps * 32) attn_join_few(const __grid_constant__ AttnArgs a, const FewArgs f) {
  __shared__ float weights[kFewWarps][kFewMost];
  __shared__ float4 meet[kFewWarps * DP / 4];
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int shared_rows = a.group * a.S, sixteens = (shared_rows + kFewRows - 1) / kFewRows;
  const int pair = (int)blockIdx.x, unit = pair / sixteens, i = (int)blockIdx.y, row = pair % sixteens * kFewRows + i;
  if (row >= shared_rows) return;
  few_row_of_block<T, DP>(a, unit / a.HK, unit % a.HK * a.group + row / a.S, row % a.S, f.parts + ((long long)pair * f.splits * kFewRows + i) * FewShape<DP>::kWidth, f.splits,
                          weights[threadIdx.x >> 5], meet);
}

}  // namespace b200
#endif
