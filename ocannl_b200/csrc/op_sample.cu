// Choosing a token for each row of logits (b200_sample_link).
//
//   w_i = exp((x_i - max) / T);  kept: the first n in the order of falling x, of rising i among equal ones;  token: where the running sum of the kept, in the
//   order of i, passes uniform * its end
//
// A row is read once, and again from L2 in two or three more passes.  A cluster of up to eight blocks takes it and exchanges sums through
// shared memory.  What is kept is all logits above a border and, of those equal to it, the ones up to an index: no sort of the row.  The border is found by a
// histogram of 32 bins, half a binade of weight each, of counts and sums of weights; every lane has columns of its own, so that nothing is added atomically, and
// adds whole numbers, so that sums come out the same in whatever order and are exact but for a weight's own rounding.  A bin that bounds what is kept, with all above
// it, is usually a few hundred logits: these go to one block, which sorts them and does the rest in 64 bits.  Where they are more than 1024, the bin is divided
// again by the bits of its logits, until it is small or of one value, and the row is passed once more for the token.
// In the passes a weight is single (the exponential's 2^-22, and what its exponent's rounding makes: equal logits have equal weights, others' errors do not add up), with
// a rate in two parts, so that borders and tokens lie where 64 bits have them but for some 2^-10 of a weight in rows of 10^5 weights of one size.
// Measured: 256 rows of 131072 logits 203 us, 64 of 50021 in bfloat16 44 us (in double precision throughout 312 and 55): 89 million instructions of warps at half of
// the issue slots; three blocks an SM wait for their logits' passes and for one another (the bytes alone: 20 us).
#include <cooperative_groups.h>

#include <cmath>
#include <type_traits>

#include "kernels/op_common.cuh"
#include "operators.hpp"

using namespace b200;
namespace cg = cooperative_groups;

namespace {

struct SampleArgs {
  const void* x;
  const float *uniform, *temperatures, *top_ps, *min_ps;
  const int* top_ks;
  int* tokens;
  float* logprob;
  unsigned int rows, vocab;
  unsigned int parts, span;            // blocks of a row, logits of a warp (in memory: of a block's eighth)
  float temperature, top_p, min_p;
  int top_k;
};

constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 32, kList = 1024, kLocal = 2 * kList, kMostParts = 8;

// A column of a histogram is two whole numbers, which do not care in which order they are added: the sum of weights in steps of 2^-22 of the bin's unit, and
// what they were rounded by in steps of 2^-34 with the number of logits above it.  (Weights of a bin are below 1.25 of its unit, so 800 logits pass neither.)
constexpr int kColumn = 800, kCountBits = 10;
struct Column {
  unsigned int sum, rest;
  // w: in units of 2^-17 of the bin's.  A sum with 2^23 has the nearest whole number in its low bits; rests lie between -1/2 and 1/2 and are counted from there.
  __device__ __forceinline__ void add(float w) {
    const float whole = fmaf(w, 32.f, 8388608.f), left = fmaf(w, 32.f, 8388608.f - whole);
    sum += __float_as_uint(whole) - 0x4b000000u;
    rest += __float_as_uint(fmaf(left, 4096.f, 8388608.f + 2048.f)) - 0x4b000000u + (1u << (32 - kCountBits));
  }
  __device__ __forceinline__ unsigned int count() const { return rest >> (32 - kCountBits); }
  // of `count` logits, in steps of 2^-34
  __device__ __forceinline__ long long total() const { return ((long long)sum << 12) + (rest & ((1u << (32 - kCountBits)) - 1u)) - 2048ll * count(); }
};

// Rises with the value; one key for both zeros, as they are equal.  What is undefined lies outside the keys of -infinity and infinity.
__device__ __forceinline__ unsigned int key_of(float x) {
  const unsigned int u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned int k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Share {                         // of a block, for the others of its cluster to read
  union {
    unsigned int local[kLocal];        // indices of logits of this block's that may be at the border
    unsigned long long list[kList];    // (rows in registers) the logits themselves, as they are sorted
  };
  unsigned int listed;                 // entries of the list (more than it holds: it is of no use)
  unsigned int joined;                 // of the first block: entries of the list that all blocks' go to
  unsigned int joined_from;            // where this block's begin there
  double sums[2][kBins];               // of one histogram and the next
  unsigned int counts[2][kBins];
  double warp_sums[kWarps];
  unsigned int warp_counts[kWarps];
  float largest;
  unsigned int first;                  // an index
  float border;                        // of the first block: the last logit that is kept, and its index
  unsigned int border_at;
  unsigned int interval[2];
  float scratch[kWarps];
  double joined_sums[kBins];           // over all blocks
  unsigned int joined_counts[kBins];
  double block_sums[kWarps];
};

struct Pick {                          // a histogram's bin
  unsigned int bin, above, in;         // logits above it, and in it
  double sum_above;
};

// The row as the blocks of its cluster hold it: E logits a thread in registers (0: they are read again every time), VEC neighbours of 16 bytes a lane, a warp's
// all in one piece.  Places count from the 16 bytes that the row begins in: `off` of them lie ahead of it.
template <class T, int E>
struct Logits {
  static constexpr int VEC = 16 / (int)sizeof(T), kAtOnce = sizeof(T) == 4 ? 4 : 2;
  float x[E ? E : 1];
  const T* row;                        // place 0
  unsigned int off, end, begin, count; // places of the row: off .. end - 1; begin: of this lane's first vector; count: vectors of a lane
  __device__ __forceinline__ bool whole(unsigned int at) const { return at >= off && at + VEC <= end; }
  __device__ __forceinline__ void some(unsigned int at, float (&v)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = at + i >= off && at + i < end ? to_float(row[at + i]) : -INFINITY;
  }
  __device__ __forceinline__ Logits(const SampleArgs& a, unsigned int r, unsigned int part) {
    row = (const T*)a.x + (unsigned long long)r * a.vocab;
    off = (unsigned int)((size_t)row / sizeof(T)) % VEC;
    row -= off;
    end = a.vocab + off;
    const unsigned int lane = threadIdx.x & 31u;
    const unsigned long long from = (unsigned long long)(part * kWarps + (threadIdx.x >> 5)) * a.span;
    begin = (unsigned int)min(from, (unsigned long long)end) + lane * VEC;
    count = from < end ? (unsigned int)((min((unsigned long long)a.span, end - from) + 32 * VEC - 1) / (32 * VEC)) : 0u;
    if constexpr (E > 0) {
#pragma unroll
      for (int v = 0; v < E / VEC; ++v) {
        float y[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[i] = -INFINITY;
        if (v < (int)count) some(begin + v * 32 * VEC, y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[v * VEC + i] = y[i];
      }
    }
  }
  static constexpr int kBatch = E ? E : kAtOnce * VEC;
  // vectors of a lane that hold no more logits than a column of a histogram counts, a whole number of batches
  static constexpr unsigned int kCounted = kColumn / kBatch * kAtOnce;
  // f(logits, index of each), kBatch at a time, which are under way together; -infinity ahead of the row and behind it, and where a lane has no more.  The
  // lanes of a warp come here together.  Of a lane's vectors those from v0 on, up to `end_v`.
  template <class F>
  __device__ __forceinline__ void batches(F f, unsigned int v0 = 0, unsigned int end_v = 0xffffffffu) const {
    if constexpr (E > 0) {
      f(x, [&](int e) { return begin + (e / VEC) * 32 * VEC + e % VEC - off; });
    } else {
      for (unsigned int v = v0; v < min(count, end_v); v += kAtOnce) {
        float y[kBatch];
        const unsigned int at = begin + v * 32 * VEC;
        Raw<T, VEC> r[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (v + k < count && whole(at + k * 32 * VEC)) r[k].load(row + at + k * 32 * VEC);
          else r[k].clear();
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          float z[VEC];
          r[k].values(z);
          // (the row's first and last 16 bytes, and what lies behind a lane's last vector)
          if (v + k >= count || !whole(at + k * 32 * VEC)) {
            if (v + k < count) some(at + k * 32 * VEC, z);
            else
#pragma unroll
              for (int i = 0; i < VEC; ++i) z[i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[k * VEC + i] = z[i];
        }
        f(y, [&](int e) { return at + (e / VEC) * 32 * VEC + e % VEC - off; });
      }
    }
  }
  // f(logit, index), in the order of the indices of a lane
  template <class F>
  __device__ __forceinline__ void each(F f, unsigned int v0 = 0, unsigned int end_v = 0xffffffffu) const {
    batches([&](const float(&y)[kBatch], auto index) {
#pragma unroll
      for (int e = 0; e < kBatch; ++e) f(y[e], index(e));
    }, v0, end_v);
  }
  // f(logits, index of the first): false ends it, for the whole warp
  template <class F>
  __device__ __forceinline__ void each_vector(F f) const {
    bool go = true;
    if constexpr (E > 0) {
#pragma unroll
      for (int v = 0; v < E / VEC; ++v)
        if (go && v < (int)count) {
          float y[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[i] = x[v * VEC + i];
          go = f(y, begin + v * 32 * VEC - off);
        }
    } else {
      for (unsigned int v = 0; go && v < count; ++v) {
        const unsigned int at = begin + v * 32 * VEC;
        float y[VEC];
        if (whole(at)) Vec<T, VEC>::load(row + at, y);
        else some(at, y);
        go = f(y, at - off);
      }
    }
  }
};

__device__ __forceinline__ void meet(unsigned int parts) {
  if (parts > 1) cg::this_cluster().sync();
  else __syncthreads();
}
__device__ __forceinline__ Share* of_part(Share* sh, unsigned int parts, unsigned int p) { return parts > 1 ? cg::this_cluster().map_shared_rank(sh, p) : sh; }

template <class V, class F>
__device__ __forceinline__ V warp_join(V v, F join) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <class V>
__device__ __forceinline__ V warp_up_to(V v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31u) >= o) v += x;
  }
  return v;
}
// the sum of the threads before this one in the block; `all`: of all of them
__device__ __forceinline__ double block_before(double v, double* scratch, double& all) {
  const double up_to = warp_up_to(v);
  __syncthreads();
  if ((threadIdx.x & 31u) == 31) scratch[threadIdx.x >> 5] = up_to;
  __syncthreads();
  double before = up_to - v;
  all = 0.0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < (int)(threadIdx.x >> 5)) before += scratch[i];
    all += scratch[i];
  }
  return before;
}

// Rising, n of at most kThreads entries, one a thread: pairs of a bitonic network lie in a warp, or, 32 entries and more apart, in shared memory.
__device__ __forceinline__ void sort_few(unsigned long long* list, unsigned int n) {
  const unsigned int n2 = n <= 2 ? 2u : 1u << (32 - __clz((int)n - 1)), i = threadIdx.x;
  __syncthreads();
  unsigned long long r = i < n ? list[i] : ~0ull;
  // (a warp behind the last power of two has nothing to do but to come to the barriers)
  for (unsigned int size = 2; size <= n2; size <<= 1)
    for (unsigned int step = size >> 1; step; step >>= 1) {
      unsigned long long p;
      if (step >= 32) {
        __syncthreads();
        list[i] = r;
        __syncthreads();
        p = list[i ^ step];
      } else {
        if ((threadIdx.x & ~31u) >= n2) continue;
        p = __shfl_xor_sync(0xffffffffu, r, step);
      }
      const bool least = ((i & size) == 0) == ((i & step) == 0);
      r = (p < r) == least ? p : r;
    }
  __syncthreads();
  if (i < n) list[i] = r;
  __syncthreads();
}
// Rising, n of at most kList entries.  A thread has four neighbours: pairs lie in it, in its warp, or, 128 entries and more apart, in shared memory.
__device__ __forceinline__ void sort_list(unsigned long long* list, unsigned int n) {
  if (n <= (unsigned int)kThreads) {
    sort_few(list, n);
    return;
  }
  static_assert(kList == 4 * kThreads, "four entries a thread");
  const unsigned int n2 = n <= 2 ? 2u : 1u << (32 - __clz((int)n - 1)), i0 = threadIdx.x * 4;
  unsigned long long r[4];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) r[k] = i0 + k < n ? list[i0 + k] : ~0ull;
  for (unsigned int size = 2; size <= n2; size <<= 1)
    for (unsigned int step = size >> 1; step; step >>= 1) {
      unsigned long long p[4];
      if (step >= 128) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) list[i0 + k] = r[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = list[(i0 + k) ^ step];
      } else if (step >= 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = __shfl_xor_sync(0xffffffffu, r[k], step >> 2);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = step == 2 ? r[k ^ 2] : r[k ^ 1];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool least = (((i0 + k) & size) == 0) == (((i0 + k) & step) == 0);
        r[k] = (p[k] < r[k]) == least ? p[k] : r[k];
      }
    }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i0 + k < n) list[i0 + k] = r[k];
  __syncthreads();
}
template <class T, int E>
__global__ void __launch_bounds__(kThreads, E == 0 ? 3 : 4) sample_rows(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) Column bins[];      // [warp][bin][lane]
  __shared__ Share sh;
  grid_begin();
  const unsigned int parts = a.parts, part = blockIdx.x % parts, row = blockIdx.x / parts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  constexpr int VEC = Logits<T, E>::VEC;
  const Logits<T, E> logits(a, row, part);
  const float temperature = a.temperatures ? a.temperatures[row] : a.temperature, top_p = a.top_ps ? a.top_ps[row] : a.top_p;
  const float min_p = fmaxf(a.min_ps ? a.min_ps[row] : a.min_p, 0.f), uniform = a.uniform[row];
  const int top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  // binades of weight of a logit (of short rows, while the logits are under way)
  const double log2e = 1.4426950408889634, early_rate = E > 0 ? log2e / (double)temperature : 0.0;
  auto larger = [](auto u, auto v) { return u > v ? u : v; };
  auto smaller = [](auto u, auto v) { return u < v ? u : v; };
  auto add = [](auto u, auto v) { return u + v; };

  // ---- the largest
  float top = -INFINITY;
  logits.each([&](float x, unsigned int) { top = fmaxf(top, x); });
  top = warp_join(top, larger);
  if (lane == 0) sh.scratch[warp] = top;
  if (threadIdx.x == 0) sh.listed = sh.joined = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sh.scratch[i]);
  if (threadIdx.x == 0) sh.largest = top;
  meet(parts);
  // (of all blocks at once: a value of another block is some 700 cycles away)
  if (parts > 1) {
    const float other = lane < parts ? of_part(&sh, parts, lane)->largest : -INFINITY;
    top = warp_join(other, larger);
  }
  top += 0.f;                          // (one zero, whichever lane or block it came from: ends of intervals are made of its bits)
  if (top == -INFINITY) {
    if (part == 0 && threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprob) a.logprob[row] = -INFINITY;
    }
    meet(parts);                       // (nobody leaves while others read of it)
    return;
  }
  if (!(temperature > 0.f)) {
    unsigned int first = 0xffffffffu;
    logits.each([&](float x, unsigned int i) {
      if (x == top) first = min(first, i);
    });
    first = warp_join(first, smaller);
    if (lane == 0) sh.warp_counts[warp] = first;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) first = min(first, sh.warp_counts[i]);
    if (threadIdx.x == 0) sh.first = first;
    meet(parts);
    if (part == 0 && threadIdx.x == 0) {
      for (unsigned int p = 1; p < parts; ++p) first = min(first, of_part(&sh, parts, p)->first);
      a.tokens[row] = (int)first;
      if (a.logprob) a.logprob[row] = 0.f;
    }
    meet(parts);
    return;
  }
  // Binades z below the largest weight: of a few logits in 64 bits, of whole rows in single precision, rounded once, by a rate in two parts: what it is
  // rounded by would move all of a row together against the largest.  (Differences are taken of logits halved where they could be infinite, and multiplied where
  // temperatures are so small that rates could be.  Not of -infinity, which is left out everywhere.)
  const bool endless = top == INFINITY;
  const float factor = top > 1e30f ? 0.5f : temperature < 1e-30f && fabsf(top) <= 1.f ? 1.2676506e30f : 1.f;      // (2^100)
  const double top64 = (double)top, rate = E > 0 ? early_rate : log2e / (double)temperature;
  const double rate_factor = endless ? 1.0 : fmin(factor == 1.f ? rate : factor < 1.f ? rate * 2.0 : rate * 7.888609052210118e-31, 3e38);
  // (what a rate above 2^20 is rounded by is left out, where differences of 2^127 would not go with it)
  const float rate_hi = (float)rate_factor, rate_lo = rate_hi <= 1048576.f ? (float)(rate_factor - (double)rate_hi) : 0.f;
  const float top_factor = endless ? 3.4028235e38f : top * factor;
  // (where the largest is infinite: 0 for those, and 2^126 at least for all others)
  auto difference = [&](float x) -> float { return fmaxf(fmaf(-x, factor, top_factor), 0.f); };
  // (a multiplied difference may be infinite, and what is undefined then as far away)
  auto below = [&](float d) -> float { return fminf(fmaf(d, rate_hi, d * rate_lo), 1e6f); };
  auto weight_at = [&](float z) -> float {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(-z));
    return w;
  };
  auto weight64 = [&](float x) -> double { return endless ? (x == top ? 1.0 : 0.0) : exp2(((double)x - top64) * rate); };

  // the least logit whose weight is min_p: those below are not kept
  float least = -INFINITY;
  if (min_p > 0.f) {
    least = top;
    if (min_p < 1.f && !endless) {
      const double at = top64 + log((double)min_p) * (double)temperature;
      least = (float)at;
      if ((double)least < at) least = of_key(key_of(least) + 1u);
    }
  }

  // ---- the border: kept are logits above it, and those equal to it up to an index
  float border = -INFINITY;
  unsigned int border_to = 0;          // indices of ties below it
  // (without branches, as all that every logit passes)
  auto kept = [&](float x, unsigned int i) { return (x > border) | ((x == border) & (i < border_to)); };
  bool by_count = top_k > 0 && (unsigned int)top_k < a.vocab;
  const bool by_sum = top_p < 1.f;
  const double share = fmax((double)top_p, 0.0);

  // the list that all blocks' entries go to, in the first one: where the histogram was
  unsigned long long* const all_list = E > 0 ? sh.list : (unsigned long long*)bins;

  unsigned int histograms = 0;
  // a histogram of the kept logits that `over` passes on and `of` gives a bin (0: the highest); bins of all blocks, joined, in sh
  // (`fresh`: nothing but -infinity has been left out yet; `weighed`: sums are wanted too; a bin's unit is 2^-unit(bin), its weights are below 1.25 of it; scale_of(bin): 2^17 / unit)
  auto histogram_of = [&](auto fresh, auto weighed, auto over, auto of, auto unit, auto scale_of) {
    const unsigned int set = histograms++ & 1u, b_mine = threadIdx.x / 8, w_mine = threadIdx.x % 8;
    Column* mine = bins + warp * kBins * 32 + lane;
    double s = 0.0;                    // eight threads a bin, a warp's columns each
    unsigned int n = 0;
    // (as many turns as it takes no column more than it counts; the same for all blocks)
    for (unsigned int v0 = 0; v0 < a.span / (32 * VEC); v0 += Logits<T, E>::kCounted) {
      __syncthreads();
      for (unsigned int i = threadIdx.x; i < kWarps * kBins * 32 / 2; i += kThreads) ((uint4*)bins)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      const bool more = over(
          [&](float x, unsigned int i) {
            const float z = below(difference(x));
            const int b = of(x, z);
            // (without branches, but for the last store)
            const unsigned int at = min((unsigned int)b, (unsigned int)kBins - 1u);
            Column v = mine[at * 32];
            if (weighed.value) v.add(weight_at(z) * scale_of((int)at));
            else ++v.sum;
            if ((fresh.value ? x > -INFINITY : kept(x, i)) & ((unsigned int)b < (unsigned int)kBins)) mine[at * 32] = v;
          },
          v0);
      __syncthreads();
      long long sum = 0;
#pragma unroll 4
      for (unsigned int i = 0; i < 32; ++i) {
        const Column v = bins[(w_mine * kBins + b_mine) * 32 + ((i + threadIdx.x) & 31u)];
        n += weighed.value ? v.count() : v.sum;
        if (weighed.value) sum += v.total();
      }
      if (weighed.value) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        s += scalbn((double)sum, -34 - unit((int)b_mine));
      }
      if (!more) break;
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (w_mine == 0) {
      sh.sums[set][b_mine] = s;
      sh.counts[set][b_mine] = n;
    }
    meet(parts);
    if (threadIdx.x < kBins) {
      double s = 0.0, of[kMostParts];
      unsigned int n = 0, in[kMostParts];
#pragma unroll
      for (unsigned int p = 0; p < kMostParts; ++p) {
        const Share* o = of_part(&sh, parts, p < parts ? p : 0);
        of[p] = p < parts ? o->sums[set][threadIdx.x] : 0.0;
        in[p] = p < parts ? o->counts[set][threadIdx.x] : 0u;
      }
#pragma unroll
      for (unsigned int p = 0; p < kMostParts; ++p) {
        s += of[p];
        n += in[p];
      }
      sh.joined_sums[threadIdx.x] = s;
      sh.joined_counts[threadIdx.x] = n;
    }
    __syncthreads();                   // (this set of shares is written again two histograms on, with a meeting between)
  };
  auto histogram = [&](bool weighed, auto over, auto of, auto unit, auto scale_of) {
    if (border == -INFINITY) weighed ? histogram_of(std::true_type(), std::true_type(), over, of, unit, scale_of) : histogram_of(std::true_type(), std::false_type(), over, of, unit, scale_of);
    else weighed ? histogram_of(std::false_type(), std::true_type(), over, of, unit, scale_of) : histogram_of(std::false_type(), std::false_type(), over, of, unit, scale_of);
  };
  // f of the logits of a turn from a lane's vector v0 on; false: there are no more
  auto whole_row = [&](auto f, unsigned int v0) {
    logits.each(f, v0, v0 + Logits<T, E>::kCounted);
    return true;
  };
  // the count and the sum of all bins: a warp, a lane a bin
  auto everything = [&](unsigned int& n, double& s) {
    n = warp_join(sh.joined_counts[lane], add);
    s = __shfl_sync(0xffffffffu, warp_up_to(sh.joined_sums[lane]), 31);
  };
  // the bin in which a count, or a sum, is reached; the last one that holds anything where it never is
  auto find = [&](bool counting, double goal) {
    const unsigned int m = sh.joined_counts[lane];
    const double w = sh.joined_sums[lane];
    const unsigned int n = warp_up_to(m);
    const double s = warp_up_to(w);
    const unsigned int any = __ballot_sync(0xffffffffu, m != 0u), far = __ballot_sync(0xffffffffu, m != 0u && (counting ? (double)n >= goal : s >= goal));
    Pick r;
    r.bin = far ? (unsigned int)__ffs((int)far) - 1u : any ? 31u - (unsigned int)__clz((int)any) : 0u;
    r.in = __shfl_sync(0xffffffffu, m, r.bin);
    r.above = __shfl_sync(0xffffffffu, n, r.bin) - r.in;
    // (not the bin's sum taken off again, which would not give the one before exactly)
    const double before = __shfl_up_sync(0xffffffffu, s, 1);
    r.sum_above = __shfl_sync(0xffffffffu, lane ? before : 0.0, r.bin);
    return r;
  };
  // puts the kept logits that `of` accepts into this block's list
  auto gather_of = [&](auto fresh, auto of) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    logits.batches([&](const auto& y, auto index) {
      unsigned int mask = 0;
#pragma unroll
      for (int e = 0; e < Logits<T, E>::kBatch; ++e) mask |= ((fresh.value ? y[e] > -INFINITY : kept(y[e], index(e))) & of(y[e])) ? 1u << e : 0u;
      if (!__any_sync(0xffffffffu, mask)) return;
      unsigned int at = mask ? atomicAdd(&sh.listed, (unsigned int)__popc((int)mask)) : 0u;
#pragma unroll
      for (int e = 0; e < Logits<T, E>::kBatch; ++e)
        if (mask >> e & 1u) {
          if constexpr (E > 0) {
            if (at < kList) sh.list[at] = (unsigned long long)~key_of(y[e]) << 32 | index(e);
          } else {
            if (at < kLocal) sh.local[at] = index(e);
          }
          ++at;
        }
    });
    __syncthreads();
  };
  auto gather = [&](auto of) {
    if (border == -INFINITY) gather_of(std::true_type(), of);
    else gather_of(std::false_type(), of);
  };
  auto logit_at = [&](unsigned int i) { return to_float(logits.row[logits.off + i]); };
  auto listed_logits = [&](auto f, unsigned int) {
    for (unsigned int k = threadIdx.x; k < sh.listed; k += kThreads) f(logit_at(sh.local[k]), sh.local[k]);
    return false;
  };
  // ... and those of the list that `of` accepts to the list of all blocks, kList in all
  auto send = [&](auto of) {
    if constexpr (E > 0) {
      if (threadIdx.x == 0) sh.joined = sh.listed;
      __syncthreads();
    } else {
      Share* first = of_part(&sh, parts, 0);
      unsigned long long* to = parts > 1 ? cg::this_cluster().map_shared_rank(all_list, 0) : all_list;
      const unsigned int n = min(sh.listed, (unsigned int)kLocal);
      // (a place in another block's list is some 1500 cycles away: one question a warp)
      unsigned long long mine[kLocal / kThreads];
      unsigned int many = 0;
#pragma unroll
      for (int k = 0; k < kLocal / kThreads; ++k) {
        const unsigned int i = threadIdx.x + k * kThreads;
        mine[k] = ~0ull;
        if (i < n) {
          const unsigned int at = sh.local[i];
          const float x = logit_at(at);
          if (of(x)) mine[k] = (unsigned long long)~key_of(x) << 32 | at, ++many;
        }
      }
      const unsigned int up_to = warp_up_to(many);
      unsigned int at = 0;
      if (lane == 31 && up_to) at = atomicAdd(&first->joined, up_to);
      at = __shfl_sync(0xffffffffu, at, 31) + up_to - many;
#pragma unroll
      for (int k = 0; k < kLocal / kThreads; ++k)
        if (mine[k] != ~0ull) {
          if (at < kList) to[at] = mine[k];
          ++at;
        }
      meet(parts);
    }
  };
  auto logit_of = [&](unsigned long long entry) { return of_key(~(unsigned int)(entry >> 32)); };
  // The first n of the sorted list that reach a goal, by count or by sum: each thread has four entries.  `ahead`: the sum ahead of the list
  auto weights_of = [&](unsigned int n, double (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = threadIdx.x * 4 + i < n ? weight64(logit_of(all_list[threadIdx.x * 4 + i])) : 0.0;
    return (w[0] + w[1]) + (w[2] + w[3]);
  };
  auto reach = [&](unsigned int n, double ahead, double goal) {
    double w[4];
    double all;
    const double own = weights_of(n, w);
    double up_to = ahead + block_before(own, sh.block_sums, all);
    unsigned int found = n;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      double s = up_to;
      for (int k = 0; k <= i; ++k) s += w[k];
      if (threadIdx.x * 4 + i < n && s >= goal) found = threadIdx.x * 4 + i + 1;
    }
    found = warp_join(found, smaller);
    __syncthreads();
    if (lane == 0) sh.warp_counts[warp] = found;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) found = min(found, sh.warp_counts[i]);
    return max(found, 1u);
  };
  auto sum_of = [&](unsigned int n) {
    double w[4];
    double all;
    block_before(weights_of(n, w), sh.block_sums, all);
    return all;
  };

  if (by_count || by_sum) {
    bool listed = false;               // the list holds all that may be kept
    double total = 0.0;                // of all logits' weights
    // (half a binade a bin, rounded to the nearest by an addition)
    auto level_at = [&](float z) { return (int)min(__float_as_uint(fmaf(z, 2.f, 8388608.f)) - 0x4b000000u, (unsigned int)(kBins - 1)); };
    auto level = [&](float x) { return level_at(below(difference(x))); };
    auto by_level = [&](float, float z) { return level_at(z); };
    auto level_unit = [](int b) { return b >> 1; };       // (z >= bin / 2 - 1/4)
    auto level_scale = [](int b) { return __uint_as_float(((unsigned int)b << 22 & 0x07800000u) | 0x48000000u); };
    Pick at = {0, 0, 0, 0.0};
    if (E > 0 || a.vocab <= kList) {
      gather([](float) { return true; });
      send([](float) { return true; });
      listed = true;
    } else {
      unsigned int n;
      if (by_count) {
        histogram(false, whole_row, by_level, level_unit, level_scale);
        everything(n, total);
        by_count = (unsigned int)top_k < n;
      }
      if (!by_count && by_sum) {
        histogram(true, whole_row, by_level, level_unit, level_scale);
        everything(n, total);
      }
      if (by_count || by_sum) {
        at = find(by_count, by_count ? (double)top_k : share * total);
        if (at.above + at.in <= kList) {
          const int last = (int)at.bin;
          gather([&](float x) { return level(x) <= last; });
          send([](float) { return true; });
          listed = true;
        }
      }
    }
    if (listed) {
      // ---- one block does the rest
      if (part != 0) return;
      unsigned int n = min(sh.joined, (unsigned int)kList);
      sort_list(all_list, n);
      if (by_count) n = min(n, (unsigned int)top_k);
      if (by_sum) n = reach(n, 0.0, share * (by_count || E > 0 || a.vocab <= kList ? sum_of(n) : total));
      double w[4];
      weights_of(n, w);
      // those above the least weight; in the order of the indices
      unsigned int here = 0;
      unsigned long long entry[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned int k = threadIdx.x * 4 + i;
        entry[i] = k < n ? all_list[k] : 0ull;
        const bool on = k < n && w[i] > 0.0 && logit_of(entry[i]) >= least;
        entry[i] = on ? entry[i] << 32 | entry[i] >> 32 : ~0ull;
        here += on;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (threadIdx.x * 4 + i < n) all_list[threadIdx.x * 4 + i] = entry[i];
      here = warp_join(here, add);
      if (lane == 0) sh.warp_counts[warp] = here;
      __syncthreads();
      here = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) here += sh.warp_counts[i];
      sort_list(all_list, n);
      double all, up_to = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned int k = threadIdx.x * 4 + i;
        w[i] = k < here ? weight64(of_key(~(unsigned int)all_list[k])) : 0.0;
        up_to += w[i];
      }
      up_to = block_before(up_to, sh.block_sums, all);
      const double goal = (uniform > 0.f ? (double)uniform : 0.0) * all;
      unsigned int found = here - 1;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        double s = up_to;
        for (int k = 0; k <= i; ++k) s += w[k];
        if (threadIdx.x * 4 + i < here && s > goal) found = min(found, threadIdx.x * 4 + i);
      }
      found = warp_join(found, smaller);
      __syncthreads();
      if (lane == 0) sh.warp_counts[warp] = found;
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int i = 0; i < kWarps; ++i) found = min(found, sh.warp_counts[i]);
        const unsigned long long e = all_list[found];
        a.tokens[row] = (int)(unsigned int)(e >> 32);
        if (a.logprob) a.logprob[row] = (float)log(weight64(of_key(~(unsigned int)e)) / all);
      }
      return;
    }
    // ---- the border by count, then by sum, over the whole row
    for (int which = by_count ? 0 : 1; which < (by_sum ? 2 : 1); ++which) {
      const bool counting = which == 0;
      double goal = (double)top_k;
      if (!counting) {
        if (by_count) {
          histogram(true, whole_row, by_level, level_unit, level_scale);
          unsigned int n;
          everything(n, total);
        }
        goal = share * total;
        at = find(false, goal);
      }
      // The logits of the bin, as an interval of keys: where the bin's number changes (it never rises with the logit).  A warp an end, 32 keys at a time.
      if (warp < 2) {
        const int bin = (int)at.bin - (int)warp;                         // the least key of a bin up to this one (none: one behind the largest)
        unsigned int l = key_of(-INFINITY) + 1, h = key_of(top) + (bin < 0);
        if (bin < 0) l = h;
        while (l < h) {
          const unsigned int step = (h - l) / 32 + 1, most = h - l, k = l + min(lane * step, most);
          const unsigned int yes = __ballot_sync(0xffffffffu, level(of_key(k)) <= bin), n = yes ? (unsigned int)__ffs((int)yes) - 1u : 32u;
          const unsigned int from = l;
          if (n) l = from + min((n - 1u) * step, most) + 1u;             // (lanes before the first have a higher one)
          if (n < 32u) h = from + min(n * step, most);
        }
        if (lane == 0) sh.interval[warp] = h - warp;
      }
      __syncthreads();
      unsigned int lo = sh.interval[0], hi = sh.interval[1];
      unsigned int above = at.above;
      double sum_above = at.sum_above;
      bool have = false;               // the blocks' lists hold the interval
      // (no logit has the key of -0, so that an interval may end ahead of it: then, and only then, floats lie inside where their keys do)
      auto inside = [&](float x) { return (x >= of_key(lo)) & (x <= of_key(hi)); };
      for (;;) {
        // (where the lists are likely to hold it; an uneven row is passed again)
        if (!have && (at.in <= kList || (lo < hi && at.in <= kLocal * parts / 4 * 3))) {
          gather(inside);
          meet(parts);
          have = true;
          have = __all_sync(0xffffffffu, lane >= parts || of_part(&sh, parts, lane)->listed <= kLocal);
          meet(parts);
        }
        // (a few hundred are divided sooner than sorted, where no pass over the row is needed for it)
        if (at.in <= (have ? kList / 4 : kList) || lo == hi) break;
        int bits = 0;
        while ((hi - lo) >> bits >= kBins) ++bits;
        auto split = [&](float x, float) { return inside(x) ? (int)((hi - key_of(x)) >> bits) : -1; };
        const int most = (int)fminf(below(difference(of_key(hi))), 100.f);     // (weights from 2^-126 on are 0)
        auto unit = [&](int) { return most; };
        auto scale_of = [&](int) { return __uint_as_float(((unsigned int)most << 23) + 0x48000000u); };
        if (have) histogram(!counting, listed_logits, split, unit, scale_of);
        else histogram(!counting, whole_row, split, unit, scale_of);
        at = find(counting, counting ? goal - above : goal - sum_above);
        above += at.above;
        sum_above += at.sum_above;
        const unsigned int cut = hi - (at.bin << bits);
        lo = cut - lo < (1u << bits) ? lo : cut - (1u << bits) + 1;
        hi = cut - (cut == 0x7fffffffu);
      }
      if (at.in <= kList) {
        send(inside);
        if (part == 0) {
          const unsigned int n = min(sh.joined, (unsigned int)kList);
          sort_list(all_list, n);
          const unsigned int many = counting ? min(max((unsigned int)top_k - above, 1u), n) : reach(n, sum_above, goal);
          if (threadIdx.x == 0) {
            const unsigned long long e = all_list[many - 1];
            sh.border = logit_of(e);
            sh.border_at = (unsigned int)e;
            sh.joined = 0;
          }
        }
        meet(parts);
        border = of_part(&sh, parts, 0)->border;
        border_to = of_part(&sh, parts, 0)->border_at + 1u;
        meet(parts);
      } else {
        // many equal ones: as many as are wanted of them, in the order of their indices
        const float value = of_key(lo);
        const double w = (double)weight_at(below(difference(value))), need = counting ? goal - above : w > 0.0 ? ceil((goal - sum_above) / w) : 1.0;
        unsigned int want = need < 1.0 ? 1u : need > (double)at.in ? at.in : (unsigned int)need, ties = 0;
        logits.each([&](float x, unsigned int i) { ties += x == value && kept(x, i); });
        ties = warp_join(ties, add);
        if (lane == 0) sh.warp_counts[warp] = ties;
        meet(parts);
        unsigned int before = 0;       // those of the warps ahead of this one
        for (unsigned int p = 0; p <= part; ++p)
          for (unsigned int i = 0; i < (p < part ? (unsigned int)kWarps : warp); ++i) before += of_part(&sh, parts, p)->warp_counts[i];
        if (before < want && want <= before + ties) {
          logits.each_vector([&](const float(&y)[VEC], unsigned int first) {
            unsigned int mine = 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) mine += y[i] == value && kept(y[i], first + i);
            const unsigned int up_to = warp_up_to(mine), all = __shfl_sync(0xffffffffu, up_to, 31);
            if (want > before + all) {
              before += all;
              return true;
            }
            unsigned int k = before + up_to - mine;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              if (y[i] == value && kept(y[i], first + i) && ++k == want) of_part(&sh, parts, 0)->border_at = first + i;
            return false;
          });
        }
        meet(parts);
        border = value;
        border_to = of_part(&sh, parts, 0)->border_at + 1u;
        meet(parts);
      }
    }
  }

  // ---- the token: in which warp the running sum passes the goal, then where in it
  if (least > border) {
    const unsigned int k = key_of(least) - 1u;
    border = of_key(k - (k == 0x7fffffffu));             // (not -0, which equals 0)
    border_to = 0;
  }
  auto chance = [&](float x, unsigned int i) -> float {
    const float w = weight_at(below(difference(x)));
    return kept(x, i) ? w : 0.f;
  };
  double mine = 0.0;
  logits.batches([&](const auto& y, auto index) {
    // (by halves, which adds equal weights exactly)
    float some[Logits<T, E>::kBatch];
#pragma unroll
    for (int e = 0; e < Logits<T, E>::kBatch; ++e) some[e] = chance(y[e], index(e));
#pragma unroll
    for (int h = Logits<T, E>::kBatch / 2; h > 0; h >>= 1)
#pragma unroll
      for (int e = 0; e < h; ++e) some[e] += some[e + h];
    mine += (double)some[0];
  });
  mine = warp_join(mine, add);
  if (lane == 0) sh.warp_sums[warp] = mine;
  meet(parts);
  // two warps' sums a lane, and where they end; all warps count the same way
  double two[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned int w = 2 * lane + k;
    two[k] = w < parts * kWarps ? of_part(&sh, parts, w / kWarps)->warp_sums[w % kWarps] : 0.0;
  }
  const double up_to = warp_up_to(two[0] + two[1]), up_to_before = __shfl_up_sync(0xffffffffu, up_to, 1), ahead = lane ? up_to_before : 0.0, middle = ahead + two[0];
  const double total = __shfl_sync(0xffffffffu, up_to, 31), goal = (uniform > 0.f ? (double)uniform : 0.0) * total;
  // the first that passes the goal, or the last that has any
  unsigned int which = warp_join(two[0] > 0.0 && middle > goal ? 2 * lane : two[1] > 0.0 && up_to > goal ? 2 * lane + 1u : 0xffffffffu, smaller);
  const unsigned int last_any = warp_join(two[1] > 0.0 ? 2 * lane + 1u : two[0] > 0.0 ? 2 * lane : 0u, larger);
  if (which == 0xffffffffu) which = last_any;
  const double even = __shfl_sync(0xffffffffu, ahead, which / 2), odd = __shfl_sync(0xffffffffu, middle, which / 2);
  double before = which & 1u ? odd : even;
  const bool owner = part * kWarps + warp == which;
  if (owner) {
    unsigned int last = 0xffffffffu, found = 0xffffffffu;
    logits.each_vector([&](const float(&y)[VEC], unsigned int first) {
      double own = 0.0;
      float w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        w[i] = chance(y[i], first + i);
        own += (double)w[i];
        if (w[i] > 0.f) last = first + i;
      }
      const double up_to = warp_up_to(own), all = __shfl_sync(0xffffffffu, up_to, 31);
      if (before + all > goal) {
        double s = before + up_to - own;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s += (double)w[i];
          if (found == 0xffffffffu && w[i] > 0.f && s > goal) found = first + i;
        }
        if (__any_sync(0xffffffffu, found != 0xffffffffu)) return false;
      }
      before += all;
      return true;
    });
    unsigned int chosen = warp_join(found, smaller);
    if (chosen == 0xffffffffu) {
      // (rounding: the last of the warp)
      chosen = warp_join(last == 0xffffffffu ? 0u : last + 1u, larger) - 1u;
      found = last;
    }
    if (found == chosen) {
      a.tokens[row] = (int)found;
      if (a.logprob) a.logprob[row] = (float)log(weight64(logit_at(found)) / total);
    }
  }
  meet(parts);
}

typedef void (*SampleKernel)(const SampleArgs);

struct SampleOperator : b200_operator {
  SampleArgs a = {};
  SampleKernel kernel = nullptr;
  size_t smem = 0;

  template <class T>
  void choose() {
    constexpr unsigned int V = 16 / (unsigned int)sizeof(T), piece = 32 * V;
    // Rows of up to a list's length lie in registers, a block each.  Longer ones are read again in every pass, from L2, by up to eight blocks of 2048 logits
    // at least, seven blocks an SM: more of them wait for one another more often than the shorter passes gain (256 rows of 131072 logits: 1, 2, 4, 8 blocks
    // a row take 339, 207, 188, 228 us).
    const unsigned int n = a.vocab;
    const bool small = n + V <= (unsigned int)kList;
    const auto blocks = [&](unsigned long long each) { return (n + each - 1) / each; };
    a.parts = small ? 1u : (unsigned int)std::max(1ull, std::min(std::min((unsigned long long)kMostParts, blocks(2048)), 7ull * (unsigned int)dev->sm_count / a.rows));
    a.span = small ? 32u * 8u : (unsigned int)(((unsigned long long)n + V + a.parts * kWarps * piece - 1) / (a.parts * kWarps * piece) * piece);
    kernel = small ? sample_rows<T, 8> : sample_rows<T, 0>;
    smem = small ? 0 : (size_t)kWarps * kBins * 32 * 8;
    ready(kernel, smem);
  }
  void run(cudaStream_t s) override {
    if (!a.rows) return;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * a.parts);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.parts > 1 ? 2 : 1;
    rt_check(cudaLaunchKernelEx(&cfg, kernel, a), "operator launch");
    ++operator_launches;
  }
};

}  // namespace

extern "C" int b200_sample_link(b200_dev* dev, const b200_sample* p, b200_operator** out) {
  return link_operator<SampleOperator>(dev, p, out, [&](SampleOperator* op) {
    Operands ops(op, "sample");
    ops.dtype(p->dtype);
    if (p->rows < 0 || p->rows > (1ll << 30)) ops.refuse("rows must be between 0 and 2^30");
    if (p->vocab < 1 || p->vocab > 0x7fffffffll) ops.refuse("vocab must be between 1 and 2^31 - 1");
    if (std::isnan(p->temperature) || std::isnan(p->top_p) || std::isnan(p->min_p)) ops.refuse("a setting is undefined");
    const unsigned long long rows = (unsigned long long)p->rows;
    SampleArgs& a = op->a;
    a.x = (const void*)ops.in(p->logits, "logits", extent_product({p->rows, p->vocab}, "sample"), dtype_bytes(p->dtype));
    a.uniform = (const float*)ops.in(p->uniform, "uniform", rows, 4);
    a.temperatures = (const float*)ops.in(p->temperatures, "temperatures", rows, 4, false);
    a.top_ps = (const float*)ops.in(p->top_ps, "top_ps", rows, 4, false);
    a.min_ps = (const float*)ops.in(p->min_ps, "min_ps", rows, 4, false);
    a.top_ks = (const int*)ops.in(p->top_ks, "top_ks", rows, 4, false);
    a.tokens = (int*)ops.out(p->tokens, "tokens", rows, 4);
    a.logprob = (float*)ops.out(p->logprob, "logprob", rows, 4, false);
    ops.check_overlaps();
    a.rows = (unsigned int)p->rows;
    a.vocab = (unsigned int)p->vocab;
    a.temperature = p->temperature;
    a.top_p = p->top_p;
    a.min_p = p->min_p;
    a.top_k = p->top_k;
    if (!a.rows) return;
    if (p->dtype == B200_F32) op->choose<float>();
    else if (p->dtype == B200_BF16) op->choose<__nv_bfloat16>();
    else op->choose<__half>();
    if ((unsigned long long)a.rows * a.parts >> 31) ops.refuse("too many rows", B200_E_UNSUPPORTED);
  });
}
