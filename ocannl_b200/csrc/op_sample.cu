// Choosing a token for each row of logits (b200_sample_link).
//
//   w_i = exp((x_i - max) / T);  kept: the first n in the order of falling x, of rising i among equal ones;  token: where the running sum of the kept, in the
//   order of i, passes uniform * its end
//
// Bound by memory: a row is read once, and again from L2 in two or three more passes.  A cluster of up to eight blocks takes it and exchanges sums through
// shared memory.  What is kept is all logits above a border and, of those equal to it, the ones up to an index: no sort of the row.  The border is found by a
// histogram of 32 bins, half a binade of weight each, of counts and sums of weights; every lane has columns of its own, so that nothing is added atomically and
// sums come out the same every time.  A bin that bounds what is kept, with all above it, is usually a few hundred logits: these go to one block, which
// sorts them and does the rest.  Where they are more than 1024, the bin is divided again by the bits of its logits, until it is small or of one value,
// and the row is passed once more for the token.  Weights are summed in double precision beyond a lane's, so that borders lie where they do in 64 bits but
// for 2^-22 of a weight.
#include <cooperative_groups.h>

#include <cmath>

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

constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 32, kList = 1024, kMostParts = 8;

// rises with the value
__device__ __forceinline__ unsigned int key_of(float x) {
  const unsigned int u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned int k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Share {                         // of a block, for the others of its cluster to read
  unsigned long long list[kList];      // of the first block: what is sorted
  double sums[kBins];
  unsigned int counts[kBins];
  double warp_sums[kWarps];
  unsigned int warp_counts[kWarps];
  float largest;
  unsigned int first;                  // an index
  unsigned int listed;                 // entries of the list
  float border;                        // what the first block has found: the last logit that is kept, and its index
  unsigned int border_at;
  float scratch[kWarps];
  double joined_sums[kBins];           // over all blocks
  unsigned int joined_counts[kBins];
  double block_sums[kWarps];
};

struct Pick {                          // a histogram's bin
  unsigned int bin, above, in;         // logits above it, and in it
  double sum_above;
};

// The row as the blocks of its cluster hold it: E logits a thread in registers (0: they are read from memory every time), VEC neighbours a lane, a warp's
// all in one piece.
template <class T, int E, int VEC>
struct Logits {
  float x[E ? E : VEC];
  const T* row;
  unsigned int n, begin, lane, count;  // begin: of this lane's first vector; count: vectors of a lane (in memory)
  __device__ __forceinline__ void fetch(unsigned int at, float* v) const {
    if (at + VEC <= n) Vec<T, VEC>::load(row + at, v);
    else
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = at + i < n ? to_float(row[at + i]) : -INFINITY;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = v[i] != v[i] ? -INFINITY : v[i] + 0.f;       // (undefined ones count as none; one zero)
  }
  __device__ __forceinline__ Logits(const SampleArgs& a, unsigned int r, unsigned int part) {
    row = (const T*)a.x + (unsigned long long)r * a.vocab;
    n = a.vocab;
    lane = threadIdx.x & 31u;
    // (beyond 2^32 a warp has nothing)
    const unsigned long long from = (unsigned long long)(part * kWarps + (threadIdx.x >> 5)) * a.span;
    begin = (unsigned int)min(from, (unsigned long long)n) + lane * VEC;
    count = from < n ? (unsigned int)((min((unsigned long long)a.span, n - from) + 32 * VEC - 1) / (32 * VEC)) : 0u;
    if constexpr (E > 0) {
#pragma unroll
      for (int v = 0; v < E / VEC; ++v) {
        if (v < (int)count) fetch(begin + v * 32 * VEC, x + v * VEC);
        else
#pragma unroll
          for (int i = 0; i < VEC; ++i) x[v * VEC + i] = -INFINITY;
      }
    }
  }
  // f(logit, index), in the order of the indices of a lane
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(x[e], begin + (e / VEC) * 32 * VEC + e % VEC);
    } else {
      for (unsigned int v = 0; v < count; ++v) {
        float y[VEC];
        fetch(begin + v * 32 * VEC, y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f(y[i], begin + v * 32 * VEC + i);
      }
    }
  }
  // f(logits, index of the first): false ends it, for the whole warp
  template <class F>
  __device__ __forceinline__ void each_vector(F f) const {
    if constexpr (E > 0) {
      bool go = true;
#pragma unroll
      for (int v = 0; v < E / VEC; ++v)
        if (go && v < (int)count) {
          float y[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[i] = x[v * VEC + i];
          go = f(y, begin + v * 32 * VEC);
        }
    } else {
      bool go = true;
      for (unsigned int v = 0; go && v < count; ++v) {
        float y[VEC];
        fetch(begin + v * 32 * VEC, y);
        go = f(y, begin + v * 32 * VEC);
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

// rising; entries n .. n2 - 1 are filled here, n2 a power of two
__device__ __forceinline__ void sort_list(unsigned long long* list, unsigned int n, unsigned int n2) {
  for (unsigned int i = n + threadIdx.x; i < n2; i += kThreads) list[i] = ~0ull;
  __syncthreads();
  for (unsigned int size = 2; size <= n2; size <<= 1)
    for (unsigned int step = size >> 1; step; step >>= 1) {
      for (unsigned int t = threadIdx.x; t < n2 / 2; t += kThreads) {
        const unsigned int i = (t / step) * 2 * step + t % step, j = i + step;
        const unsigned long long u = list[i], v = list[j];
        if ((u > v) == ((i & size) == 0)) {
          list[i] = v;
          list[j] = u;
        }
      }
      // (a warp's 32 pairs lie in 64 entries of their own once they are less than 64 apart)
      if (step > 32 || n2 > 64 * kWarps) __syncthreads();
      else if (step == 1) __syncthreads();
      else __syncwarp();
    }
}
__device__ __forceinline__ unsigned int power_above(unsigned int n) { return n <= 2 ? 2u : 1u << (32 - __clz((int)n - 1)); }

template <class T, int E, int VEC>
__global__ void __launch_bounds__(kThreads, E == 0 ? 3 : 4) sample_rows(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint2 bins[];       // [warp][bin][lane]: sum of weights, count
  __shared__ Share sh;
  grid_begin();
  const unsigned int parts = a.parts, part = blockIdx.x % parts, row = blockIdx.x / parts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const Logits<T, E, VEC> logits(a, row, part);
  const float temperature = a.temperatures ? a.temperatures[row] : a.temperature, top_p = a.top_ps ? a.top_ps[row] : a.top_p;
  const float min_p = a.min_ps ? a.min_ps[row] : a.min_p, uniform = a.uniform[row];
  const int top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  auto larger = [](auto u, auto v) { return u > v ? u : v; };
  auto smaller = [](auto u, auto v) { return u < v ? u : v; };
  auto add = [](auto u, auto v) { return u + v; };

  // ---- the largest
  float top = -INFINITY;
  logits.each([&](float x, unsigned int) { top = fmaxf(top, x); });
  top = warp_join(top, larger);
  if (lane == 0) sh.scratch[warp] = top;
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sh.scratch[i]);
  if (threadIdx.x == 0) sh.largest = top;
  meet(parts);
  for (unsigned int p = 0; p < parts; ++p) top = fmaxf(top, of_part(&sh, parts, p)->largest);
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
  // (never zero, so that -infinity stays that)
  const float rate = fmaxf((float)(1.4426950408889634 / (double)temperature), 1e-37f);
  const bool endless = top == INFINITY;
  auto below = [&](float x) -> float { return x == top ? 0.f : endless ? INFINITY : (top - x) * rate; };      // binades below the largest weight
  auto weight = [&](float x) -> float {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(-below(x)));
    return w;
  };

  // ---- the border: kept are logits above it, and those equal to it up to an index
  float border = -INFINITY;
  unsigned int border_at = 0xffffffffu;
  auto kept = [&](float x, unsigned int i) { return x > border || (x == border && i <= border_at && x != -INFINITY); };
  bool by_count = top_k > 0 && (unsigned int)top_k < a.vocab;
  const bool by_sum = top_p < 1.f;
  const double share = fmax((double)top_p, 0.0);

  // a histogram of the kept logits that `of` gives a bin (0: the highest); bins of all blocks, joined, in sh
  auto histogram = [&](auto of) {
    for (unsigned int i = threadIdx.x; i < kWarps * kBins * 32 / 2; i += kThreads) ((uint4*)bins)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    uint2* mine = bins + warp * kBins * 32 + lane;
    logits.each([&](float x, unsigned int i) {
      if (!kept(x, i)) return;
      const int b = of(x);
      if (b < 0) return;
      uint2 v = mine[b * 32];
      v.x = __float_as_uint(__uint_as_float(v.x) + weight(x));
      ++v.y;
      mine[b * 32] = v;
    });
    __syncthreads();
    // eight threads a bin, a warp's columns each
    {
      const unsigned int b = threadIdx.x / 8, w = threadIdx.x % 8;
      double s = 0.0;
      unsigned int n = 0;
#pragma unroll 4
      for (unsigned int i = 0; i < 32; ++i) {
        const uint2 v = bins[(w * kBins + b) * 32 + ((i + threadIdx.x) & 31u)];
        s += (double)__uint_as_float(v.x);
        n += v.y;
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
      }
      if (w == 0) {
        sh.sums[b] = s;
        sh.counts[b] = n;
      }
    }
    meet(parts);
    if (threadIdx.x < kBins) {
      double s = 0.0;
      unsigned int n = 0;
      for (unsigned int p = 0; p < parts; ++p) {
        const Share* o = of_part(&sh, parts, p);
        s += o->sums[threadIdx.x];
        n += o->counts[threadIdx.x];
      }
      sh.joined_sums[threadIdx.x] = s;
      sh.joined_counts[threadIdx.x] = n;
    }
    meet(parts);                       // (the shares are written again)
  };
  // the bin in which a count, or a sum, is reached; the last one that holds anything where it never is
  auto find = [&](bool counting, double goal) {
    Pick r = {0, 0, 0, 0.0};
    unsigned int n = 0;
    double s = 0.0;
    for (unsigned int b = 0; b < kBins; ++b) {
      const unsigned int m = sh.joined_counts[b];
      if (!m) continue;
      r.bin = b;
      r.above = n;
      r.in = m;
      r.sum_above = s;
      n += m;
      s += sh.joined_sums[b];
      if (counting ? (double)n >= goal : s >= goal) break;
    }
    return r;
  };
  // puts the kept logits that `of` accepts into the first block's list
  auto gather = [&](auto of) {
    unsigned int n = 0;
    logits.each([&](float x, unsigned int i) { n += kept(x, i) && of(x); });
    const unsigned int up_to = warp_up_to(n);
    unsigned int at = 0;
    Share* first = of_part(&sh, parts, 0);
    if (lane == 31 && up_to) at = atomicAdd(&first->listed, up_to);
    at = __shfl_sync(0xffffffffu, at, 31) + up_to - n;
    if (n)
      logits.each([&](float x, unsigned int i) {
        if (!kept(x, i) || !of(x)) return;
        if (at < kList) first->list[at] = (unsigned long long)~key_of(x) << 32 | i;
        ++at;
      });
    meet(parts);
  };
  auto logit_of = [&](unsigned long long entry) { return of_key(~(unsigned int)(entry >> 32)); };
  // The first n of the sorted list that reach a goal, by count or by sum: each thread has four entries.  `ahead`: the sum ahead of the list
  auto weights_of = [&](unsigned int n, float (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = threadIdx.x * 4 + i < n ? weight(logit_of(sh.list[threadIdx.x * 4 + i])) : 0.f;
    return ((double)w[0] + w[1]) + ((double)w[2] + w[3]);
  };
  auto reach = [&](unsigned int n, double ahead, double goal) {
    float w[4];
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
    float w[4];
    double all;
    block_before(weights_of(n, w), sh.block_sums, all);
    return all;
  };

  if (by_count || by_sum) {
    bool listed = false;               // the list holds all that may be kept
    double total = 0.0;                // of all logits' weights
    auto level = [&](float x) { return min((int)(below(x) * 2.f), kBins - 1); };
    Pick at = {0, 0, 0, 0.0};
    if (a.vocab <= kList) {
      gather([](float) { return true; });
      listed = true;
    } else {
      histogram(level);
      unsigned int n = 0;
      for (int b = 0; b < kBins; ++b) n += sh.joined_counts[b], total += sh.joined_sums[b];
      by_count = by_count && (unsigned int)top_k < n;
      if (by_count || by_sum) {
        at = find(by_count, by_count ? (double)top_k : share * total);
        if (at.above + at.in <= kList) {
          const int last = (int)at.bin;
          gather([&](float x) { return level(x) <= last; });
          listed = true;
        }
      }
    }
    if (listed) {
      // ---- one block does the rest
      if (part != 0) return;
      unsigned int n = min(sh.listed, (unsigned int)kList);
      sort_list(sh.list, n, power_above(n));
      if (by_count) n = min(n, (unsigned int)top_k);
      if (by_sum) n = reach(n, 0.0, share * (by_count || a.vocab <= kList ? sum_of(n) : total));
      float w[4];
      weights_of(n, w);
      // those above the least weight; in the order of the indices
      unsigned int here = 0;
      unsigned long long entry[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned int k = threadIdx.x * 4 + i;
        entry[i] = k < n ? sh.list[k] : 0ull;
        const bool on = k < n && w[i] > 0.f && (w[i] >= min_p || logit_of(entry[i]) == top);
        entry[i] = on ? entry[i] << 32 | entry[i] >> 32 : ~0ull;
        here += on;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (threadIdx.x * 4 + i < n) sh.list[threadIdx.x * 4 + i] = entry[i];
      here = warp_join(here, add);
      if (lane == 0) sh.warp_counts[warp] = here;
      __syncthreads();
      here = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) here += sh.warp_counts[i];
      sort_list(sh.list, n, power_above(n));
      double all, up_to = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned int k = threadIdx.x * 4 + i;
        w[i] = k < here ? weight(of_key(~(unsigned int)sh.list[k])) : 0.f;
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
        const unsigned long long e = sh.list[found];
        a.tokens[row] = (int)(unsigned int)(e >> 32);
        if (a.logprob) a.logprob[row] = (float)log((double)weight(of_key(~(unsigned int)e)) / all);
      }
      return;
    }
    // ---- the border by count, then by sum, over the whole row
    for (int which = by_count ? 0 : 1; which < (by_sum ? 2 : 1); ++which) {
      const bool counting = which == 0;
      double goal = (double)top_k;
      if (!counting) {
        if (by_count) {
          histogram(level);
          total = 0.0;
          for (int b = 0; b < kBins; ++b) total += sh.joined_sums[b];
        }
        goal = share * total;
        at = find(false, goal);
      }
      // the logits of the bin, as an interval of keys: where the bin's number changes (it never rises with the logit)
      unsigned int lo = key_of(-INFINITY) + 1, hi = key_of(top);
      {
        unsigned int l = lo, h = hi;
        while (l < h) {                // the least key of a bin up to this one
          const unsigned int mid = l + (h - l) / 2;
          if (level(of_key(mid)) <= (int)at.bin) h = mid;
          else l = mid + 1;
        }
        const unsigned int least = l;
        l = least, h = hi;
        while (l < h) {                // the largest of this one
          const unsigned int mid = h - (h - l) / 2;
          if (level(of_key(mid)) >= (int)at.bin) l = mid;
          else h = mid - 1;
        }
        lo = least;
        hi = l;
      }
      unsigned int above = at.above;
      double sum_above = at.sum_above;
      while (at.in > kList && lo < hi) {
        int bits = 0;
        while ((hi - lo) >> bits >= kBins) ++bits;
        const unsigned int l = lo, h = hi;
        histogram([&](float x) {
          const unsigned int k = key_of(x);
          return k < l || k > h ? -1 : (int)((h - k) >> bits);
        });
        at = find(counting, counting ? goal - above : goal - sum_above);
        above += at.above;
        sum_above += at.sum_above;
        const unsigned int cut = h - (at.bin << bits);
        lo = cut - l < (1u << bits) ? l : cut - (1u << bits) + 1;
        hi = cut;
      }
      if (at.in <= kList) {
        const unsigned int l = lo, h = hi;
        gather([&](float x) {
          const unsigned int k = key_of(x);
          return k >= l && k <= h;
        });
        if (part == 0) {
          const unsigned int n = min(sh.listed, (unsigned int)kList);
          sort_list(sh.list, n, power_above(n));
          const unsigned int many = counting ? min(max((unsigned int)top_k - above, 1u), n) : reach(n, sum_above, goal);
          if (threadIdx.x == 0) {
            const unsigned long long e = sh.list[many - 1];
            sh.border = logit_of(e);
            sh.border_at = (unsigned int)e;
            sh.listed = 0;
          }
        }
        meet(parts);
        border = of_part(&sh, parts, 0)->border;
        border_at = of_part(&sh, parts, 0)->border_at;
        meet(parts);
      } else {
        // many equal ones: as many as are wanted of them, in the order of their indices
        const float value = of_key(lo);
        const double w = (double)weight(value), need = counting ? goal - above : w > 0.0 ? ceil((goal - sum_above) / w) : 1.0;
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
        border_at = of_part(&sh, parts, 0)->border_at;
        meet(parts);
      }
    }
  }

  // ---- the token: in which warp the running sum passes the goal, then where in it
  auto chance = [&](float x, unsigned int i) -> float {
    if (!kept(x, i)) return 0.f;
    const float w = weight(x);
    return w >= min_p || x == top ? w : 0.f;
  };
  double mine = 0.0;
  logits.each([&](float x, unsigned int i) { mine += (double)chance(x, i); });
  mine = warp_join(mine, add);
  if (lane == 0) sh.warp_sums[warp] = mine;
  meet(parts);
  double total = 0.0, before = 0.0;
  unsigned int last_any = 0;           // the last warp that has any
  for (unsigned int p = 0; p < parts; ++p)
    for (unsigned int i = 0; i < kWarps; ++i) {
      if (p == part && i == warp) before = total;
      const double s = of_part(&sh, parts, p)->warp_sums[i];
      if (s > 0.0) last_any = p * kWarps + i;
      total += s;
    }
  const double goal = (uniform > 0.f ? (double)uniform : 0.0) * total;
  const bool owner = goal < total ? before <= goal && before + mine > goal : part * kWarps + warp == last_any;
  if (owner) {
    unsigned int last = 0xffffffffu, found = 0xffffffffu;
    float last_w = 0.f, found_w = 0.f;
    logits.each_vector([&](const float(&y)[VEC], unsigned int first) {
      double own = 0.0;
      float w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        w[i] = chance(y[i], first + i);
        own += (double)w[i];
        if (w[i] > 0.f) last = first + i, last_w = w[i];
      }
      const double up_to = warp_up_to(own), all = __shfl_sync(0xffffffffu, up_to, 31);
      if (before + all > goal) {
        double s = before + up_to - own;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s += (double)w[i];
          if (found == 0xffffffffu && w[i] > 0.f && s > goal) found = first + i, found_w = w[i];
        }
        if (__any_sync(0xffffffffu, found != 0xffffffffu)) return false;
      }
      before += all;
      return true;
    });
    unsigned int least = warp_join(found, smaller);
    if (least == 0xffffffffu) {
      // (rounding: the last of the warp)
      least = warp_join(last == 0xffffffffu ? 0u : last + 1u, larger) - 1u;
      found = last;
      found_w = last_w;
    }
    if (found == least) {
      a.tokens[row] = (int)found;
      if (a.logprob) a.logprob[row] = (float)log((double)found_w / total);
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
  void choose(bool vec) {
    constexpr int V = 16 / (int)sizeof(T);
    // Rows of up to a list's length lie in registers, a block each.  Longer ones are read again in every pass, from L2: a block of 16384 logits where the
    // rows fill the machine, of 4096 where they do not, eight at most.
    const unsigned int n = a.vocab;
    const auto blocks = [&](unsigned int each) { return (unsigned int)std::min<unsigned long long>(kMostParts, ((unsigned long long)n + each - 1) / each); };
    const bool small = n <= (unsigned int)kList;
    a.parts = small ? 1u : (unsigned long long)a.rows * blocks(4096) <= 3ull * dev->sm_count ? blocks(4096) : blocks(16384);
    const unsigned int piece = 32u * (vec ? (unsigned int)V : 1u);
    a.span = small ? 32u * (V == 8 ? 8u : 4u) : (unsigned int)(((unsigned long long)n + a.parts * kWarps * piece - 1) / (a.parts * kWarps * piece) * piece);
    kernel = small ? (vec ? sample_rows<T, V == 8 ? 8 : 4, V> : sample_rows<T, V == 8 ? 8 : 4, 1>) : (vec ? sample_rows<T, 0, V> : sample_rows<T, 0, 1>);
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
    const size_t size = dtype_bytes(p->dtype);
    const bool vec = ((size_t)a.x & 15) == 0 && (size_t)a.vocab * size % 16 == 0;
    if (p->dtype == B200_F32) op->choose<float>(vec);
    else if (p->dtype == B200_BF16) op->choose<__nv_bfloat16>(vec);
    else op->choose<__half>(vec);
    if ((unsigned long long)a.rows * a.parts >> 31) ops.refuse("too many rows", B200_E_UNSUPPORTED);
  });
}
