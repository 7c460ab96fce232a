// Choosing a token for each row of logits (b200_sample_link).
//
//   w_i = exp((x_i - max) / T);  kept: the first n in the order of falling x, of rising i among equal ones;  token: where the running sum of the kept, in the
//   order of i, passes uniform * its end
//
// Logits are compared as whole numbers in their order (`key`).  What is kept is then all keys above a border and, of those equal to it, the ones up to
// an index.  The borders are found bit by bit, a pass over the row each; sums are in double precision, so that they lie where they do in 64 bits.
#include <cmath>

#include "kernels/op_common.cuh"
#include "operators.hpp"

using namespace b200;

namespace {

struct SampleArgs {
  const void* x;
  const float *uniform, *temperatures, *top_ps, *min_ps;
  const int* top_ks;
  int* tokens;
  float* logprob;
  unsigned int rows, vocab;
  float temperature, top_p, min_p;
  int top_k;
};

constexpr int kThreads = 256;

// rises with the value; the two zeros are one, what is undefined is the least of all, -infinity
__device__ __forceinline__ unsigned int key_of(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const unsigned int u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned int k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

template <class V, class F>
__device__ __forceinline__ V block_reduce(V v, V* sh, F join) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v = join(v, sh[i]);
  return v;
}
// the sum of the threads before this one, and of all
template <class V>
__device__ __forceinline__ V block_before(V v, V* sh, V& all) {
  V up_to = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, up_to, o);
    if ((int)(threadIdx.x & 31u) >= o) up_to += x;
  }
  __syncthreads();
  if ((threadIdx.x & 31u) == 31) sh[threadIdx.x >> 5] = up_to;
  __syncthreads();
  V before = up_to - v;
  all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    if (i < (int)(threadIdx.x >> 5)) before += sh[i];
    all += sh[i];
  }
  return before;
}

template <class T>
__global__ void __launch_bounds__(kThreads) sample_rows(const __grid_constant__ SampleArgs a) {
  __shared__ double sums[kThreads / 32];
  __shared__ unsigned long long numbers[kThreads / 32];
  __shared__ int chosen;
  grid_begin();
  const unsigned int row = blockIdx.x, n = a.vocab;
  const T* x = (const T*)a.x + (unsigned long long)row * n;
  const float temperature = a.temperatures ? a.temperatures[row] : a.temperature, top_p = a.top_ps ? a.top_ps[row] : a.top_p;
  const float min_p = a.min_ps ? a.min_ps[row] : a.min_p;
  const int top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  auto add = [](auto u, auto v) { return u + v; };
  auto greater = [](auto u, auto v) { return u > v ? u : v; };
  // the largest key, and the first index that has it
  unsigned long long best = 0;
  for (unsigned int i = threadIdx.x; i < n; i += kThreads) best = greater(best, (unsigned long long)key_of(to_float(x[i])) << 32 | (0xffffffffu - i));
  best = block_reduce(best, numbers, greater);
  const unsigned int top = (unsigned int)(best >> 32), none = key_of(-INFINITY);
  if (top == none || !(temperature > 0.f)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = top == none ? -1 : (int)(0xffffffffu - (unsigned int)best);
      if (a.logprob) a.logprob[row] = top == none ? -INFINITY : 0.f;
    }
    return;
  }
  const float largest = of_key(top);
  auto weight = [&](unsigned int k) -> float { return k == top ? 1.f : largest == INFINITY || k == none ? 0.f : expf((of_key(k) - largest) / temperature); };
  // (count, sum) of the keys from `from` on
  auto count_from = [&](unsigned int from) {
    unsigned long long c = 0;
    for (unsigned int i = threadIdx.x; i < n; i += kThreads) c += key_of(to_float(x[i])) >= from;
    return block_reduce(c, numbers, add);
  };
  auto sum_from = [&](unsigned int from) {
    double s = 0.0;
    for (unsigned int i = threadIdx.x; i < n; i += kThreads) {
      const unsigned int k = key_of(to_float(x[i]));
      if (k >= from) s += (double)weight(k);
    }
    return block_reduce(s, sums, add);
  };
  // kept: keys above `border`, and `ties` of those equal to it
  unsigned int border = none;
  unsigned long long ties = n;
  if (top_k > 0 && (unsigned int)top_k < n) {
    border = 0;
    for (unsigned int bit = 0x80000000u; bit; bit >>= 1)
      if (count_from(border | bit) >= (unsigned long long)top_k) border |= bit;
    ties = (unsigned long long)top_k - (border == 0xffffffffu ? 0ull : count_from(border + 1));
  }
  if (top_p < 1.f) {
    const double above_k = border == 0xffffffffu ? 0.0 : sum_from(border + 1), w_k = (double)weight(border);
    const double all = ties >= n ? sum_from(0) : above_k + (double)ties * w_k, target = fmax((double)top_p, 0.0) * all;
    unsigned int t = 0;
    for (unsigned int bit = 0x80000000u; bit; bit >>= 1)
      if ((t | bit) <= border || sum_from(t | bit) >= target) t |= bit;
    // (a target of nothing is reached above all keys: the largest is kept all the same)
    t = min(t, top);
    const double above = sum_from(t + 1), w = (double)weight(t);
    const double need = w > 0.0 ? ceil((target - above) / w) : 1.0;
    const unsigned long long r = need < 1.0 ? 1ull : need > 4e9 ? (unsigned long long)n : (unsigned long long)need;
    ties = t == border ? min(ties, r) : r;
    border = t;
  }
  // the index of the last tie that is kept
  unsigned int last_tie = n;
  if (ties < n) {
    unsigned long long seen = 0, all;
    if (threadIdx.x == 0) chosen = (int)n;
    for (unsigned int i0 = 0; i0 < n && seen < ties; i0 += kThreads) {
      const unsigned int i = i0 + threadIdx.x;
      const unsigned long long mine = i < n && key_of(to_float(x[i])) == border;
      const unsigned long long before = block_before(mine, numbers, all);
      if (mine && seen + before + 1 == ties) chosen = (int)i;
      seen += all;
    }
    __syncthreads();
    last_tie = (unsigned int)chosen;
    __syncthreads();
  }
  auto kept = [&](unsigned int i) -> float {
    if (i >= n) return 0.f;
    const unsigned int k = key_of(to_float(x[i]));
    if (k < border || (k == border && i > last_tie)) return 0.f;
    const float w = weight(k);
    return k == top || !(w < min_p) ? w : 0.f;
  };
  double total = 0.0;
  for (unsigned int i = threadIdx.x; i < n; i += kThreads) total += (double)kept(i);
  total = block_reduce(total, sums, add);
  const float u = a.uniform[row];
  const double target = (u > 0.f ? (double)u : 0.0) * total;
  // the first whose running sum passes the target; the last kept one where none does
  double before = 0.0, all;
  if (threadIdx.x == 0) chosen = 0x7fffffff;
  unsigned long long last = 0;
  __syncthreads();
  for (unsigned int i0 = 0; i0 < n; i0 += kThreads) {
    const unsigned int i = i0 + threadIdx.x;
    const float w = kept(i);
    const double up_to = before + block_before((double)w, sums, all) + (double)w;
    if (w > 0.f) {
      last = i + 1;
      if (up_to > target) atomicMin(&chosen, (int)i);
    }
    before += all;
    __syncthreads();
    if (chosen != 0x7fffffff) break;
    __syncthreads();
  }
  last = block_reduce(last, numbers, greater);
  if (threadIdx.x == 0) {
    const unsigned int i = chosen != 0x7fffffff ? (unsigned int)chosen : (unsigned int)(last - 1);
    a.tokens[row] = (int)i;
    if (a.logprob) a.logprob[row] = (float)log((double)weight(key_of(to_float(x[i]))) / total);
  }
}

typedef void (*SampleKernel)(const SampleArgs);

struct SampleOperator : b200_operator {
  SampleArgs a = {};
  SampleKernel kernel = nullptr;
  void run(cudaStream_t s) override {
    if (a.rows) launch(kernel, dim3(a.rows), kThreads, 0, s, a);
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
    op->kernel = p->dtype == B200_F32 ? sample_rows<float> : p->dtype == B200_BF16 ? sample_rows<__nv_bfloat16> : sample_rows<__half>;
    ready(op->kernel);
  });
}
