// Attention over a paged cache (b200_cache_attention_link): the choice of kernels and their launch.
#include <cmath>

#include "cache.hpp"
#include "kernels/cache_attn_terms.cuh"

using namespace b200;

namespace {

// ---- row by row, a warp each
template <class T, bool CODED>
__global__ void __launch_bounds__(256) cache_attention_rows(const __grid_constant__ CacheAttnArgs a) {
  grid_begin();
  const unsigned int lane = threadIdx.x & 31u;
  const CacheArgs& c = a.c;
  const long long n = (long long)c.tokens * a.H;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (long long)gridDim.x * 8) {
    const int row = (int)(i / a.H);
    int b;
    if (c.starts) {
      int lo = 0, hi = c.batch;                  // the last sequence that starts at the row or before it
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(c.starts + mid) <= row) lo = mid;
        else hi = mid;
      }
      b = lo;
    } else {
      b = row / c.each;
    }
    const CacheSeq s = cache_seq(c, b);
    if (row < s.first || row >= s.first + s.count) continue;
    cache_attention_row<T, CODED>(a, b, (int)(i - (long long)row * a.H), row, s.pos0 + (row - s.first), lane);
  }
}

typedef void (*RowsKernel)(const CacheAttnArgs);

struct CacheAttnOperator : b200_operator {
  CacheAttnArgs a = {};
  int dtype = 0;
  bool coded = false;
  RowsKernel rows = nullptr;
  unsigned int grid = 0;
  void choose() {
    const long long n = (long long)a.c.tokens * a.H;
    if (!n || !a.c.batch) return;
    rows = dtype == B200_F32 ? (coded ? cache_attention_rows<float, true> : cache_attention_rows<float, false>)
         : dtype == B200_BF16 ? (coded ? cache_attention_rows<__nv_bfloat16, true> : cache_attention_rows<__nv_bfloat16, false>)
                              : (coded ? cache_attention_rows<__half, true> : cache_attention_rows<__half, false>);
    ready(rows);
    grid = (unsigned int)std::min<long long>((n + 7) / 8, 16ll * dev->sm_count);
  }
  void run(cudaStream_t s) override {
    if (grid) launch(rows, dim3(grid), 256, 0, s, a);
  }
};

}  // namespace

extern "C" int b200_cache_attention_link(b200_dev* dev, const b200_cache_attention* p, b200_operator** out) {
  return link_operator<CacheAttnOperator>(dev, p, out, [&](CacheAttnOperator* op) {
    Operands ops(op, "cache_attention");
    ops.dtype(p->dtype);
    const b200_cache& pc = p->cache;
    CacheAttnArgs& a = op->a;
    a.c = bind_cache(ops, pc, p->dtype, false);
    if (pc.d > 128) ops.refuse("heads of more than 128 elements", B200_E_UNSUPPORTED);
    if (p->heads < 1 || p->heads > 65535 || p->heads % pc.kv_heads) ops.refuse("heads must be a multiple of kv_heads, between 1 and 65535");
    if (!(p->scale > 0.f) || !std::isfinite(p->scale)) ops.refuse("the scale must be positive and finite");
    if (!(p->cap >= 0.f) || !std::isfinite(p->cap)) ops.refuse("the cap must be finite and not negative (0: none)");
    if (!std::isfinite(p->scale * kCacheLog2e)) ops.refuse("the scale is too large");
    if (p->cap > 0.f && (!std::isfinite(p->cap * kCacheLog2e) || !std::isnormal(p->scale / p->cap))) ops.refuse("the cap is too far from the scale");
    if (p->window < 0 || p->sinks < 0) ops.refuse("window and sinks must not be negative");
    const unsigned long long n = extent_product({pc.tokens, p->heads, pc.d}, "cache_attention");
    const size_t size = dtype_bytes(p->dtype);
    a.q = (const void*)ops.in(p->q, "q", n, size);
    a.out = (void*)ops.out(p->out, "out", n, size);
    a.lse = (float*)ops.out(p->lse, "lse", extent_product({pc.tokens, p->heads}, "cache_attention"), 4, false);
    a.slopes = (const float*)ops.in(p->slopes, "slopes", (unsigned long long)p->heads, 4, false);
    ops.check_overlaps();
    op->dtype = p->dtype;
    op->coded = pc.dtype == B200_E4M3;
    a.status = (unsigned int*)dev->status_dev;
    a.H = p->heads;
    a.group = p->heads / pc.kv_heads;
    // (positions are below 2^31: a window beyond that is none)
    const bool none = p->window == 0 || p->window >= 0x7fffffffll;
    a.window = none ? 0 : (int)p->window;
    a.sinks = none ? 0 : (int)std::min<int64_t>(p->sinks, 0x7fffffff);
    a.scale = p->scale;
    a.cap = p->cap;
    a.over = p->cap > 0.f ? p->scale / p->cap : 0.f;
    op->choose();
  });
}
