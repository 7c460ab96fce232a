// Attention and its gradients (b200_attention_link, b200_attention_grad_link): the choice of kernels and their launch.
#include <cmath>
#include <cstring>

#include "operators.hpp"
#include "kernels/attn_fwd_sm100.cuh"
#include "kernels/attn_terms.cuh"

using namespace b200;

namespace {

// ---- row by row, a warp each
template <class T>
__global__ void __launch_bounds__(256) attn_forward_rows(const __grid_constant__ AttnArgs a) {
  grid_begin();
  const unsigned int lane = threadIdx.x & 31u;
  const long long n = (long long)a.B * a.S * a.H;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (long long)gridDim.x * 8) {
    const long long bs = i / a.H;
    attn_forward_row<T>(a, (int)(bs / a.S), (int)(i - bs * a.H), (int)(bs % a.S), lane);
  }
}
// delta_r = <d_out_r, out_r>
template <class T>
__global__ void __launch_bounds__(256) attn_delta(const __grid_constant__ AttnArgs a) {
  grid_begin();
  const unsigned int lane = threadIdx.x & 31u;
  const long long n = (long long)a.B * a.S * a.H;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (long long)gridDim.x * 8) {
    const long long bs = i / a.H;
    const int b = (int)(bs / a.S), h = (int)(i - bs * a.H), r = (int)(bs % a.S);
    float x[4], y[4];
    attn_load_row<T>(a, a.o, attn_q_at(a, b, r, h), lane, x);
    attn_load_row<T>(a, a.d_out, attn_q_at(a, b, r, h), lane, y);
    const float s = attn_dot(x, y);
    if (lane == 0) a.delta[((long long)b * a.H + h) * a.S + r] = s;
  }
}
template <class T>
__global__ void __launch_bounds__(256) attn_dq_rows(const __grid_constant__ AttnArgs a) {
  grid_begin();
  const unsigned int lane = threadIdx.x & 31u;
  const long long n = (long long)a.B * a.S * a.H;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (long long)gridDim.x * 8) {
    const long long bs = i / a.H;
    attn_dq_row<T>(a, (int)(bs / a.S), (int)(i - bs * a.H), (int)(bs % a.S), lane);
  }
}
template <class T>
__global__ void __launch_bounds__(256) attn_dkv_rows(const __grid_constant__ AttnArgs a) {
  grid_begin();
  const unsigned int lane = threadIdx.x & 31u;
  const long long n = (long long)a.B * a.T * a.HK;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (long long)gridDim.x * 8) {
    const long long bt = i / a.HK;
    attn_dkv_row<T>(a, (int)(bt / a.T), (int)(i - bt * a.HK), (int)(bt % a.T), lane, 3);
  }
}

// ---- rows of `d` elements to or from rows of `ld` (heads that no tensor map describes pass through padded copies)
__global__ void __launch_bounds__(256) attn_copy_rows(const unsigned short* src, unsigned short* dst, long long rows, int d, int from, int to) {
  grid_begin();
  const long long n = rows * d;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / d;
    const int e = (int)(i - row * d);
    dst[row * to + e] = src[row * from + e];
  }
}

typedef void (*AttnKernel)(const AttnArgs);
typedef void (*ForwardKernel)(const b200_tmap, const b200_tmap, const b200_tmap, const b200_tmap, const AttnArgs);

template <class T, int DP, int NQ>
ForwardKernel forward_of(bool cap, bool bias) {
  if (cap) return bias ? attn_forward_tc<T, DP, NQ, true, true> : attn_forward_tc<T, DP, NQ, true, false>;
  return bias ? attn_forward_tc<T, DP, NQ, false, true> : attn_forward_tc<T, DP, NQ, false, false>;
}

// [batch, length, heads, d] in boxes of 128 positions x 64 elements of a head, swizzled as the tensor cores read them
b200_tmap head_map(const void* p, int dtype, int batch, int length, int heads, int d, int ld) {
  CUtensorMap map;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)length, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)heads * ld * 2, (cuuint64_t)ld * 2, (cuuint64_t)length * heads * ld * 2};
  const cuuint32_t box[4] = {64, 128, 1, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = cu().cuTensorMapEncodeTiled_(&map, dtype == B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, (void*)p,
                                                  dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(B200_E_UNSUPPORTED, "attention: a node's layout cannot be described to the TMA unit (CUresult " + std::to_string((int)r) + ")");
  static_assert(sizeof(b200_tmap) == sizeof(CUtensorMap), "tensor map");
  b200_tmap m;
  memcpy(&m, &map, sizeof m);
  return m;
}

template <class F>
auto by_type(int dtype, F&& f) {
  if (dtype == B200_F32) return f(float());
  if (dtype == B200_BF16) return f(__nv_bfloat16());
  return f(__half());
}

struct AttnOperator : b200_operator {
  AttnArgs a = {};
  int dtype = 0;
  bool grad = false;
  long long rows = 0, key_rows = 0;
  // tensor-core form
  bool tc = false;
  ForwardKernel forward = nullptr;
  b200_tmap map_q, map_k, map_v, map_o;
  unsigned int threads = 0, grid = 0;
  size_t smem = 0;
  // padded copies: what is copied before and after the kernels
  struct Copy {
    const void* src;
    void* dst;
    long long rows;
    int from, to;
  };
  std::vector<Copy> before, after;
  int head = 0;                // elements of a head that the caller's nodes have

  AttnKernel kernel(int which) const {
    return by_type(dtype, [&](auto t) -> AttnKernel {
      typedef decltype(t) T;
      return which == 0 ? attn_forward_rows<T> : which == 1 ? attn_delta<T> : which == 2 ? attn_dq_rows<T> : attn_dkv_rows<T>;
    });
  }
  void choose() {
    head = a.D;
    for (int i = 0; i < 4; ++i) ready(kernel(i));
    ready(attn_copy_rows);
    tc = dtype != B200_F32 && rows && key_rows && !grad;
    if (grad) {
      take_workspace((size_t)rows * 4);
      a.delta = (float*)workspace;
    }
    if (tc) choose_tc();
  }
  // Heads whose rows or addresses are no multiples of 16 bytes go through copies with padded rows.
  void pad() {
    bool plain = a.D % 8 == 0;
    for (const void* p : {a.q, a.k, a.v, (const void*)a.out}) plain &= ((size_t)p & 15) == 0;
    if (plain) return;
    const int ld = (a.D + 7) / 8 * 8;
    size_t at = 0;
    auto room = [&](long long n) {
      const size_t here = at;
      at += ((size_t)n * ld * 2 + 255) & ~(size_t)255;
      return here;
    };
    const size_t q = room(rows), k = room(key_rows), v = room(key_rows), o = room(rows);
    take_workspace(at);
    auto in = [&](const void*& p, size_t where, long long n) {
      before.push_back({p, (void*)(workspace + where), n, a.D, ld});
      p = (const void*)(workspace + where);
    };
    in(a.q, q, rows);
    in(a.k, k, key_rows);
    in(a.v, v, key_rows);
    after.push_back({(const void*)(workspace + o), a.out, rows, ld, a.D});
    a.out = (void*)(workspace + o);
    a.ld = ld;
  }
  void choose_tc() {
    pad();
    map_q = head_map(a.q, dtype, a.B, a.S, a.H, a.D, a.ld);
    map_k = head_map(a.k, dtype, a.B, a.T, a.HK, a.D, a.ld);
    map_v = head_map(a.v, dtype, a.B, a.T, a.HK, a.D, a.ld);
    map_o = head_map(a.out, dtype, a.B, a.S, a.H, a.D, a.ld);
    const bool cap = a.cap > 0.f, bias = a.slopes != nullptr;
    const int tiles = (a.T + 127) / 128;
    const long long heads = (long long)a.B * a.H;
    // Heads of more than 64 elements: two query tiles a CTA share each key tile (64 KB per tile of 128 x 128 would otherwise
    // come in from L2 for 1024 cycles of products), unless that leaves SMs without work.
    const bool two = a.D > 64 && heads * ((a.S + 255) / 256) >= dev->sm_count;
    by_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      if constexpr (sizeof(T) == 2) {
        if (a.D <= 64) set<T, 64, 1>(cap, bias, tiles);
        else if (two) set<T, 128, 2>(cap, bias, tiles);
        else set<T, 128, 1>(cap, bias, tiles);
      }
      return 0;
    });
    const long long n = heads * ((a.S + 128 * (two ? 2 : 1) - 1) / (128 * (two ? 2 : 1)));
    if (n >> 31) throw Error(B200_E_UNSUPPORTED, "attention: too many rows");
    grid = (unsigned int)n;
    if (smem > 227 * 1024) throw Error(B200_E_UNSUPPORTED, "attention: too many keys");
    ready(forward, smem);
  }
  template <class T, int DP, int NQ>
  void set(bool cap, bool bias, int tiles) {
    forward = forward_of<T, DP, NQ>(cap, bias);
    threads = FwdShape<DP, NQ>::kThreads;
    smem = FwdShape<DP, NQ>::smem(tiles);
  }
  void copy(const std::vector<Copy>& list, cudaStream_t s) {
    for (auto& c : list)
      launch(attn_copy_rows, (unsigned int)std::min<long long>((c.rows * head + 1023) / 1024, 16ll * dev->sm_count), 256, 0, s, (const unsigned short*)c.src,
             (unsigned short*)c.dst, c.rows, head, c.from, c.to);
  }
  unsigned int blocks(long long n) const { return (unsigned int)std::min<long long>((n + 7) / 8, 16ll * dev->sm_count); }
  void run(cudaStream_t s) override {
    if (tc) {
      copy(before, s);
      launch(forward, grid, threads, smem, s, map_q, map_k, map_v, map_o, a);
      copy(after, s);
      return;
    }
    if (!grad) {
      if (rows) launch(kernel(0), blocks(rows), 256, 0, s, a);
      return;
    }
    if (rows) {
      launch(kernel(1), blocks(rows), 256, 0, s, a);
      launch(kernel(2), blocks(rows), 256, 0, s, a);
    }
    if (key_rows) launch(kernel(3), blocks(key_rows), 256, 0, s, a);
  }
};

void bind(const b200_attention& p, AttnOperator* op, bool grad) {
  Operands ops(op, grad ? "attention_grad" : "attention");
  ops.dtype(p.dtype);
  const long long most = 1ll << 30;
  if (p.batch < 0 || p.batch > most || p.queries < 0 || p.queries > most || p.keys < 0 || p.keys > most) ops.refuse("batch, queries and keys must be between 0 and 2^30");
  if (p.heads < 1 || p.kv_heads < 1 || p.heads > 65535 || p.heads % p.kv_heads) ops.refuse("heads must be a multiple of kv_heads, between 1 and 65535");
  if (p.d < 1) ops.refuse("d must be positive");
  if (p.d > 128) ops.refuse("heads of more than 128 elements", B200_E_UNSUPPORTED);
  if (!(p.scale > 0.f) || !std::isfinite(p.scale)) ops.refuse("the scale must be positive and finite");
  if (!(p.cap >= 0.f) || !std::isfinite(p.cap)) ops.refuse("the cap must be finite and not negative (0: none)");
  if (p.mask < B200_MASK_NONE || p.mask > B200_MASK_PREFIX) ops.refuse("unknown mask " + std::to_string(p.mask));
  if ((p.mask == B200_MASK_PREFIX) != (p.prefix.pool_id >= 0)) ops.refuse("'prefix' goes with the prefix mask");
  if ((p.query_documents.pool_id >= 0) != (p.key_documents.pool_id >= 0)) ops.refuse("documents are given for queries and keys, or for neither");
  const size_t size = dtype_bytes(p.dtype);
  const unsigned long long nq = extent_product({p.batch, p.queries, p.heads, p.d}, "attention");
  const unsigned long long nk = extent_product({p.batch, p.keys, p.kv_heads, p.d}, "attention");
  AttnArgs& a = op->a;
  op->dtype = p.dtype;
  op->grad = grad;
  op->rows = (long long)(nq / (unsigned)p.d);
  op->key_rows = (long long)(nk / (unsigned)p.d);
  a.q = (const void*)ops.in(p.q, "q", nq, size);
  a.k = (const void*)ops.in(p.k, "k", nk, size);
  a.v = (const void*)ops.in(p.v, "v", nk, size);
  if (grad) {
    a.o = (const void*)ops.in(p.out, "out", nq, size);
    a.lse = (float*)ops.in(p.lse, "lse", (unsigned long long)op->rows, 4);
    a.d_out = (const void*)ops.in(p.d_out, "d_out", nq, size);
    a.dq = (void*)ops.out(p.dq, "dq", nq, size);
    a.dk = (void*)ops.out(p.dk, "dk", nk, size);
    a.dv = (void*)ops.out(p.dv, "dv", nk, size);
  } else {
    a.out = (void*)ops.out(p.out, "out", nq, size);
    a.lse = (float*)ops.out(p.lse, "lse", (unsigned long long)op->rows, 4, false);
  }
  a.lengths = (const int*)ops.in(p.lengths, "lengths", (unsigned long long)p.batch, 4, false);
  a.prefix = (const int*)ops.in(p.prefix, "prefix", (unsigned long long)p.batch, 4, false);
  a.qdoc = (const int*)ops.in(p.query_documents, "query_documents", extent_product({p.batch, p.queries}, "attention"), 4, false);
  a.kdoc = (const int*)ops.in(p.key_documents, "key_documents", extent_product({p.batch, p.keys}, "attention"), 4, false);
  a.slopes = (const float*)ops.in(p.slopes, "slopes", (unsigned long long)p.heads, 4, false);
  ops.check_overlaps();
  a.status = (unsigned int*)op->dev->status_dev;
  a.B = (int)p.batch;
  a.S = (int)p.queries;
  a.T = (int)p.keys;
  a.H = p.heads;
  a.HK = p.kv_heads;
  a.D = a.ld = p.d;
  a.group = p.heads / p.kv_heads;
  a.mask = p.mask;
  a.scale = p.scale;
  a.cap = p.cap;
  op->choose();
}

}  // namespace

extern "C" int b200_attention_link(b200_dev* dev, const b200_attention* p, b200_operator** out) {
  return link_operator<AttnOperator>(dev, p, out, [&](AttnOperator* op) { bind(*p, op, false); });
}

extern "C" int b200_attention_grad_link(b200_dev* dev, const b200_attention* p, b200_operator** out) {
  return link_operator<AttnOperator>(dev, p, out, [&](AttnOperator* op) { bind(*p, op, true); });
}
