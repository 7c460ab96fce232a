// Attention and its gradients (b200_attention_link, b200_attention_grad_link): the choice of kernels and their launch.
#include <cmath>
#include <cstring>

#include "operators.hpp"
#include "kernels/attn_bwd_sm100.cuh"
#include "kernels/attn_few_sm100.cuh"
#include "kernels/attn_fwd_sm100.cuh"
#include "kernels/attn_single.cuh"
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
// What the gradients need of every row: its lse and <d_out, out> (and of half heads the sizes of rows and values), tile by tile of 128 queries, G threads a row.  out and d_out are read
// once, kRowsAtOnce rows of a thread under way together; what bounds it is the arithmetic of indices around 32 bytes a lane, so that
// is kept to 32 bits (64 x 256 positions, 8 heads of 64: 14.4 us with more of it).  Rows that see nothing get weights of zero; the places
// behind the last row are filled at link.
constexpr int kRowsAtOnce = 4;

template <class T, int VEC, int G>
__global__ void __launch_bounds__(256) attn_statistics(const __grid_constant__ AttnArgs a, const Divisor by_heads, const Divisor by_length) {
  grid_begin();
  constexpr unsigned int rows = 256 / G;
  constexpr bool kSizes = std::is_same<T, __half>::value;
  constexpr int chunks = VEC > 1 ? 1 : 128 / G;
  const int lane = (int)threadIdx.x % G;
  const unsigned int heads = (unsigned int)a.H, length = (unsigned int)a.S, tiles = (length + 127) / 128;
  const unsigned int n = (unsigned int)a.B * length * heads, step = gridDim.x * rows * kRowsAtOnce;
  for (unsigned int base = blockIdx.x * rows * kRowsAtOnce + threadIdx.x / G; base - threadIdx.x / G < n; base += step) {
    Raw<T, VEC> x[kRowsAtOnce][chunks], y[kRowsAtOnce][chunks];
    float lse[kRowsAtOnce];
    unsigned int stat[kRowsAtOnce];
#pragma unroll
    for (int k = 0; k < kRowsAtOnce; ++k) {
      const unsigned int i = base + k * rows;
      lse[k] = -INFINITY;
#pragma unroll
      for (int c = 0; c < chunks; ++c) {
        x[k][c].clear();
        y[k][c].clear();
      }
      if (i >= n) continue;
      const unsigned long long at = (unsigned long long)i * (unsigned int)a.ld;      // (the rows lie in this order)
#pragma unroll
      for (int c = 0; c < chunks; ++c) {
        const int e = (c * G + lane) * VEC;
        if (e >= a.D) continue;
        x[k][c].load((const T*)a.o + at + e);
        y[k][c].load((const T*)a.d_out + at + e);
      }
      const unsigned int bs = by_heads.of(i), h = i - bs * heads, b = by_length.of(bs), r = bs - b * length, bh = b * heads + h;
      lse[k] = a.lse[bh * length + r];
      stat[k] = (bh * tiles + (r >> 7)) * 256 + (r & 127);
    }
#pragma unroll
    for (int k = 0; k < kRowsAtOnce; ++k) {
      float delta = 0.f, of_d_out = 0.f, of_out = 0.f;
#pragma unroll
      for (int c = 0; c < chunks; ++c) {
        float u[VEC], w[VEC];
        x[k][c].values(u);
        y[k][c].values(w);
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          // (rows of padded copies end in zeros)
          delta = fmaf(u[q], w[q], delta);
          if constexpr (kSizes) {
            of_d_out = fmaf(w[q], w[q], of_d_out);
            of_out = fmaf(u[q], u[q], of_out);
          }
        }
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) {
        delta += __shfl_xor_sync(0xffffffffu, delta, o);
        if constexpr (kSizes) {
          of_d_out += __shfl_xor_sync(0xffffffffu, of_d_out, o);
          of_out += __shfl_xor_sync(0xffffffffu, of_out, o);
        }
      }
      const bool empty = lse[k] == -INFINITY;
      if (lane == 0 && base + k * rows < n) {
        a.stat[stat[k]] = empty ? INFINITY : sizeof(T) == 4 ? lse[k] : lse[k] * kLog2e - kWeightLog<T>;
        a.stat[stat[k] + 128] = empty ? 0.f : delta;
        if constexpr (kSizes) {
          // (what is infinite or undefined has results that are done again: it is left out here)
          const float x = sqrtf(of_d_out), y = x * sqrtf(of_out);
          a.row_sizes[(stat[k] >> 8) * 128 + (stat[k] & 127u)] = make_float2(!empty && x < INFINITY ? x : 0.f, !empty && y < INFINITY ? y : 0.f);
        }
      }
    }
  }
  if constexpr (kSizes) {
    const long long keys = (long long)a.B * a.T * a.HK;
    for (long long first = (long long)blockIdx.x * rows * kRowsAtOnce; first < keys; first += (long long)gridDim.x * rows * kRowsAtOnce) {
      const long long i = first + threadIdx.x / G;
      Raw<T, VEC> x[kRowsAtOnce][chunks];
#pragma unroll
      for (int k = 0; k < kRowsAtOnce; ++k)
#pragma unroll
        for (int c = 0; c < chunks; ++c) {
          const int e = (c * G + lane) * VEC;
          x[k][c].clear();
          if (i + k * rows < keys && e < a.D) x[k][c].load((const T*)a.v + (i + k * rows) * a.ld + e);
        }
#pragma unroll
      for (int k = 0; k < kRowsAtOnce; ++k) {
        float of_v = 0.f;
#pragma unroll
        for (int c = 0; c < chunks; ++c) {
          float u[VEC];
          x[k][c].values(u);
#pragma unroll
          for (int q = 0; q < VEC; ++q) of_v = fmaf(u[q], u[q], of_v);
        }
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) of_v += __shfl_xor_sync(0xffffffffu, of_v, o);
        if (lane == 0 && i + k * rows < keys) a.value_sizes[i + k * rows] = of_v < INFINITY ? sqrtf(of_v) : 0.f;
      }
    }
  }
}
typedef void (*StatisticsKernel)(const AttnArgs, const Divisor, const Divisor);

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

// ---- rows of `d` elements to or from rows of `ld` (heads that no tensor map describes pass through padded copies); the padding is zeros
__global__ void __launch_bounds__(256) attn_copy_rows(const unsigned short* src, unsigned short* dst, long long rows, int d, int from, int to) {
  grid_begin();
  const long long n = rows * to;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / to;
    const int e = (int)(i - row * to);
    dst[i] = e < d ? src[row * from + e] : (unsigned short)0;
  }
}

typedef void (*GradKernel)(const GradMaps, const AttnArgs, unsigned int);
typedef void (*SingleKernel)(const AttnArgs, int, int, int);
typedef void (*SingleGradKernel)(const AttnArgs, int, int, int, unsigned int);
typedef void (*FewKernel)(const AttnArgs, const FewArgs);
typedef void (*FewJoinKernel)(const AttnArgs, const FewArgs);

template <class T, int DP>
FewKernel few_of(bool cap, bool bias) {
  if (cap) return bias ? attn_forward_few<T, DP, true, true> : attn_forward_few<T, DP, true, false>;
  return bias ? attn_forward_few<T, DP, false, true> : attn_forward_few<T, DP, false, false>;
}
template <class T, int DP, int CW>
GradKernel grad_of(bool cap, bool bias) {
  if (cap) return bias ? attn_grad_tc<T, DP, CW, true, true> : attn_grad_tc<T, DP, CW, true, false>;
  return bias ? attn_grad_tc<T, DP, CW, false, true> : attn_grad_tc<T, DP, CW, false, false>;
}

typedef void (*AttnKernel)(const AttnArgs);
typedef void (*ForwardKernel)(const b200_tmap, const b200_tmap, const b200_tmap, const b200_tmap, const AttnArgs);

// (two query tiles: key tiles of 64 where scores are capped, of 128 else)
template <class T, int DP, int NQ, int KW, bool SUMS>
ForwardKernel forward_of(bool cap, bool bias) {
  if constexpr (NQ == 2) {
    constexpr bool kCap = KW == 64;
    return bias ? attn_forward_tc<T, DP, NQ, KW, kCap, true, SUMS> : attn_forward_tc<T, DP, NQ, KW, kCap, false, SUMS>;
  } else {
    if (cap) return bias ? attn_forward_tc<T, DP, NQ, KW, true, true, SUMS> : attn_forward_tc<T, DP, NQ, KW, true, false, SUMS>;
    return bias ? attn_forward_tc<T, DP, NQ, KW, false, true, SUMS> : attn_forward_tc<T, DP, NQ, KW, false, false, SUMS>;
  }
}

// [batch, length, heads, d] in boxes of `box_rows` positions x 64 elements of a head, swizzled as the tensor cores read them
b200_tmap head_map(const void* p, int dtype, int batch, int length, int heads, int d, int ld, int box_rows) {
  CUtensorMap map;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)length, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)heads * ld * 2, (cuuint64_t)ld * 2, (cuuint64_t)length * heads * ld * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
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
  StatisticsKernel statistics = nullptr;
  unsigned int statistics_grid = 0;
  Divisor by_heads, by_length;
  // tensor-core form
  bool tc = false;
  ForwardKernel forward = nullptr;
  GradKernel gradients = nullptr;
  AttnKernel join = nullptr;
  GradMaps maps;
  SingleKernel single = nullptr;
  SingleGradKernel single_grad = nullptr;
  int vec = 0, places = 1, groups = 4;
  FewKernel few = nullptr;
  FewJoinKernel few_join = nullptr;
  FewArgs few_args = {};
  b200_tmap map_q, map_k, map_v, map_o;
  unsigned int threads = 0, grid = 0, keys_grid = 0;
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
  size_t reserved = 0;         // of the workspace, while the operator is put together

  AttnKernel kernel(int which) const {
    return by_type(dtype, [&](auto t) -> AttnKernel {
      typedef decltype(t) T;
      return which == 0 ? attn_forward_rows<T> : which == 1 ? attn_dq_rows<T> : attn_dkv_rows<T>;
    });
  }
  size_t reserve(size_t bytes) {
    const size_t here = reserved;
    reserved += (bytes + 255) & ~(size_t)255;
    return here;
  }
  void choose() {
    head = a.D;
    tc = dtype != B200_F32 && rows && key_rows;
    if (dtype == B200_F32 && rows && key_rows) choose_single();
    else if (!tc)
      for (int i = 0; i < 3; ++i) ready(kernel(i));
    // Heads whose rows or addresses are no multiples of 16 bytes go through copies with padded rows.
    // (each operand has a copy of its own: those that are read may be one node, of which each takes as many rows as it has)
    struct Padded {
      const void** node;
      bool written, of_keys;
      size_t at;
    };
    std::vector<Padded> nodes;
    for (auto& n : {Padded{&a.q, false, false, 0}, {&a.k, false, true, 0}, {&a.v, false, true, 0}, {&a.o, false, false, 0}, {&a.d_out, false, false, 0},
                    {(const void**)&a.out, true, false, 0}, {(const void**)&a.dq, true, false, 0}, {(const void**)&a.dk, true, true, 0},
                    {(const void**)&a.dv, true, true, 0}})
      if (*n.node) nodes.push_back(n);
    bool plain = a.D % 8 == 0;
    for (auto& n : nodes) plain &= ((size_t)*n.node & 15) == 0;
    const int ld = (a.D + 7) / 8 * 8;
    const bool pad = tc && !plain;
    if (pad)
      for (auto& n : nodes) n.at = reserve((size_t)(n.of_keys ? key_rows : rows) * ld * 2);
    size_t stat = 0, row_sizes = 0, value_sizes = 0, parts = 0, tickets = 0, sums = 0;
    a.n_parts = 1;
    a.part_heads = a.group;
    if (tc && grad) {
      // A block walks all query heads that share its keys.  Where that leaves SMs without a block (two for heads of up to 64
      // elements), as many blocks share a key tile as divide the query heads and are needed, and their sums are joined.
      const long long blocks = (long long)a.B * a.HK * ((a.T + 127) / 128), want = (a.D <= 64 ? 2ll : 1ll) * dev->sm_count;
      while (a.n_parts < a.group && blocks * a.n_parts < want)
        do ++a.n_parts; while (a.group % a.n_parts);
      a.part_heads = a.group / a.n_parts;
      if (a.n_parts > 1) parts = reserve((size_t)a.n_parts * 2 * key_rows * (a.D <= 64 ? 64 : 128) * 4);
    }
    a.parts_of = Divisor((unsigned int)a.n_parts);
    if (tc && !grad && few_rows()) choose_few(&parts, &tickets);
    const bool summed = tc && !grad && !few && a.T > kSumKeys;
    if (summed) sums = reserve((size_t)rows * (a.D <= 64 ? 64 : 128) * 4);
    if (grad && rows) {
      const long long padded = (long long)a.B * a.H * ((a.S + 127) / 128) * 128;
      const int size = (int)dtype_bytes(dtype);
      const bool vec = tc || (a.D * size % 16 == 0 && (((size_t)a.o | (size_t)a.d_out) & 15) == 0);
      if (padded >> 30) throw Error(B200_E_UNSUPPORTED, "attention: too many rows");
      int group = 32;
      statistics = by_type(dtype, [&](auto t) -> StatisticsKernel {
        typedef decltype(t) T;
        constexpr int V = 16 / (int)sizeof(T), G = 128 / V;
        if (!vec) return attn_statistics<T, 1, 32>;
        group = a.D <= 64 ? G / 2 : G;
        return a.D <= 64 ? attn_statistics<T, V, G / 2> : attn_statistics<T, V, G>;
      });
      ready(statistics);
      by_heads = Divisor((unsigned int)a.H);
      by_length = Divisor((unsigned int)a.S);
      const long long at_once = 256 / group * kRowsAtOnce;
      statistics_grid = (unsigned int)std::min<long long>((rows + at_once - 1) / at_once, 8ll * dev->sm_count);
      stat = reserve((size_t)padded * 8);
      if (dtype == B200_F16) {
        row_sizes = reserve((size_t)padded * 8);
        value_sizes = reserve((size_t)key_rows * 4);
      }
    }
    take_workspace(reserved);
    if (grad && rows) {
      a.stat = (float*)(workspace + stat);
      // the places behind a head's last row: a finite lse beyond all scores (3.4e38), so that what lies there weighs nothing
      cu_check(cu().cuMemsetD8Async_(workspace + stat, 0x7f, (size_t)a.B * a.H * ((a.S + 127) / 128) * 1024, dev->stream), "cuMemsetD8Async(statistics)");
      if (dtype == B200_F16) {
        a.row_sizes = (float2*)(workspace + row_sizes);
        a.value_sizes = (float*)(workspace + value_sizes);
        cu_check(cu().cuMemsetD8Async_(workspace + row_sizes, 0, (size_t)a.B * a.H * ((a.S + 127) / 128) * 1024, dev->stream), "cuMemsetD8Async(sizes)");
      }
    }
    if (pad) {
      ready(attn_copy_rows);
      for (auto& n : nodes) {
        void* copy = (void*)(workspace + n.at);
        const long long many = n.of_keys ? key_rows : rows;
        if (n.written) after.push_back({copy, (void*)*n.node, many, ld, a.D});
        else before.push_back({*n.node, copy, many, a.D, ld});
        *n.node = copy;
      }
      a.ld = ld;
    }
    if (summed) a.sums = (float*)(workspace + sums);
    if (a.n_parts > 1) {
      a.parts = (float*)(workspace + parts);
      join = by_type(dtype, [&](auto t) -> AttnKernel {
        typedef decltype(t) T;
        if constexpr (sizeof(T) == 2) return a.D <= 64 ? attn_join_parts<T, 64> : attn_join_parts<T, 128>;
        return nullptr;
      });
      ready(join);
    }
    if (few) {
      few_args.parts = (float*)(workspace + parts);
      few_args.tickets = (unsigned int*)(workspace + tickets);
      cu_check(cu().cuMemsetD8Async_(workspace + tickets, 0, (size_t)grid * 4, dev->stream), "cuMemsetD8Async(tickets)");
      ready(few, smem);
      if (few_join) ready(few_join);
    } else if (tc) {
      choose_tc();
    }
  }
  // A tile of the tensor-core kernel has 128 queries of one head.  Up to 16 queries go sixteen rows at a time (of all heads that
  // share the keys), the keys split over the machine, and so do up to 128 over many keys, whose tiles would leave most of the machine idle
  // for the length of one walk: over 8192 keys a walk of tiles takes 100 us, and 17 queries of 8 heads of 64 take 16, 128 of them 29, 128 of
  // 32 heads over 8 (256 sixteens) 70; of heads of 128 20, 48 and (64 queries, 128 sixteens) 79.  Over 2048 keys the walk takes 29, half as
  // many sixteens 22 to 28; so the shorter the keys, the fewer.
  long long sixteens() const { return (long long)a.B * a.HK * (((long long)a.group * a.S + kFewRows - 1) / kFewRows); }
  bool few_rows() const { return a.S <= 16 || (a.S <= 128 && a.T >= 1024 && sixteens() * (a.D <= 64 ? 16 : 32) <= std::min(a.T, 4096)); }
  void choose_few(size_t* parts, size_t* tickets) {
    const long long pairs = sixteens();
    grid = blocks_of(pairs);
    by_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      if constexpr (sizeof(T) == 2) {
        few = a.D <= 64 ? few_of<T, 64>(a.cap > 0.f, a.slopes != nullptr) : few_of<T, 128>(a.cap > 0.f, a.slopes != nullptr);
        smem = a.D <= 64 ? FewShape<64>::smem() : FewShape<128>::smem();
      }
      return 0;
    });
    // Ranges of at least 256 keys, as many as give every SM four blocks: sequences of different lengths even out.
    const long long most = (a.T + 255) / 256, want = (4ll * dev->sm_count + pairs - 1) / pairs;
    const int step = kFewStep * kFewWarps, splits = (int)std::max<long long>(1, std::min<long long>(std::min(most, want), kFewMost));
    few_args.per_split = ((a.T + splits - 1) / splits + step - 1) / step * step;
    few_args.splits = (a.T + few_args.per_split - 1) / few_args.per_split;
    few_args.join_later = few_args.splits > 1 && a.group * a.S > kFewWarps;
    if (few_args.join_later)
      few_join = by_type(dtype, [&](auto t) -> FewJoinKernel {
        typedef decltype(t) T;
        if constexpr (sizeof(T) == 2) return a.D <= 64 ? attn_join_few<T, 64> : attn_join_few<T, 128>;
        return nullptr;
      });
    const int width = a.D <= 64 ? FewShape<64>::kWidth : FewShape<128>::kWidth;
    *parts = reserve(few_args.splits > 1 ? (size_t)pairs * few_args.splits * kFewRows * width * 4 : 0);
    *tickets = reserve((size_t)pairs * 4);
  }
  void choose_single() {
    vec = a.D % 4 == 0;
    for (const void* p : {a.q, a.k, a.v, a.d_out}) vec &= ((size_t)p & 15) == 0;
    // Blocks of 64 rows, two warps for 16 of them; where that leaves SMs without a block, of 16 rows and four warps (below that they read
    // the others four times as often for nothing: gradients of 2 x 1024 positions, 8 heads of 64, 220 us and 309).
    const long long blocks64 = (long long)a.B * (a.H * ((a.S + 63ll) / 64) + (grad ? a.HK * ((a.T + 63ll) / 64) : 0));
    groups = blocks64 < dev->sm_count ? 1 : 4;
    const int shares = groups == 1 ? 4 : 2, rows_each = 16 * groups, own = grad ? 2 : 1;
    threads = (unsigned int)(32 * groups * shares);
    keys_grid = grad ? blocks_of((long long)a.B * a.HK * ((a.T + rows_each - 1) / rows_each)) : 0;
    grid = blocks_of((long long)a.B * a.H * ((a.S + rows_each - 1) / rows_each) + keys_grid);
    // two places where that leaves heads of up to 64 elements two blocks an SM, and wider ones, which have one, room at all
    places = SingleShape::smem(a.D, groups, shares, own, 2) <= (size_t)(a.D <= 64 ? 113 : 227) * 1024 ? 2 : 1;
    smem = SingleShape::smem(a.D, groups, shares, own, places);
    if (!SingleShape::room_to_meet(a.D, groups, shares, own, places, a.D <= 64 ? 8 : 16)) throw Error(B200_E_UNSUPPORTED, "attention: internal error: no room to meet");
    if (grad) {
      single_grad = a.D <= 64 ? attn_grad_single<8> : attn_grad_single<16>;
      ready(single_grad, smem);
    } else {
      single = a.D <= 64 ? attn_forward_single<8> : attn_forward_single<16>;
      ready(single, smem);
    }
  }
  unsigned int blocks_of(long long n) const {
    if (n >> 31) throw Error(B200_E_UNSUPPORTED, "attention: too many rows");
    return (unsigned int)n;
  }
  void choose_tc() {
    // results leave 32 rows at a time
    if (grad) {
      maps.dq = of_queries(a.dq, 32);
      maps.dk = of_keys(a.dk, 32);
      maps.dv = of_keys(a.dv, 32);
    } else {
      map_q = of_queries(a.q, 128);
      map_o = of_queries(a.out, 32);
    }
    const long long heads = (long long)a.B * a.H;
    // Heads of more than 64 elements: two query tiles a CTA share each key tile (64 KB per tile of 128 x 128 would otherwise
    // come in from L2 for 1024 cycles of products), unless that leaves SMs without work.
    const bool two = a.D > 64 && heads * ((a.S + 255) / 256) >= dev->sm_count;
    // Key tiles of 64, whose next scores are formed during the softmax of the ones before, where that takes long (capped scores: 2 x 4096
    // positions, 16 heads of 128, causal 261 us with tiles of 128, 226 with 64) and for heads of up to 64 elements (239 and 228); tiles
    // of 128 else (281 and 304 without a mask, 209 and 213 with a bias).
    by_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      if constexpr (sizeof(T) == 2) {
        if (grad) {
          if (a.D <= 64) set_grad<T, 64, 64>();
          else set_grad<T, 128, 128>();
        } else {
          if (a.D <= 64) set<T, 64, 1, 64>();
          else if (two && a.cap > 0.f) set<T, 128, 2, 64>();
          else if (two) set<T, 128, 2, 128>();
          else set<T, 128, 1, 64>();
        }
      }
      return 0;
    });
    grid = blocks_of(heads * ((a.S + 128 * (!grad && two ? 2 : 1) - 1) / (128 * (!grad && two ? 2 : 1))));
    if (grad) {
      keys_grid = blocks_of((long long)a.B * a.HK * ((a.T + 127) / 128) * a.n_parts);
      grid = blocks_of((long long)grid + keys_grid);
    }
    if (smem > 227 * 1024) throw Error(B200_E_UNSUPPORTED, "attention: too many keys or queries with documents");
    if (grad) ready(gradients, smem);
    else ready(forward, smem);
  }
  template <class T, int DP, int NQ, int KW>
  void set() {
    forward = a.sums ? forward_of<T, DP, NQ, KW, true>(a.cap > 0.f, a.slopes != nullptr) : forward_of<T, DP, NQ, KW, false>(a.cap > 0.f, a.slopes != nullptr);
    threads = FwdShape<DP, NQ, KW>::kThreads;
    smem = FwdShape<DP, NQ, KW>::smem(a.kdoc ? (a.T + KW - 1) / KW : 0);      // (tiles have classes in memory with documents alone)
    map_k = of_keys(a.k, KW);
    map_v = of_keys(a.v, KW);
  }
  template <class T, int DP, int CW>
  void set_grad() {
    typedef BwdShape<DP, CW> Sh;
    gradients = grad_of<T, DP, CW>(a.cap > 0.f, a.slopes != nullptr);
    threads = Sh::kThreads;
    smem = Sh::smem(a.kdoc ? (std::max(a.S, a.T) + CW - 1) / CW : 0);
    maps.own_q = of_queries(a.q, 128);
    maps.own_d_out = of_queries(a.d_out, 128);
    maps.own_k = of_keys(a.k, 128);
    maps.own_v = of_keys(a.v, 128);
    maps.q = of_queries(a.q, CW);
    maps.d_out = of_queries(a.d_out, CW);
    maps.k = of_keys(a.k, CW);
    maps.v = of_keys(a.v, CW);
  }
  b200_tmap of_queries(const void* p, int rows) const { return head_map(p, dtype, a.B, a.S, a.H, a.D, a.ld, rows); }
  b200_tmap of_keys(const void* p, int rows) const { return head_map(p, dtype, a.B, a.T, a.HK, a.D, a.ld, rows); }
  void copy(const std::vector<Copy>& list, cudaStream_t s) {
    for (auto& c : list)
      launch(attn_copy_rows, (unsigned int)std::min<long long>((c.rows * head + 1023) / 1024, 16ll * dev->sm_count), 256, 0, s, (const unsigned short*)c.src,
             (unsigned short*)c.dst, c.rows, head, c.from, c.to);
  }
  unsigned int blocks(long long n) const { return (unsigned int)std::min<long long>((n + 7) / 8, 16ll * dev->sm_count); }
  void run(cudaStream_t s) override {
    copy(before, s);
    if (grad && rows) launch(statistics, statistics_grid, 256, 0, s, a, by_heads, by_length);
    if (tc && grad) {
      launch(gradients, grid, threads, smem, s, maps, a, keys_grid);
      if (join) launch(join, blocks(key_rows), 256, 0, s, a);
    } else if (few) {
      launch(few, dim3(grid, (unsigned int)few_args.splits), kFewWarps * 32, smem, s, a, few_args);
      if (few_join) launch(few_join, dim3(grid, (unsigned int)std::min(kFewRows, a.group * a.S)), kFewWarps * 32, 0, s, a, few_args);
    } else if (tc) {
      launch(forward, grid, threads, smem, s, map_q, map_k, map_v, map_o, a);
    } else if (single) {
      launch(single, grid, threads, smem, s, a, vec, places, groups);
    } else if (single_grad) {
      launch(single_grad, grid, threads, smem, s, a, vec, places, groups, keys_grid);
    } else if (grad) {
      if (rows) launch(kernel(1), blocks(rows), 256, 0, s, a);
      if (key_rows) launch(kernel(2), blocks(key_rows), 256, 0, s, a);
    } else if (rows) {
      launch(kernel(0), blocks(rows), 256, 0, s, a);
    }
    copy(after, s);
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
  // (what the scores are multiplied by: infinite, or too small for all its bits, it would make every score undefined or rough)
  if (!std::isfinite(p.scale * kLog2e)) ops.refuse("the scale is too large");
  if (p.cap > 0.f && (!std::isfinite(p.cap * kLog2e) || !std::isnormal(p.scale / p.cap))) ops.refuse("the cap is too far from the scale");
  if (p.mask < B200_MASK_NONE || p.mask > B200_MASK_PREFIX) ops.refuse("unknown mask " + std::to_string(p.mask));
  if ((p.mask == B200_MASK_PREFIX) != (p.prefix.pool_id >= 0)) ops.refuse("'prefix' goes with the prefix mask");
  if (p.query_documents.pool_id >= 0 && p.key_documents.pool_id < 0) ops.refuse("documents of queries go with documents of keys");
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
  a.over = p.cap > 0.f ? p.scale / p.cap : 0.f;
  // (blocks are numbered by heads only where there are rows, and then less than 2^31 of them)
  a.heads = Divisor((unsigned int)a.H);
  a.key_heads = Divisor((unsigned int)a.HK);
  a.per_key_head = Divisor((unsigned int)a.group);
  const long long all = (long long)a.B * a.H;
  if (all >= 1 && all < (1ll << 31)) {
    a.all_heads = Divisor((unsigned int)all);
    a.all_key_heads = Divisor((unsigned int)a.B * (unsigned int)a.HK);
  }
  op->choose();
}

}  // namespace

extern "C" int b200_attention_link(b200_dev* dev, const b200_attention* p, b200_operator** out) {
  return link_operator<AttnOperator>(dev, p, out, [&](AttnOperator* op) { bind(*p, op, false); });
}

extern "C" int b200_attention_grad_link(b200_dev* dev, const b200_attention* p, b200_operator** out) {
  return link_operator<AttnOperator>(dev, p, out, [&](AttnOperator* op) { bind(*p, op, true); });
}
