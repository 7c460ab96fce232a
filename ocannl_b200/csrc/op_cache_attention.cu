// Attention over a paged cache (b200_cache_attention_link): the choice of kernels and their launch.
#include <cmath>
#include <cstring>

#include "cache.hpp"
#include "kernels/cache_attn_any.cuh"
#include "kernels/cache_attn_few_sm100.cuh"
#include "kernels/cache_attn_fwd_sm100.cuh"
#include "kernels/cache_attn_terms.cuh"

using namespace b200;

namespace {

typedef void (*AnyKernel)(const CacheAttnArgs, const CacheFewArgs, int);
typedef void (*FewKernel)(const b200_tmap, const b200_tmap, const CacheAttnArgs, const CacheFewArgs);

// [dims[3]][dims[2]][dims[1]][dims[0]] elements in boxes of box[0] x box[1] x 1 x box[3]
b200_tmap box_map(const void* p, CUtensorMapDataType type, int size, const cuuint64_t (&dims)[4], const cuuint32_t (&box)[4], CUtensorMapSwizzle swizzle) {
  CUtensorMap map;
  const cuuint64_t strides[3] = {dims[0] * size, dims[0] * dims[1] * size, dims[0] * dims[1] * dims[2] * size};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = cu().cuTensorMapEncodeTiled_(&map, type, 4, (void*)p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                  swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(B200_E_UNSUPPORTED, "cache_attention: a node's layout cannot be described to the TMA unit (CUresult " + std::to_string((int)r) + ")");
  static_assert(sizeof(b200_tmap) == sizeof(CUtensorMap), "tensor map");
  b200_tmap m;
  memcpy(&m, &map, sizeof m);
  return m;
}

struct CacheAttnOperator : b200_operator {
  CacheAttnArgs a = {};
  int dtype = 0;
  bool coded = false;
  AnyKernel any = nullptr;
  int vec = 0;
  FewKernel few = nullptr;
  CacheFewArgs few_args = {};
  CacheTiles tiles = {};
  CacheTileArgs tile_args = {};
  b200_tmap map_q, map_k, map_v;
  unsigned int grid = 0;
  size_t smem = 0;
  int tile = 16, width = 0, resident = 1;      // rows of a tile, floats of a row of its parts, blocks of an SM

  template <class T>
  void set_any() { any = coded ? cache_attention_any<T, true> : cache_attention_any<T, false>; }
  template <class T, int DP, bool CODED, int NR>
  void set_few() {
    typedef CacheFewShape<DP, CODED, NR> Sh;
    few = a.c.page % 16 == 0 && a.c.n_pages ? cache_attention_few<T, DP, CODED, NR, true> : cache_attention_few<T, DP, CODED, NR, false>;
    smem = Sh::smem();
    tile = Sh::kRows;
    width = Sh::kWidth;
    resident = std::min<int>(Sh::kBlocks, 227 * 1024 / (Sh::smem() + 6 * 1024));
  }
  template <class T, int DP>
  void set_few(bool wide) {
    if (coded) wide ? set_few<T, DP, true, 2>() : set_few<T, DP, true, 1>();
    else wide ? set_few<T, DP, false, 2>() : set_few<T, DP, false, 1>();
  }
  unsigned int blocks_of(long long n) const {
    if (n >> 31) throw Error(B200_E_UNSUPPORTED, "cache_attention: too many rows");
    return (unsigned int)n;
  }
  // whole 16-byte pieces of rows
  bool pieces() const {
    bool ok = dtype != B200_F32 && a.c.D % (coded ? 16 : 8) == 0 && ((long long)a.c.tokens * a.group >> 31) == 0;
    for (const void* p : {a.q, (const void*)a.c.k, (const void*)a.c.v}) ok &= ((size_t)p & 15) == 0;
    return ok;
  }
  void choose() {
    const long long n = (long long)a.c.tokens * a.H;
    if (!n || !a.c.batch) return;
    if (pieces()) return many() ? choose_tiles() : choose_few();
    choose_any();
  }
  // Rows in tiles, whose tokens are dealt out evenly to as many blocks as the machine holds, `least` 64s of them at least.
  void choose_parts(int rows_of_tile, int floats, int blocks, int least) {
    const CacheArgs& c = a.c;
    // A sequence of n tokens has n group rows.
    const long long some = std::min(c.batch, c.tokens), tiles = ((long long)c.tokens * a.group + (rows_of_tile - 1) * some) / rows_of_tile * c.HK;
    const long long capacity = (std::min<long long>((long long)c.max_pages * c.page, 0x7fffffff) + 127) / 64;       // 64s
    const CachePlan plan = cache_plan(blocks_of(tiles), (unsigned long long)capacity, (unsigned int)(dev->sm_count * blocks), (unsigned int)least, kFewMost);
    few_args.blocks = plan.blocks;
    few_args.least = plan.least;
    few_args.enough = (unsigned int)dev->sm_count;
    // Short sequences: a tile a block.
    few_args.single = plan.single;
    few_args.by_group = Divisor((unsigned int)a.group);
    few_args.by_key_heads = Divisor((unsigned int)c.HK);
    if (few_args.single) {
      grid = blocks_of(tiles);
      if (!c.starts) {
        const long long each = ((long long)c.each * a.group + rows_of_tile - 1) / rows_of_tile * c.HK;
        few_args.by_units = Divisor(blocks_of(each));
        grid = blocks_of(each * c.batch);
      }
      return;
    }
    grid = blocks_of((long long)plan.grid);
    const size_t parts = ((size_t)grid + 1) * 2 * rows_of_tile * floats * 4;
    take_workspace(parts + (size_t)grid * 4);
    few_args.parts = (float*)workspace;
    few_args.tickets = (unsigned int*)(workspace + parts);
    cu_check(cu().cuMemsetD8Async_(workspace + parts, 0, (size_t)grid * 4, dev->stream), "cuMemsetD8Async(tickets)");
  }
  void choose_any() {
    const int size = coded ? 1 : (int)dtype_bytes(dtype), v = coded ? 4 : 16 / size;
    vec = a.c.D % v == 0;
    for (const void* p : {(const void*)a.c.k, (const void*)a.c.v}) vec &= ((size_t)p & 15) == 0;
    if (((long long)a.c.tokens * a.group) >> 31) throw Error(B200_E_UNSUPPORTED, "cache_attention: too many rows");
    if (dtype == B200_F32) set_any<float>();
    else if (dtype == B200_BF16) set_any<__nv_bfloat16>();
    else set_any<__half>();
    smem = any_smem(a.c.D);
    choose_parts(kAnyRows, kAnyWidth, (int)std::min<size_t>(6, 220 * 1024 / (smem + 7 * 1024)), 4);
    ready(any, smem);
  }
  // Tiles of 128 rows walk all their tokens in one block, some 0.85 us for 64 of them; tiles of 16 spread them over the machine, which gets through some
  // 18000 tokens of a tile in a us in 8 bits, 10000 else.  So there have to be tiles of 128 enough, and rows enough in them (measured, us by sixteens and by
  // 128s: 64 new tokens of 32 heads over 8 key heads and 8192 tokens, 8 bits, 31 and 108; 300 each of four sequences, 8 over 1, 4096, 8 bits, 70 and 56; 512 of 8 over
  // 8, 2048 tokens, 24 and 22; 64 each of eight, 32 over 8, 2048 tokens, 102 and 33).
  bool many() const {
    const CacheArgs& c = a.c;
    const bool boxes = c.n_pages && c.page % 16 == 0 && (c.page % 64 == 0 || 64 % c.page == 0);
    const long long rows = (long long)c.tokens * a.group;
    return boxes && a.group <= 128 && ((size_t)a.out & 15) == 0 && rows >= 32ll * std::min(c.batch, c.tokens) && rows * c.HK >= 128ll * (coded ? 72 : 32);
  }
  void choose_tiles() {
    const CacheArgs& c = a.c;
    tile_args.tokens = 128 / a.group;
    tile_args.box = c.page % 64 == 0 ? 64 : (int)c.page;
    tile_args.by_group = Divisor((unsigned int)a.group);
    tile_args.by_key_heads = Divisor((unsigned int)c.HK);
    const long long capacity = (long long)c.max_pages * c.page, some = std::min(c.batch, c.tokens);
    auto blocks = [&](int nq) { return (c.tokens + (nq * tile_args.tokens - 1) * some) / (nq * tile_args.tokens) * c.HK; };
    tile_args.sums = capacity > kSumKeys;
    // Two row tiles a block share their keys and wait in turn: they take hardly longer than one.  One a block where all blocks run at once that way, or there
    // are sums beside the accumulators.  (us, one and two: 700 tokens of 32 heads over 8 of 128, codes, 176 blocks and 88, 295 and 150; 1100 of heads of 64 in 16 bits, two
    // blocks of one tile an SM, 280 and 144, 137 and 166.)
    const long long about = (c.tokens + tile_args.tokens / 2 * some) / tile_args.tokens * c.HK;
    const bool two = !tile_args.sums && about > (long long)dev->sm_count * (c.D <= 64 && !coded ? 2 : 1);
    tiles = cache_tiles(dtype, coded, c.D > 64, two);
    grid = blocks_of(blocks(two ? 2 : 1));
    const cuuint64_t of_q[4] = {(cuuint64_t)c.D, (cuuint64_t)a.group, (cuuint64_t)c.HK, (cuuint64_t)c.tokens};
    const cuuint32_t box_q[4] = {64, (cuuint32_t)a.group, 1, (cuuint32_t)tile_args.tokens};
    map_q = box_map(a.q, type(), 2, of_q, box_q, CU_TENSOR_MAP_SWIZZLE_128B);
    // (codes are made halves where they lie: rows one behind the other)
    cache_maps(tile_args.box, coded ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B);
  }
  CUtensorMapDataType type() const { return dtype == B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }
  void cache_maps(int rows, CUtensorMapSwizzle swizzle) {
    const CacheArgs& c = a.c;
    const cuuint64_t of_c[4] = {(cuuint64_t)c.D, c.page, (cuuint64_t)c.HK, c.n_pages};
    const cuuint32_t box_c[4] = {coded && c.D > 64 ? 128u : 64u, (cuuint32_t)rows, 1, 1};
    map_k = box_map(c.k, coded ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type(), coded ? 1 : 2, of_c, box_c, swizzle);
    map_v = box_map(c.v, coded ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type(), coded ? 1 : 2, of_c, box_c, swizzle);
  }
  void choose_few() {
    const CacheArgs& c = a.c;
    // (rows of a sequence, on average: up to 8 take tiles of 8)
    const bool wide = (long long)c.tokens * a.group > 8ll * std::min(c.batch, c.tokens);
    if (dtype == B200_BF16) c.D <= 64 ? set_few<__nv_bfloat16, 64>(wide) : set_few<__nv_bfloat16, 128>(wide);
    else c.D <= 64 ? set_few<__half, 64>(wide) : set_few<__half, 128>(wide);
    choose_parts(tile, width, resident, 4);
    // (one box a step; codes of heads of up to 64 elements have rows of 64 bytes)
    if (c.page % 16 == 0 && c.n_pages) cache_maps(16, coded && c.D <= 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    ready(few, smem);
  }
  void run(cudaStream_t s) override {
    if (!grid) return;
    if (tiles.kernel) launch(tiles.kernel, dim3(grid), tiles.threads, tiles.smem, s, map_q, map_k, map_v, a, tile_args);
    else if (few) launch(few, dim3(grid), kCacheFewThreads, smem, s, map_k, map_v, a, few_args);
    else launch(any, dim3(grid), kCacheFewThreads, smem, s, a, few_args, vec);
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
