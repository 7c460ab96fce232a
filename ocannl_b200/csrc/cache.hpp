// What the operators over a paged cache check at link: the cache's extents, its nodes, and the arguments that the kernels get of them.
#pragma once
#include "kernels/cache_terms.cuh"
#include "operators.hpp"

struct b200_tmap;

namespace b200 {

// The kernel of attention over a paged cache for many new tokens (op_cache_prompts.cu): of 16-bit types, for heads of up to 64 or 128 elements, one or two row
// tiles a block.
struct CacheAttnArgs;
struct CacheTileArgs;
struct CacheTiles {
  void (*kernel)(const b200_tmap, const b200_tmap, const b200_tmap, const CacheAttnArgs, const CacheTileArgs);
  unsigned int threads;
  size_t smem;
};
CacheTiles cache_tiles(int dtype, bool coded, bool wide, bool two);

// `written`: the caches and their scales are outputs
inline CacheArgs bind_cache(Operands& ops, const b200_cache& p, int dtype, bool written) {
  const bool coded = p.dtype == B200_E4M3;
  if (!coded && p.dtype != dtype) ops.refuse("the cache is of the new tokens' type or in 8 bits");
  const long long most = 1ll << 30;
  if (p.batch < 0 || p.batch > most || p.tokens < 0 || p.tokens > most) ops.refuse("batch and tokens must be between 0 and 2^30");
  if (p.pages < 0 || p.pages > most || p.max_pages < 0 || p.max_pages > most) ops.refuse("pages and max_pages must be between 0 and 2^30");
  if (p.page < 1 || p.page > (1 << 20)) ops.refuse("a page holds between 1 and 2^20 tokens");
  if (p.kv_heads < 1 || p.kv_heads > 65535) ops.refuse("kv_heads must be between 1 and 65535");
  if (p.d < 1) ops.refuse("d must be positive");
  if (coded != (p.k_scale.pool_id >= 0) || coded != (p.v_scale.pool_id >= 0)) ops.refuse("scales go with a cache in 8 bits");
  if (p.starts.pool_id < 0 && (p.batch ? p.tokens % p.batch : p.tokens) != 0) ops.refuse("without starts, tokens must be a multiple of batch");
  const unsigned long long count = extent_product({p.pages, p.kv_heads, p.page, p.d}, "cache"), scales = extent_product({p.pages, p.kv_heads}, "cache");
  const size_t size = coded ? 1 : dtype_bytes(dtype);
  auto node = [&](const b200_operand& o, const char* name, unsigned long long n, size_t elem, bool required) {
    return written ? ops.out(o, name, n, elem, required) : ops.in(o, name, n, elem, required);
  };
  CacheArgs c = {};
  c.k = (void*)node(p.k, "cache.k", count, size, true);
  c.v = (void*)node(p.v, "cache.v", count, size, true);
  c.k_scale = (float*)node(p.k_scale, "cache.k_scale", scales, 4, coded);
  c.v_scale = (float*)node(p.v_scale, "cache.v_scale", scales, 4, coded);
  c.pages = (const int*)ops.in(p.page_table, "page_table", extent_product({p.batch, p.max_pages}, "cache"), 4);
  c.lengths = (const int*)ops.in(p.lengths, "lengths", (unsigned long long)p.batch, 4);
  c.starts = (const int*)ops.in(p.starts, "starts", (unsigned long long)p.batch + 1, 4, false);
  c.n_pages = (unsigned int)p.pages;
  c.page = (unsigned int)p.page;
  c.max_pages = (unsigned int)p.max_pages;
  c.batch = (int)p.batch;
  c.tokens = (int)p.tokens;
  c.each = p.batch ? (int)(p.tokens / p.batch) : 0;
  c.HK = p.kv_heads;
  c.D = p.d;
  c.by_page = Divisor(c.page);
  return c;
}

}  // namespace b200
