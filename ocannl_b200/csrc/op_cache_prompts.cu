// The kernels of attention over a paged cache for many new tokens, apart from the operator that launches them: they take long to compile.
#include "cache.hpp"
#include "kernels/cache_attn_fwd_sm100.cuh"

namespace b200 {

namespace {

template <class T, int DP, int NQ, bool CODED>
CacheTiles of() {
  typedef CacheTileShape<DP, NQ, CODED> Sh;
  CacheTiles k = {cache_attention_tc<T, DP, NQ, CODED>, Sh::kThreads, Sh::kSmem};
  ready(k.kernel, k.smem);
  return k;
}
template <class T, int DP>
CacheTiles of(bool coded, bool two) {
  if (coded) return two ? of<T, DP, 2, true>() : of<T, DP, 1, true>();
  return two ? of<T, DP, 2, false>() : of<T, DP, 1, false>();
}

}  // namespace

CacheTiles cache_tiles(int dtype, bool coded, bool wide, bool two) {
  if (dtype == B200_BF16) return wide ? of<__nv_bfloat16, 128>(coded, two) : of<__nv_bfloat16, 64>(coded, two);
  return wide ? of<__half, 128>(coded, two) : of<__half, 64>(coded, two);
}

}  // namespace b200
