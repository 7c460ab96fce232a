// How the walk over all tiles of attention over a paged cache is dealt out to blocks: the rules that the host (grid and workspace, from what may come) and
// the blocks (from the lengths that have come) both follow.  Lengths are in 64s of tokens.
#ifndef B200_CACHE_PLAN_HPP
#define B200_CACHE_PLAN_HPP

#ifdef __CUDACC__
#define B200_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define B200_HOST_DEVICE inline
#endif

namespace b200 {

constexpr unsigned int kCachePart = 1024;     // of a block at most, a quarter of them a warp's: its accumulators' cut-off sums lose 2^-13 (see kSumKeys)

// a block's part of the walk: an even share of it, but no less than `least` (kCachePart at most) and no more than kCachePart
B200_HOST_DEVICE unsigned long long cache_quota(unsigned long long even, unsigned int least) {
  const unsigned long long q = even > least ? even : least;
  return q < kCachePart ? q : kCachePart;
}

struct CachePlan {
  unsigned int blocks;           // that fill the machine
  unsigned int least;            // of a block at least
  bool single;                   // a tile a block, whatever the lengths
  unsigned long long grid;       // blocks that a walk can ask for at most (not `single`)
};
// tiles of `capacity` 64s at most; `joined`: parts of a tile that are joined at once (more of them are in turns, from some 16 million tokens on)
inline CachePlan cache_plan(unsigned long long tiles, unsigned long long capacity, unsigned int blocks, unsigned int least, unsigned int joined) {
  CachePlan p = {};
  p.blocks = blocks;
  const unsigned long long wanted = capacity / (joined - 4) + 1, enough = wanted > least ? wanted : least;
  p.least = (unsigned int)(enough < kCachePart ? enough : kCachePart);
  p.single = capacity <= (unsigned long long)p.least + p.least / 2;
  // (more blocks only where an even share would be longer than a part may be; fewer where there is not that much)
  const unsigned __int128 walk = (unsigned __int128)tiles * capacity, cut = walk / kCachePart + 1, most = walk / p.least + 1;
  unsigned __int128 grid = cut > blocks ? cut : blocks;
  if (grid > most) grid = most;
  p.grid = grid >> 62 ? 1ull << 62 : (unsigned long long)grid;
  return p;
}

}  // namespace b200
#endif
