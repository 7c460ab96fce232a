// Attention of new tokens over a paged cache, 16-bit heads, 8 or 16 rows at a time: the next tokens of sequences, and ragged batches of them.
//
// The keys and values are read once and bound it.  The query heads that share a key head, and their tokens, are the columns of mma.m16n8k16 (tcgen05
// has no tile of 8 or 16 rows): scores' = K q', 16 tokens at a time, and out' = V' weights', so that 8 rows, as many as heads usually share a key, waste
// nothing, and take half the registers and products of a tile of 16.  A product does not care in which order its elements are added, so the order is
// chosen for the loads: of the 16 elements of a step each of the four lanes that share a token has four neighbours, and the rows of the second product
// are dealt out as neighbours to a lane too, so that every operand is read as whole 16-byte pieces by the lane that multiplies it.  A warp's ring is
// its own, with no barrier between warps: pages that hold whole steps of 16 tokens arrive as boxes of the TMA unit, two or four a step (64
// sequences of up to 8192, 32 heads over 8 of 128, codes: 145 us, 5.5 TB/s; by 16-byte copies of all lanes 182, and 183 without the products), others by cp.async.  Codes of 8 bits become halves in registers, two to an instruction; a transposed pair of values is one byte
// permutation, and the weights turn from scores' to operand's layout by a transpose of 8 x 8 between lanes.  Codes are multiplied as they are: a
// page's scale of the keys goes onto its scores, the logarithm of its scale of the values onto the exponents of its weights, which the row's sum takes off
// again: out = sum w code / sum (w / scale), so that weights stay in the range of a half whatever the scales.  (bfloat16 queries beside codes become
// halves too, each row multiplied by the power of two that brings its largest to 2^14.)
//
// The tokens that all tiles see (with a window: the sinks' and the window's, as one range), tile behind tile, are one long walk, of which every block takes
// an equal part: the end of one tile, some whole ones, the beginning of another.  Every block finds its part from the lengths of all sequences, so that sequences
// of all lengths fill the machine evenly, in one round of blocks.  (Chunks of a tile a block, three rounds of them, with copies of all lanes: 193 us, parts 182.)  The
// block of a tile that comes last joins its parts in their order: the same bits whoever comes last.
#ifndef B200_CACHE_ATTN_FEW_SM100_CUH
#define B200_CACHE_ATTN_FEW_SM100_CUH
#include "../cache_plan.hpp"
#include "attn_few_sm100.cuh"
#include "cache_attn_terms.cuh"

namespace b200 {

struct CacheFewArgs {
  float* parts;            // [block][2][rows of a tile][DP + 4]: output (not divided), maximum, sum; of the tile that begins ahead of the block's part, then of
                           // the one that ends behind it
  unsigned int* tickets;   // [block], zero between runs: of the tile that begins in a block and ends in another
  unsigned int blocks;     // that fill the machine
  unsigned int least;      // 64s of tokens of a block at least
  unsigned int enough;     // tiles that need not be cut for the machine to be busy
  int single;              // a tile a block, whatever the lengths
  Divisor by_group, by_key_heads, by_units;     // by_units: without starts, tiles of a sequence (single)
};

constexpr int kCacheFewWarps = 4, kCacheFewThreads = 32 * kCacheFewWarps;
constexpr unsigned int kCacheShort = 24;      // 64s of tokens, at most, of tiles that are not cut (32 sequences with a window of 1024: 25 us, 27 cut)

template <int DP, bool CODED, int NR>
struct CacheFewShape {
  static constexpr int kRows = 8 * NR;
  static constexpr int kPerKey = CODED ? DP / 64 : DP / 32;            // 16-byte pieces of a key that a lane has
  static constexpr int kValueBytes = CODED ? DP / 8 : DP / 4;          // bytes of a value that a lane has
  static constexpr int kValueWidth = kValueBytes < 16 ? kValueBytes : 16, kPerValue = kValueBytes / kValueWidth;
  static constexpr int kKeys = 2 * kPerKey * 512, kValues = 4 * kPerValue * 32 * kValueWidth;
  static constexpr int kStage = kKeys + kValues;                       // bytes of a warp
  static constexpr int kStages = kStage <= 4096 ? 4 : 3;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kWidth = DP + 4;
  static constexpr int kJoin = kCacheFewWarps * kRows * kWidth * 4;
  static constexpr int smem() { return 1024 + (kCacheFewWarps * kRing > kJoin ? kCacheFewWarps * kRing : kJoin); }     // (boxes lie on 1024 bytes)
  static constexpr int kLine = DP * (CODED ? 1 : 2) < 128 ? DP * (CODED ? 1 : 2) : 128, kPanels = DP * (CODED ? 1 : 2) / kLine;   // a box: 16 rows of so many bytes
  static constexpr int kBlocks = kStage > 4096 ? 2 : NR == 1 && DP == 64 ? 4 : 3;      // of an SM
};

// BYTES from memory, of which those behind `bytes` are zeros
template <int BYTES>
__device__ __forceinline__ void copy_in(unsigned int dst, const void* src, int bytes) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 from_shared16(unsigned int at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 from_shared8(unsigned int at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}

// 8 x 8 values of 16 bits, two to a lane, transposed between the lanes
__device__ __forceinline__ unsigned int transpose8(unsigned int x) {
  unsigned int y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// What a sequence's tiles look at: its rows of a key head, in tiles, and no fewer 64s of tokens than any of them sees, as they are walked
struct CacheWalk {
  unsigned int tiles, length;
};
template <int ROWS>
__device__ __forceinline__ CacheWalk cache_walk(const CacheAttnArgs& a, const CacheSeq& s) {
  CacheWalk w;
  w.tiles = ((unsigned int)s.count * (unsigned int)a.group + (ROWS - 1)) / ROWS * (unsigned int)a.c.HK;
  long long n = (long long)cache_last(a, s.pos0 + s.count - 1) + 1;
  if (a.window) n = min(n, (long long)a.window + ((a.sinks + 15ll) & ~15ll) + ROWS / a.group + 17);
  w.length = (unsigned int)((max(n, 1ll) + 63) / 64);
  return w;
}

// A block's part of the walk over all tiles: where it begins, and how much is left of it.
struct CachePart {
  int b;
  unsigned int tile, at, left;         // tile of the sequence (key heads beside each other); 64s
  unsigned long long ahead, quota;     // of the sequence: 64s of the sequences before it; a block's part
  CacheSeq s;
  CacheWalk walk;
  bool whole;                          // no tile is cut: a walk of tiles, each of length 1
};
// A piece of a tile: which rows of a key head, and which of the tokens that they see.
struct CachePiece {
  int hk, first_row, rows;             // rows of the tile that there are
  int least_pos, most_pos, end;        // positions of its rows; tokens that some row sees lie before `end`
  int sink_end, shift;                 // the walk: tokens 0 .. sink_end - 1, then those from sink_end + shift on
  int begin, stop;                     // of the walk, this piece's
  unsigned int parts, part, first_block;     // of the tile
  bool meets;                          // all its parts' blocks are in the grid (starts that fall may ask for more: such a tile is left, and takes no tickets)
  __device__ __forceinline__ int token_of(int v) const { return v < sink_end ? v : v + shift; }
};
// a part's place: of the tile that begins in `first_block`
__device__ __forceinline__ long long cache_part_at(unsigned int first_block, unsigned int part) { return ((long long)first_block + part) * 2 + (part == 0 ? 1 : 0); }

// (64-bit quotients take some 100 instructions, and walks are hardly ever that long)
__device__ __forceinline__ unsigned long long quotient(unsigned long long n, unsigned long long d) {
  return (n | d) >> 32 ? n / d : (unsigned long long)((unsigned int)n / (unsigned int)d);
}

template <int NT, int ROWS>
__device__ __forceinline__ bool cache_part(const CacheAttnArgs& a, const CacheFewArgs& f, CachePart& p) {
  const CacheArgs& c = a.c;
  if (f.single) {
    unsigned int nth;
    if (c.starts) {
      if (!find_unit<NT>(c.batch, blockIdx.x, [&](int i) { return cache_walk<ROWS>(a, cache_seq(c, i)).tiles; }, p.b, nth)) return false;
    } else {
      p.b = (int)f.by_units.of(blockIdx.x);
      nth = blockIdx.x - (unsigned int)p.b * f.by_units.d;
      if (p.b >= c.batch) return false;
    }
    p.s = cache_seq(c, p.b);
    p.walk = cache_walk<ROWS>(a, p.s);
    p.tile = nth;
    p.at = 0;
    p.left = p.walk.length;
    p.ahead = p.quota = 0;
    p.whole = false;
    return true;
  }
  __shared__ unsigned long long sums[2][NT / 32], found[2];
  __shared__ unsigned int longest_of[NT / 32];
  const unsigned int lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  // of NT sequences from i0 on: 64s and tiles, this thread's, those before it, and added to all
  auto sums_of = [&](int i0, unsigned long long& all, unsigned long long& tiles, unsigned long long& mine, unsigned long long& mine_tiles, unsigned long long& before,
                     unsigned long long& before_tiles, unsigned int& longest) {
    unsigned int length = 0;
    const int i = i0 + (int)threadIdx.x;
    mine = mine_tiles = 0;
    if (i < c.batch) {
      const CacheSeq s = cache_seq(c, i);
      if (s.count) {
        const CacheWalk w = cache_walk<ROWS>(a, s);
        mine_tiles = w.tiles;
        length = w.length;
        mine = mine_tiles * length;
      }
    }
    unsigned long long up_to[2] = {mine, mine_tiles};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, up_to[k], o);
        if (lane >= (unsigned int)o) up_to[k] += x;
      }
    __syncthreads();
    length = __reduce_max_sync(0xffffffffu, length);
    if (lane == 31) sums[0][warp] = up_to[0], sums[1][warp] = up_to[1], longest_of[warp] = length;
    __syncthreads();
    before = all + up_to[0] - mine;
    before_tiles = tiles + up_to[1] - mine_tiles;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      if (w < (int)warp) before += sums[0][w], before_tiles += sums[1][w];
      all += sums[0][w];
      tiles += sums[1][w];
      longest = max(longest, longest_of[w]);
    }
  };
  // the whole walk, and its tiles; with a sequence a thread, one look at the lengths finds the block's own place as well
  unsigned long long all = 0, tiles = 0, mine = 0, mine_tiles = 0, before = 0, before_tiles = 0;
  unsigned int longest = 0;
  for (int i0 = 0; i0 < c.batch; i0 += NT) {
    sums_of(i0, all, tiles, mine, mine_tiles, before, before_tiles, longest);
  }
  // Short tiles, and enough of them for the machine: none is cut (32 sequences of 8 key heads, 1044 tokens each: 25.8 us, 27.2 cut).
  p.whole = tiles >= f.enough && longest <= kCacheShort;
  if (p.whole) {
    all = tiles;
    mine = mine_tiles;
    before = before_tiles;
  }
  p.quota = quotient(all + f.blocks - 1, f.blocks);
  if (!p.whole) p.quota = cache_quota(p.quota, f.least);
  const unsigned long long from = p.quota * blockIdx.x;
  if (from >= all) return false;
  if (c.batch <= NT) {
    if (before <= from && from < before + mine) {
      found[0] = threadIdx.x;
      found[1] = before;
    }
  } else {
    unsigned long long sum = 0, sum_tiles = 0;
    for (int i0 = 0; i0 < c.batch; i0 += NT) {
      sums_of(i0, sum, sum_tiles, mine, mine_tiles, before, before_tiles, longest);
      if (p.whole) {
        mine = mine_tiles;
        before = before_tiles;
      }
      if (before <= from && from < before + mine) {
        found[0] = (unsigned long long)(i0 + (int)threadIdx.x);
        found[1] = before;
      }
    }
  }
  __syncthreads();
  p.b = (int)found[0];
  p.ahead = found[1];
  p.s = cache_seq(c, p.b);
  p.walk = cache_walk<ROWS>(a, p.s);
  if (p.whole) p.walk.length = 1;
  const unsigned long long rest = from - p.ahead;
  p.tile = (unsigned int)quotient(rest, p.walk.length);
  p.at = (unsigned int)(rest - (unsigned long long)p.tile * p.walk.length);
  p.left = (unsigned int)min(p.quota, all - from);
  return true;
}
// the next piece of the part; false: there is none
template <int ROWS>
__device__ __forceinline__ bool cache_piece(const CacheAttnArgs& a, const CacheFewArgs& f, CachePart& p, CachePiece& piece) {
  const CacheArgs& c = a.c;
  if (!p.left) return false;
  const unsigned int take = min(p.left, p.walk.length - p.at), tile = f.by_key_heads.of(p.tile);
  piece.hk = (int)(p.tile - tile * (unsigned int)c.HK);
  piece.first_row = (int)tile * ROWS;
  piece.rows = min(ROWS, p.s.count * a.group - piece.first_row);
  piece.least_pos = p.s.pos0 + (int)f.by_group.of((unsigned int)piece.first_row);
  piece.most_pos = p.s.pos0 + (int)f.by_group.of((unsigned int)(piece.first_row + piece.rows - 1));
  piece.end = cache_last(a, piece.most_pos) + 1;
  piece.sink_end = piece.shift = 0;
  if (a.window) {
    piece.sink_end = (int)min(((long long)min(a.sinks, max(piece.end, 0)) + 15) & ~15ll, 0x7ffffff0ll);
    piece.shift = max((cache_first(a, piece.least_pos) & ~15) - piece.sink_end, 0);
  }
  const int n_tokens = piece.shift ? max(piece.end - piece.shift, piece.sink_end) : max(piece.end, 0);       // (the window may lie behind the last page)
  piece.begin = (int)min((long long)p.at * 64, (long long)n_tokens);
  piece.stop = p.whole ? n_tokens : (int)min((long long)(p.at + take) * 64, (long long)n_tokens);
  piece.parts = 1;
  piece.part = 0;
  piece.first_block = blockIdx.x;
  piece.meets = true;
  if (take < p.walk.length) {
    const unsigned long long from = p.ahead + (unsigned long long)p.tile * p.walk.length;
    piece.first_block = (unsigned int)quotient(from, p.quota);
    piece.parts = (unsigned int)quotient(from + p.walk.length - 1, p.quota) - piece.first_block + 1;
    piece.part = blockIdx.x - piece.first_block;
    piece.meets = (unsigned long long)piece.first_block + piece.parts <= gridDim.x;
  }
  return true;
}
// ... and on behind it
template <int ROWS>
__device__ __forceinline__ void cache_advance(const CacheAttnArgs& a, CachePart& p) {
  p.left -= min(p.left, p.walk.length - p.at);
  p.at = 0;
  if (!p.left || ++p.tile < p.walk.tiles) return;
  p.tile = 0;
  p.ahead += (unsigned long long)p.walk.tiles * p.walk.length;
  do {
    p.s = cache_seq(a.c, ++p.b);
  } while (!p.s.count && p.b + 1 < a.c.batch);
  p.walk = cache_walk<ROWS>(a, p.s);
  if (p.whole) p.walk.length = 1;
}

// The parts of a row: the first lies a place behind the others' line, (2 k - 1) places on for k > 0
template <int DP, int R>
__device__ __forceinline__ const float* cache_part_row(const float* first, int k) { return first + (k ? (2 * k - 1) : 0) * (long long)(R * (DP + 4)); }
// what a part counts for beside the largest maximum: see few_weigh.  `ex`: a weight from a difference in the scores' unit
template <class Ex>
__device__ __forceinline__ float cache_part_weight(Ex ex, float part_top, float part_sum, float top) {
  return part_sum == 0.f ? 0.f : part_top == -INFINITY ? 1.f : ex(part_top - top);
}
// the maximum and sum of n of them (kFewMost at most) from k0 on, and in `weight` what each is multiplied by: a warp
template <int DP, int R, class Ex>
__device__ __forceinline__ void cache_weigh(Ex ex, const float* first, int k0, int n, float* weight, float& top, float& sum) {
  const unsigned int lane = threadIdx.x & 31u;
  float t[kFewMost / 32], u[kFewMost / 32];
  top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kFewMost / 32; ++k) {
    const int i = (int)lane + 32 * k;
    t[k] = -INFINITY;
    u[k] = 0.f;
    if (i < n) {
      const float* row = cache_part_row<DP, R>(first, k0 + i);
      t[k] = row[DP];
      u[k] = row[DP + 1];
    }
    top = fmaxf(top, t[k]);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  sum = 0.f;
  __syncwarp();                     // (all lanes have read the weights of the row before)
#pragma unroll
  for (int k = 0; k < kFewMost / 32; ++k) {
    const float w = cache_part_weight(ex, t[k], u[k], top);
    if ((int)lane + 32 * k < n) weight[lane + 32 * k] = w;
    if (w != 0.f) sum = fmaf(w, u[k], sum);
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  __syncwarp();
}
// four elements of their weighed sum, in their order; eight loads under way together
template <int DP, int R>
__device__ __forceinline__ float4 cache_gather(const float* first, int k0, int n, const float* weight, int e) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < n; i += 8) {
    float4 x[8];
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int at = i + k;
      w[k] = at < n ? weight[at] : 0.f;
      x[k] = *(const float4*)(cache_part_row<DP, R>(first, k0 + (at < n ? at : i)) + e);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (w[k] != 0.f) v = make_float4(fmaf(w[k], x[k].x, v.x), fmaf(w[k], x[k].y, v.y), fmaf(w[k], x[k].z, v.z), fmaf(w[k], x[k].w, v.w));
  }
  return v;
}
// A row of any number of parts by a warp: its maximum and sum, and elements e .. e + 3 (none where `on` is not set).  More than kFewMost, which only
// sequences of some 16 million tokens have, are joined in turns, each to what the turns before have come to.
template <int DP, int R, class Ex>
__device__ __forceinline__ float4 cache_join(Ex ex, const float* first, int n, float* weight, bool on, int e, float& top, float& sum) {
  const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
  cache_weigh<DP, R>(ex, first, 0, min(n, kFewMost), weight, top, sum);
  float4 v = on ? cache_gather<DP, R>(first, 0, min(n, kFewMost), weight, e) : none;
  for (int k0 = kFewMost; k0 < n; k0 += kFewMost) {
    float t, u;
    cache_weigh<DP, R>(ex, first, k0, min(n - k0, kFewMost), weight, t, u);
    const float4 x = on ? cache_gather<DP, R>(first, k0, min(n - k0, kFewMost), weight, e) : none;
    const float next = fmaxf(top, t), by = cache_part_weight(ex, top, sum, next), w = cache_part_weight(ex, t, u, next);
    v = by != 0.f ? make_float4(v.x * by, v.y * by, v.z * by, v.w * by) : none;
    sum = by != 0.f ? sum * by : 0.f;
    if (w != 0.f) {
      v = make_float4(fmaf(w, x.x, v.x), fmaf(w, x.y, v.y), fmaf(w, x.z, v.z), fmaf(w, x.w, v.w));
      sum = fmaf(w, u, sum);
    }
    top = next;
  }
  return v;
}

// Writes four elements of a row and, with the first, its lse; false: one is infinite or undefined, and the row has to be done again
template <class T>
__device__ __forceinline__ bool cache_finish(const CacheAttnArgs& a, int row, int h, int e, const float4& v, float top, float sum, float lift) {
  const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const float y[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
  const long long at = (long long)row * a.H + h;
  T* to = (T*)a.out + at * a.c.D + e;
  bool fine = true;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (e + k < a.c.D) {
      from_float(y[k], to[k]);
      fine = fine && y[k] * 0.f == 0.f;
    }
  if (e == 0 && a.lse) a.lse[at] = by != 0.f ? (top - lift + log2f(sum)) * kCacheLn2 : -INFINITY;
  return fine;
}

// WHOLE: pages hold a multiple of 16 tokens, so that a step's tokens lie in one
template <class T, int DP, bool CODED, int NR, bool WHOLE>
__global__ void __launch_bounds__(kCacheFewThreads, (CacheFewShape<DP, CODED, NR>::kBlocks)) cache_attention_few(const __grid_constant__ b200_tmap map_k,
                                                                                                               const __grid_constant__ b200_tmap map_v,
                                                                                                               const __grid_constant__ CacheAttnArgs a,
                                                                                                               const __grid_constant__ CacheFewArgs f) {
  typedef CacheFewShape<DP, CODED, NR> Sh;
  typedef typename std::conditional<CODED, __half, T>::type M;          // what is multiplied
  constexpr int KS = DP / 16, W = Sh::kWidth, R = Sh::kRows;
  constexpr float kUp = kLift<M>;
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ unsigned int last_block;
  __shared__ unsigned long long arrived[kCacheFewWarps][Sh::kStages];
  __shared__ volatile unsigned int abort_flag;
  const CacheArgs& c = a.c;
  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, q4 = lane & 3u;
  const unsigned int dyn_at = (b200_smem_addr(dyn) + 1023u) & ~1023u, bars = b200_smem_addr(arrived[warp]);
  unsigned char* const gen = dyn + (dyn_at - b200_smem_addr(dyn));
  if constexpr (WHOLE) {
    if (lane < (unsigned int)Sh::kStages) b200_mbar_init(bars + 8 * lane, 1);
    if (threadIdx.x == 0) abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
  }
  grid_begin();
  unsigned int filled = 0, taken = 0;                  // steps that this warp has asked for, and used

  CachePart part;
  if (!cache_part<kCacheFewThreads, R>(a, f, part)) return;
  CachePiece plan;
  for (; cache_piece<R>(a, f, part, plan); cache_advance<R>(a, part)) {
  const CacheSeq s = part.s;
  const int b = part.b, hk = plan.hk, first_row = plan.first_row, rows = plan.rows, end = plan.end, v_begin = plan.begin, v_end = plan.stop;
  auto query_of = [&](int i) { return (int)f.by_group.of((unsigned int)(first_row + i)); };
  auto head_of = [&](int i) { return hk * a.group + first_row + i - query_of(i) * a.group; };
  // (this lane's columns are rows 8 r + 2 q4 and the next one)
  const int all_see = cache_last(a, plan.least_pos), all_from = cache_first(a, plan.most_pos);

  // ---- the queries as the B operand, in the order of the keys' pieces: row 8 r + g.  Under way before the pages are looked up.
  unsigned int q[NR][KS][2];
  float unit[NR][2];                                 // what a column's products have to be multiplied by
  {
    constexpr int kRun = CODED ? 16 : 8;             // neighbouring elements of a lane
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int i = (int)g + 8 * r;
      const bool on = i < rows;
      const unsigned short* from = (const unsigned short*)a.q + (on ? ((long long)(s.first + query_of(i)) * a.H + head_of(i)) * c.D : 0);
#pragma unroll
      for (int p = 0; p < DP / (4 * kRun); ++p)
#pragma unroll
        for (int t = 0; t < kRun / 8; ++t) {
          const int e = p * 4 * kRun + (int)q4 * kRun + t * 8, ks = p * (kRun / 4) + 2 * t;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (on && e < c.D) v = *(const uint4*)(from + e);
          q[r][ks][0] = v.x;
          q[r][ks][1] = v.y;
          q[r][ks + 1][0] = v.z;
          q[r][ks + 1][1] = v.w;
        }
    }
  }

  // ---- the ring: steps of 16 tokens, every fourth of them this warp's
  const unsigned int ring = dyn_at + warp * Sh::kRing;
  const int steps = v_end > v_begin ? (v_end - v_begin + 15) / 16 : 0;
  const int mine = steps > (int)warp ? (steps - (int)warp + kCacheFewWarps - 1) / kCacheFewWarps : 0;
  auto token_of = [&](int n) { return plan.token_of(v_begin + ((int)warp + n * kCacheFewWarps) * 16); };
  auto page_of = [&](int j) { return cache_page_at(c, b, c.by_page.of((unsigned int)j)); };
  constexpr int kSize = CODED ? 1 : 2;
  const unsigned char *const keys = (const unsigned char*)c.k, *const values = (const unsigned char*)c.v;
  const int line = c.D * kSize;                      // bytes of a row
  // bytes that this lane takes at its keys' and its values' pieces (none behind the head's end)
  auto key_bytes = [&](int p) { return (int)q4 * 16 + p * 64 < line ? 16 : 0; };
  auto value_bytes = [&](int p) { return (int)g * Sh::kValueBytes + p * 16 < line ? Sh::kValueWidth : 0; };
  // WHOLE: the pages of 32 steps, a lane each (-1: none), their slots there, and their pages' scales; and the same of the 32 steps behind them
  int where[2] = {-1, -1}, slots[2] = {0, 0};
  struct Scales {
    float down, back, raise;                         // of the keys; of the values its inverse and its logarithm
    __device__ __forceinline__ void of(const CacheArgs& c, long long at) {
      down = cache_scale(__ldg(c.k_scale + at));
      const float v = cache_scale(__ldg(c.v_scale + at));
      back = rcp(v);
      asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(raise) : "f"(v));
    }
  } scales[2] = {{1.f, 1.f, 0.f}, {1.f, 1.f, 0.f}};
  auto look = [&](int n0, int k) {
    const int n = n0 + (int)lane;
    where[k] = -1;
    if (n >= mine) return;
    const int j = token_of(n);
    const unsigned int index = c.by_page.of((unsigned int)j);
    const int page = cache_page_at(c, b, index);
    where[k] = page;
    slots[k] = (int)((unsigned int)j - index * c.page);
    if (CODED && page >= 0) scales[k].of(c, (long long)page * c.HK + hk);
  };
  if (WHOLE) {
    look(0, 0);
    if (mine > 32) look(32, 1);
  }
  int first_of = 0;                                  // the step that where[0] begins with
  auto fetch = [&](int n) {
    if (n < mine) {
      const unsigned int to = filled++ % Sh::kStages;
      if constexpr (WHOLE) {
        const bool near = n - first_of < 32;
        const int page = __shfl_sync(0xffffffffu, near ? where[0] : where[1], n & 31), at = __shfl_sync(0xffffffffu, near ? slots[0] : slots[1], n & 31);
        if (b200_elect()) {
          const unsigned int bar = bars + 8 * to, dst = ring + to * Sh::kStage;
          b200_mbar_expect_tx(bar, Sh::kStage);
          // (no page: a box outside the cache, zeros)
#pragma unroll
          for (int p = 0; p < Sh::kPanels; ++p) {
            b200_tma_load_4d(dst + p * 16 * Sh::kLine, &map_k, bar, p * 64, at, hk, page < 0 ? (int)c.n_pages : page);
            b200_tma_load_4d(dst + Sh::kKeys + p * 16 * Sh::kLine, &map_v, bar, p * 64, at, hk, page < 0 ? (int)c.n_pages : page);
          }
        }
      } else {
        const int j0 = token_of(n);
        const unsigned int at_k = ring + to * Sh::kStage + lane * 16, at_v = ring + to * Sh::kStage + Sh::kKeys + lane * Sh::kValueWidth;
        // byte of a token's row, -1: not there
        auto place = [&](int j) -> long long {
          if (j >= end) return -1;
          const unsigned int index = c.by_page.of((unsigned int)j);
          const int p = cache_page_at(c, b, index);
          return p < 0 ? -1 : (cache_at(c, p, hk) + (long long)((unsigned int)j - index * c.page) * c.D) * kSize;
        };
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const long long from = place(j0 + (int)g + 8 * k);
#pragma unroll
          for (int p = 0; p < Sh::kPerKey; ++p) {
            const int bytes = from >= 0 ? key_bytes(p) : 0;
            copy_in<16>(at_k + (k * Sh::kPerKey + p) * 512, keys + (bytes ? from + (int)q4 * 16 + p * 64 : 0), bytes);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const long long from = place(j0 + (int)q4 * 2 + (k & 1) + 8 * (k >> 1));
#pragma unroll
          for (int p = 0; p < Sh::kPerValue; ++p) {
            const int bytes = from >= 0 ? value_bytes(p) : 0;
            copy_in<Sh::kValueWidth>(at_v + (k * Sh::kPerValue + p) * 32 * Sh::kValueWidth, values + (bytes ? from + (int)g * Sh::kValueBytes + p * 16 : 0), bytes);
          }
        }
      }
    }
    if (!WHOLE) asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < Sh::kStages - 1; ++i) fetch(i);

  // (their conversion, once the first copies are under way)
  {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float mine_unit = 1.f;
      if constexpr (CODED && std::is_same<T, __nv_bfloat16>::value) {
        unsigned int most = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int k = 0; k < 2; ++k) most = max(most, max(q[r][ks][k] & 0x7fffu, (q[r][ks][k] >> 16) & 0x7fffu));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the exponent of the largest, which goes to 14 (none for zeros, and for what is infinite or undefined)
        const int e = (int)(most >> 7);
        const int up = e == 0 || e == 255 ? 0 : min(max(127 + 14 - e, -126), 126);
        const float by = power_of_two(up);
        mine_unit = power_of_two(-up);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = unpack2(q[r][ks][k], __nv_bfloat16());
            q[r][ks][k] = pack2(x.x * by, x.y * by, __half());
          }
      }
      mine_unit *= a.cap > 0.f ? a.over : a.scale * kCacheLog2e;
#pragma unroll
      for (int k = 0; k < 2; ++k) unit[r][k] = __shfl_sync(0xffffffffu, mine_unit, (2 * q4 + k) * 4);
    }
  }
  const float to_log2 = a.cap * kCacheLog2e;
  int pos[NR][2];
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = 8 * r + 2 * (int)q4 + k;
      pos[r][k] = s.pos0 + query_of(min(i, rows - 1));       // (rows behind the last are columns that nobody reads)
    }

  // element g * DP / 8 + 2 i + (k >> 1) of column k & 1 is o[r][i][k]
  float o[NR][DP / 16][4], m[NR][2], l[NR][2], limit[NR][2], off[NR][2];       // (the maximum in use, what outgrows it, what is taken off)
#pragma unroll
  for (int r = 0; r < NR; ++r) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[r][i][k] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) m[r][k] = limit[r][k] = -INFINITY, l[r][k] = off[r][k] = 0.f;
  }

  // (not WHOLE: of this lane's tokens g and g + 8 of the step at hand, a step ahead)
  bool there[2] = {false, false};
  auto look_at = [&](int n) {
    if (n >= mine) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = token_of(n) + (int)g + 8 * k, page = j < end ? page_of(j) : -1;
      there[k] = page >= 0;
      if (CODED && page >= 0) scales[k].of(c, (long long)page * c.HK + hk);
    }
  };
  if (!WHOLE) look_at(0);
  // where a lane's pieces lie in a stage: boxes swizzled by the copies, or a piece of all lanes behind the other
  auto box_at = [&](unsigned int row, unsigned int byte) {
    const unsigned int chunk = byte % Sh::kLine / 16, turn = Sh::kLine == 128 ? row & 7u : row >> 1 & 3u;
    return byte / Sh::kLine * (16 * Sh::kLine) + row * Sh::kLine + ((chunk ^ turn) << 4) + byte % 16;
  };
  bool live = true;
  for (int n = 0; n < mine && live; ++n) {
    const int j0 = token_of(n);
    if (WHOLE && n - first_of == 32) {
      // (copies are at most a few steps ahead: in the second 32)
      first_of = n;
      where[0] = where[1];
      slots[0] = slots[1];
      scales[0] = scales[1];
      if (mine - n > 32) look(n + 32, 1);
    }
    const bool here[2] = {WHOLE ? __shfl_sync(0xffffffffu, (int)(where[0] >= 0), n & 31) != 0 : there[0], there[1]};
    float down[2] = {1.f, 1.f}, back[2] = {1.f, 1.f}, raise[2] = {0.f, 0.f};
    if constexpr (CODED) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const Scales& of = scales[WHOLE ? 0 : k];
        if (WHOLE && k == 1) {
          down[1] = down[0], back[1] = back[0], raise[1] = raise[0];
        } else {
          down[k] = WHOLE ? __shfl_sync(0xffffffffu, of.down, n & 31) : of.down;
          back[k] = WHOLE ? __shfl_sync(0xffffffffu, of.back, n & 31) : of.back;
          raise[k] = WHOLE ? __shfl_sync(0xffffffffu, of.raise, n & 31) : of.raise;
        }
      }
    }
    if (!WHOLE) look_at(n + 1);
    const unsigned int slot = taken % Sh::kStages, stage = ring + slot * Sh::kStage;
    if constexpr (WHOLE) {
      live = b200_wait(bars + 8 * slot, taken / Sh::kStages & 1u, &abort_flag, a.status, 81u);
      live = __all_sync(0xffffffffu, live);         // (and all lanes have read the step before)
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(Sh::kStages - 2) : "memory");
    }
    ++taken;
    if (live) fetch(n + Sh::kStages - 1);           // into the slot of the step before
    if (!live) break;
    if (WHOLE && !here[0]) continue;
    // scores of tokens g (x[.][0, 1]) and g + 8 ([2, 3])
    float x[NR][4];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) x[r][k] = 0.f;
#pragma unroll
    for (int p = 0; p < Sh::kPerKey; ++p) {
      const uint4 u = from_shared16(stage + (WHOLE ? box_at(g, q4 * 16 + p * 64) : p * 512 + lane * 16)),
                  w = from_shared16(stage + (WHOLE ? box_at(g + 8, q4 * 16 + p * 64) : (Sh::kPerKey + p) * 512 + lane * 16));
      const unsigned int uu[4] = {u.x, u.y, u.z, u.w}, ww[4] = {w.x, w.y, w.z, w.w};
      if constexpr (CODED) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          unsigned int y[4];
          e4m3_split(uu[t], y[0], y[2]);
          e4m3_split(ww[t], y[1], y[3]);
#pragma unroll
          for (int r = 0; r < NR; ++r) mma16<M>(x[r], y, q[r][4 * p + t][0], q[r][4 * p + t][1]);
        }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const unsigned int y[4] = {uu[2 * t], ww[2 * t], uu[2 * t + 1], ww[2 * t + 1]};
#pragma unroll
          for (int r = 0; r < NR; ++r) mma16<M>(x[r], y, q[r][2 * p + t][0], q[r][2 * p + t][1]);
        }
      }
    }
    const bool beyond = j0 + 15 >= end;
    const bool some_hidden = !WHOLE || j0 + 15 > all_see || (a.window && j0 < all_from && j0 + 15 >= a.sinks);
    bool grows = false;
    float top[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (a.cap > 0.f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[r][k] *= CODED ? unit[r][k & 1] * down[k >> 1] : unit[r][k & 1];
        tanh_chunk(x[r], 1.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[r][k] = CODED ? fmaf(x[r][k], to_log2, raise[k >> 1]) : x[r][k] * to_log2;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[r][k] = CODED ? fmaf(x[r][k], unit[r][k & 1] * down[k >> 1], raise[k >> 1]) : x[r][k] * unit[r][k & 1];
      }
      if (a.slopes)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = min(8 * r + 2 * (int)q4 + (k & 1), rows - 1);
          x[r][k] = fmaf(-a.slopes[head_of(i)] * kCacheLog2e, (float)(pos[r][k & 1] - j0 - (int)g - 8 * (k >> 1)), x[r][k]);
        }
      if (some_hidden)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = j0 + (int)g + 8 * (k >> 1), at = pos[r][k & 1];
          const bool on = j <= at && j < end && (j >= cache_first(a, at) || j < a.sinks) && here[WHOLE ? 0 : k >> 1];
          x[r][k] = on ? x[r][k] : -INFINITY;
        }
      top[r][0] = fmaxf(x[r][0], x[r][2]);
      top[r][1] = fmaxf(x[r][1], x[r][3]);
      grows = grows || top[r][0] > limit[r][0] || top[r][1] > limit[r][1];
    }
    // the maximum in use moves when a row has outgrown it by 2^8 (or has had none): hardly ever after the first steps
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top[r][k] = fmaxf(top[r][k], __shfl_xor_sync(0xffffffffu, top[r][k], d));
          const float next = fmaxf(m[r][k], top[r][k]);
          const float by = m[r][k] == next ? 1.f : m[r][k] == -INFINITY ? 0.f : ex2(m[r][k] - next);
          m[r][k] = next;
          limit[r][k] = next + 8.f;
          off[r][k] = next == -INFINITY ? 0.f : next - kUp;
          l[r][k] *= by;
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {
            o[r][i][k] *= by;
            o[r][i][2 + k] *= by;
          }
        }
    }
    // weights as the B operand: tokens 0-7 and 8-15 of a row
    unsigned int wt[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float p0 = ex2(x[r][0] - off[r][0]), p1 = ex2(x[r][1] - off[r][1]), p2 = ex2(x[r][2] - off[r][0]), p3 = ex2(x[r][3] - off[r][1]);
      if constexpr (CODED) {
        l[r][0] = fmaf(p0, back[0], fmaf(p2, back[1], l[r][0]));
        l[r][1] = fmaf(p1, back[0], fmaf(p3, back[1], l[r][1]));
      } else {
        l[r][0] += p0 + p2;
        l[r][1] += p1 + p3;
      }
      wt[r][0] = transpose8(pack2(p0, p1, M()));
      wt[r][1] = transpose8(pack2(p2, p3, M()));
    }
    // values: elements g * DP / 8 + 2 i and the next one are rows g and g + 8 of tile i
#pragma unroll
    for (int piece = 0; piece < Sh::kPerValue; ++piece) {
      constexpr int kWords = Sh::kValueWidth / 4;
      unsigned int y[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned int token = q4 * 2 + (k & 1) + 8 * (k >> 1);
        const unsigned int from = stage + Sh::kKeys + (WHOLE ? box_at(token, g * Sh::kValueBytes + piece * 16) : (k * Sh::kPerValue + piece) * 32 * Sh::kValueWidth + lane * Sh::kValueWidth);
        if constexpr (kWords == 4) {
          const uint4 v = from_shared16(from);
          y[k][0] = v.x; y[k][1] = v.y; y[k][2] = v.z; y[k][3] = v.w;
        } else {
          const uint2 v = from_shared8(from);
          y[k][0] = v.x; y[k][1] = v.y;
        }
        // (a box has its page's slots behind the last token too)
        if (WHOLE && beyond)
#pragma unroll
          for (int i = 0; i < kWords; ++i) y[k][i] = j0 + (int)token < end ? y[k][i] : 0u;
      }
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (CODED) {
          // tokens 2 q4, 2 q4 + 1 of elements 4 i, 4 i + 1, then of the next two; the same for the tokens 8 further
          unsigned int z[2][4];
          e4m3_split(__byte_perm(y[0][i], y[1][i], 0x5140), z[0][0], z[0][1]);
          e4m3_split(__byte_perm(y[2][i], y[3][i], 0x5140), z[0][2], z[0][3]);
          e4m3_split(__byte_perm(y[0][i], y[1][i], 0x7362), z[1][0], z[1][1]);
          e4m3_split(__byte_perm(y[2][i], y[3][i], 0x7362), z[1][2], z[1][3]);
          const int at = (piece * kWords + i) * 2;
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            mma16<M>(o[r][at], z[0], wt[r][0], wt[r][1]);
            mma16<M>(o[r][at + 1], z[1], wt[r][0], wt[r][1]);
          }
        } else {
          const unsigned int z[4] = {__byte_perm(y[0][i], y[1][i], 0x5410), __byte_perm(y[0][i], y[1][i], 0x7632), __byte_perm(y[2][i], y[3][i], 0x5410),
                                     __byte_perm(y[2][i], y[3][i], 0x7632)};
#pragma unroll
          for (int r = 0; r < NR; ++r) mma16<M>(o[r][piece * kWords + i], z, wt[r][0], wt[r][1]);
        }
      }
    }
  }
  if constexpr (WHOLE) {
    // (after a wait that gave up, what is under way lands before shared memory has another use)
    if (!live)
      for (; taken != filled; ++taken)
        for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bars + 8 * (taken % Sh::kStages), taken / Sh::kStages & 1u); ++tries) {}
  } else {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[r][k] += __shfl_xor_sync(0xffffffffu, l[r][k], d);
  __syncthreads();                    // the rings become the place where the warps meet
  float* join = (float*)gen;
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float* row = join + (warp * R + 8 * r + 2 * q4 + k) * W;
#pragma unroll
      for (int i = 0; i < DP / 16; i += 2) *(float4*)(row + g * (DP / 8) + 2 * i) = make_float4(o[r][i][k], o[r][i][2 + k], o[r][i + 1][k], o[r][i + 1][2 + k]);
      if (g == 0) {
        row[DP] = m[r][k];
        row[DP + 1] = l[r][k];
      }
    }
  __syncthreads();
  const int lane_e = 4 * (int)lane;
  __shared__ float weights[kCacheFewWarps][kFewMost];
  // a warp takes every fourth row
  bool last = true;
  if (plan.parts > 1) {
    float* parts = f.parts + cache_part_at(plan.first_block, plan.part) * R * W;
    for (int i = (int)warp; i < rows; i += kCacheFewWarps) {
      float most, sum;
      few_weigh<DP>(join + i * W, kCacheFewWarps, R * W, weights[warp], most, sum);
      if (lane_e < DP) *(float4*)(parts + i * W + lane_e) = few_gather(join + i * W, kCacheFewWarps, R * W, weights[warp], lane_e, 0, 1);
      if (lane == 0) {
        parts[i * W + DP] = most;
        parts[i * W + DP + 1] = sum;
      }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      last_block = plan.meets && atomicAdd(&f.tickets[plan.first_block], 1u) == plan.parts - 1u;
      if (last_block) f.tickets[plan.first_block] = 0u;       // for the next run
    }
    __syncthreads();
    last = last_block != 0u;
    __threadfence();
  }
  if (last) {
    // (parts lie two a block apart, but for the first, which is the second of its block)
    const bool joined = plan.parts > 1;
    const float* all = joined ? f.parts + cache_part_at(plan.first_block, 0) * R * W : join;
    const int n_parts = joined ? (int)plan.parts : kCacheFewWarps;
    for (int i = (int)warp; i < rows; i += kCacheFewWarps) {
      float most, sum;
      bool fine = true;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (joined) {
        v = cache_join<DP, R>([](float x) { return ex2(x); }, all + i * W, n_parts, weights[warp], lane_e < DP, lane_e, most, sum);
      } else {
        few_weigh<DP>(all + i * W, n_parts, R * W, weights[warp], most, sum);
        if (lane_e < DP) v = few_gather(all + i * W, n_parts, R * W, weights[warp], lane_e, 0, 1);
      }
      if (lane_e < DP) fine = cache_finish<T>(a, s.first + query_of(i), head_of(i), lane_e, v, most, sum, kUp);
      if (attn_again(fine)) cache_attention_row<T, CODED>(a, b, head_of(i), s.first + query_of(i), s.pos0 + query_of(i), lane);
    }
  }
  if constexpr (WHOLE) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();                    // (the rings, and what lies where they were, are written again)
  }
}

}  // namespace b200
#endif
