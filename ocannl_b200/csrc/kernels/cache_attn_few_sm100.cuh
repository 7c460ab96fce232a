// Attention of new tokens over a paged cache, 16-bit heads, 8 or 16 rows at a time: the next tokens of sequences, and ragged batches of them.
//
// The keys and values are read once and bound it.  The query heads that share a key head, and their tokens, are the columns of mma.m16n8k16 (tcgen05
// has no tile of 8 or 16 rows): scores' = K q', 16 tokens at a time, and out' = V' weights', so that 8 rows, as many as heads usually share a key, waste
// nothing, and take half the registers and products of a tile of 16.  A product does not care in which order its elements are added, so the order is
// chosen for the loads: of the 16 elements of a step each of the four lanes that share a token has four neighbours, and the rows of the second product
// are dealt out as neighbours to a lane too, so that every operand is read as whole 16-byte pieces by the lane that multiplies it.  A lane's cp.async
// ring is its own, with no barrier between lanes; codes of 8 bits become halves in registers, two to an instruction; a transposed pair of values is one byte
// permutation, and the weights turn from scores' to operand's layout by a transpose of 8 x 8 between lanes.  Codes are multiplied as they are: a
// page's scale of the keys goes onto its scores, the logarithm of its scale of the values onto the exponents of its weights, which the row's sum takes off
// again: out = sum w code / sum (w / scale), so that weights stay in the range of a half whatever the scales.  (bfloat16 queries beside codes become
// halves too, each row multiplied by the power of two that brings its largest to 2^14.)
//
// The tokens that a tile sees (with a window: the sinks' and the window's, as one range) are cut into chunks, so that sequences of all lengths fill the
// machine evenly: every block sums the lengths of all sequences, from which all find the same size of a chunk and each its own.  The block of a tile that
// comes last joins the chunks in their order: the same bits whoever comes last.
#ifndef B200_CACHE_ATTN_FEW_SM100_CUH
#define B200_CACHE_ATTN_FEW_SM100_CUH
#include "attn_few_sm100.cuh"
#include "cache_attn_terms.cuh"

namespace b200 {

struct CacheFewArgs {
  float* parts;            // [unit][rows of a tile][DP + 4]: output (not divided), maximum, sum
  unsigned int* tickets;   // [unit], zero between runs
  long long target;        // chunks that fill the machine
  int least, most;         // tokens of a chunk, about, at least; chunks of a tile at most
  int single;              // one chunk a tile, whatever the lengths
  Divisor by_group, by_key_heads, by_units;     // by_units: without starts, units of a sequence (single)
};

constexpr int kCacheFewWarps = 4, kCacheFewThreads = 32 * kCacheFewWarps;
constexpr int kCacheChunk = 65536;     // tokens of a chunk at most, a quarter of them a warp's: its accumulators' cut-off sums lose 2^-13 (see kSumKeys)

template <int DP, bool CODED, int NR>
struct CacheFewShape {
  static constexpr int kRows = 8 * NR;
  static constexpr int kPerKey = CODED ? DP / 64 : DP / 32;            // 16-byte pieces of a key that a lane has
  static constexpr int kValueBytes = CODED ? DP / 8 : DP / 4;          // bytes of a value that a lane has
  static constexpr int kValueWidth = kValueBytes < 16 ? kValueBytes : 16, kPerValue = kValueBytes / kValueWidth;
  static constexpr int kKeys = 2 * kPerKey * 512, kValues = 4 * kPerValue * 32 * kValueWidth;
  static constexpr int kStage = kKeys + kValues;                       // bytes of a warp
  static constexpr int kStages = CODED ? (DP == 64 ? 4 : 3) : DP == 64 ? 3 : 2;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kWidth = DP + 4;
  static constexpr int kJoin = kCacheFewWarps * kRows * kWidth * 4;
  static constexpr int smem() { return kCacheFewWarps * kRing > kJoin ? kCacheFewWarps * kRing : kJoin; }
  static constexpr int kBlocks = NR == 1 ? 4 : 3;                      // of an SM
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
// What a sequence's tiles look at: its rows of a key head, in tiles, and no fewer tokens than any of them sees, as they are walked
struct CacheWalk {
  unsigned int tiles;
  int tokens;
};
template <int ROWS>
__device__ __forceinline__ CacheWalk cache_walk(const CacheAttnArgs& a, const CacheSeq& s) {
  CacheWalk w;
  w.tiles = ((unsigned int)s.count * (unsigned int)a.group + (ROWS - 1)) / ROWS;
  long long n = (long long)cache_last(a, s.pos0 + s.count - 1) + 1;
  if (a.window) n = min(n, (long long)a.window + ((a.sinks + 15ll) & ~15ll) + ROWS / a.group + 17);
  w.tokens = (int)max(n, 1ll);
  return w;
}
// chunks of about `size` tokens: the nearest number
__device__ __forceinline__ unsigned int cache_chunks(const CacheFewArgs& f, int tokens, int size) {
  const unsigned int n = ((unsigned int)tokens + (unsigned int)(size >> 1)) / (unsigned int)size;
  return min(max(n, 1u), (unsigned int)f.most);
}

// A block's chunk: of a sequence, a tile of its rows of a key head, and how the tile's tokens are walked.
struct CachePlan {
  int b, hk, first_row, rows;          // rows of the tile that there are
  CacheSeq s;
  unsigned int chunks, first_unit;     // of the tile; the number of its first block
  int least_pos, most_pos, end;        // positions of its rows; tokens that some row sees lie before `end`
  int sink_end, shift;                 // the walk: tokens 0 .. sink_end - 1, then those from sink_end + shift on
  int begin, stop;                     // of the walk, this chunk's
  __device__ __forceinline__ int token_of(int v) const { return v < sink_end ? v : v + shift; }
};
template <int NT, int ROWS>
__device__ __forceinline__ bool cache_plan(const CacheAttnArgs& a, const CacheFewArgs& f, CachePlan& p) {
  const CacheArgs& c = a.c;
  __shared__ unsigned long long works[NT / 32];
  unsigned int nth;
  p.chunks = 1;
  if (f.single && !c.starts) {
    p.b = (int)f.by_units.of(blockIdx.x);
    nth = blockIdx.x - (unsigned int)p.b * f.by_units.d;
    if (p.b >= c.batch) return false;
  } else {
    int size = 0x7fffffff;
    if (!f.single) {
      unsigned long long work = 0;
      for (int i = (int)threadIdx.x; i < c.batch; i += NT) {
        const CacheSeq s = cache_seq(c, i);
        if (s.count) {
          const CacheWalk w = cache_walk<ROWS>(a, s);
          work += (unsigned long long)w.tiles * (unsigned int)w.tokens;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
      if ((threadIdx.x & 31u) == 0) works[threadIdx.x >> 5] = work;
      __syncthreads();
      work = 0;
#pragma unroll
      for (int i = 0; i < NT / 32; ++i) work += works[i];
      size = (int)min(max((long long)(work * (unsigned int)c.HK / (unsigned long long)f.target) + 1, (long long)f.least), (long long)kCacheChunk);
    }
    const bool found = find_unit<NT>(
        c.batch, blockIdx.x,
        [&](int i) {
          const CacheSeq s = cache_seq(c, i);
          if (!s.count) return 0u;
          const CacheWalk w = cache_walk<ROWS>(a, s);
          return w.tiles * (unsigned int)c.HK * (f.single ? 1u : cache_chunks(f, w.tokens, size));
        },
        p.b, nth);
    if (!found) return false;
    if (!f.single) p.chunks = cache_chunks(f, cache_walk<ROWS>(a, cache_seq(c, p.b)).tokens, size);
  }
  p.s = cache_seq(c, p.b);
  const unsigned int pair = nth / p.chunks, chunk = nth - pair * p.chunks;
  const unsigned int tile = f.by_key_heads.of(pair);
  p.first_unit = blockIdx.x - chunk;
  p.hk = (int)(pair - tile * (unsigned int)c.HK);
  p.first_row = (int)tile * ROWS;
  p.rows = min(ROWS, p.s.count * a.group - p.first_row);
  p.least_pos = p.s.pos0 + (int)f.by_group.of((unsigned int)p.first_row);
  p.most_pos = p.s.pos0 + (int)f.by_group.of((unsigned int)(p.first_row + p.rows - 1));
  p.end = cache_last(a, p.most_pos) + 1;
  p.sink_end = p.shift = 0;
  if (a.window) {
    p.sink_end = (int)min(((long long)min(a.sinks, max(p.end, 0)) + 15) & ~15ll, 0x7ffffff0ll);
    p.shift = max((cache_first(a, p.least_pos) & ~15) - p.sink_end, 0);
  }
  const int n_tokens = p.shift ? max(p.end - p.shift, p.sink_end) : max(p.end, 0);       // (the window may lie behind the last page)
  const int per = (int)((((long long)n_tokens + p.chunks - 1) / p.chunks + 63) & ~63ll);
  p.begin = (int)min((long long)chunk * per, (long long)n_tokens);
  p.stop = (int)min((long long)p.begin + per, (long long)n_tokens);
  return true;
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
__global__ void __launch_bounds__(kCacheFewThreads, (CacheFewShape<DP, CODED, NR>::kBlocks)) cache_attention_few(const __grid_constant__ CacheAttnArgs a,
                                                                                                               const __grid_constant__ CacheFewArgs f) {
  typedef CacheFewShape<DP, CODED, NR> Sh;
  typedef typename std::conditional<CODED, __half, T>::type M;          // what is multiplied
  constexpr int KS = DP / 16, W = Sh::kWidth, R = Sh::kRows;
  constexpr float kUp = kLift<M>;
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ unsigned int last_block;
  const CacheArgs& c = a.c;
  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, q4 = lane & 3u;
  grid_begin();

  CachePlan plan;
  if (!cache_plan<kCacheFewThreads, R>(a, f, plan)) return;
  const CacheSeq& s = plan.s;
  const int b = plan.b, hk = plan.hk, first_row = plan.first_row, rows = plan.rows, end = plan.end, v_begin = plan.begin, v_end = plan.stop;
  const unsigned int chunks = plan.chunks, first_unit = plan.first_unit;
  auto query_of = [&](int i) { return (int)f.by_group.of((unsigned int)(first_row + i)); };
  auto head_of = [&](int i) { return hk * a.group + first_row + i - query_of(i) * a.group; };
  // (this lane's columns are rows 8 r + 2 q4 and the next one)
  const int all_see = cache_last(a, plan.least_pos), all_from = cache_first(a, plan.most_pos);

  // ---- the ring: steps of 16 tokens, every fourth of them this warp's
  const unsigned int ring = b200_smem_addr(dyn) + warp * Sh::kRing;
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
  const int key_at = (int)g * line + (int)q4 * 16, value_at = (int)q4 * 2 * line + (int)g * Sh::kValueBytes;
  int ahead = 0 < mine ? page_of(token_of(0)) : -1;  // the page of the step that is fetched next
  unsigned int to = 0;                               // the slot that is filled next
  auto fetch = [&](int n) {
    if (n < mine) {
      const int j0 = token_of(n);
      const unsigned int at_k = ring + to * Sh::kStage + lane * 16, at_v = ring + to * Sh::kStage + Sh::kKeys + lane * Sh::kValueWidth;
      const int page = ahead;
      if (WHOLE) {
        if (n + 1 < mine) ahead = page_of(token_of(n + 1));
        const unsigned int slot0 = (unsigned int)j0 - c.by_page.of((unsigned int)j0) * c.page;
        const long long from = page >= 0 ? (cache_at(c, page, hk) + (long long)slot0 * c.D) * kSize : 0;
        const int left = page >= 0 ? end - j0 : 0;   // tokens of the step that are there
        const unsigned char *const k0 = keys + from + key_at, *const v0 = values + from + value_at;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const bool on = (int)g + 8 * k < left;
#pragma unroll
          for (int p = 0; p < Sh::kPerKey; ++p) {
            const int bytes = on ? key_bytes(p) : 0;
            copy_in<16>(at_k + (k * Sh::kPerKey + p) * 512, bytes ? k0 + k * 8 * line + p * 64 : keys, bytes);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool on = (int)q4 * 2 + (k & 1) + 8 * (k >> 1) < left;
#pragma unroll
          for (int p = 0; p < Sh::kPerValue; ++p) {
            const int bytes = on ? value_bytes(p) : 0;
            copy_in<Sh::kValueWidth>(at_v + (k * Sh::kPerValue + p) * 32 * Sh::kValueWidth, bytes ? v0 + ((k & 1) + 8 * (k >> 1)) * line + p * 16 : values, bytes);
          }
        }
      } else {
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
      to = to + 1 == Sh::kStages ? 0 : to + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < Sh::kStages - 1; ++i) fetch(i);

  // ---- the queries as the B operand, in the order of the keys' pieces: row 8 r + g
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
  float o[NR][DP / 16][4], m[NR][2], l[NR][2];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[r][i][k] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) m[r][k] = -INFINITY, l[r][k] = 0.f;
  }

  // the page of the step at hand, or (not WHOLE) those of this lane's tokens g and g + 8, and their scales: a step ahead
  int there[2] = {-1, -1};
  float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
  auto look = [&](int n) {
    if (n >= mine) return;
    const int j0 = token_of(n);
#pragma unroll
    for (int k = 0; k < (WHOLE ? 1 : 2); ++k) {
      const int j = WHOLE ? j0 : j0 + (int)g + 8 * k;
      there[k] = j < end ? page_of(j) : -1;
      if (CODED && there[k] >= 0) {
        ks[k] = __ldg(c.k_scale + (long long)there[k] * c.HK + hk);
        vs[k] = __ldg(c.v_scale + (long long)there[k] * c.HK + hk);
      }
    }
  };
  look(0);
  unsigned int slot = 0;
  for (int n = 0; n < mine; ++n) {
    const int j0 = token_of(n);
    const int here[2] = {there[0], WHOLE ? there[0] : there[1]};
    // scale of the keys; of the values its inverse and its logarithm
    float down[2] = {1.f, 1.f}, back[2] = {1.f, 1.f}, raise[2] = {0.f, 0.f};
    if constexpr (CODED) {
#pragma unroll
      for (int k = 0; k < (WHOLE ? 1 : 2); ++k) {
        down[k] = cache_scale(ks[k]);
        const float v = cache_scale(vs[k]);
        back[k] = rcp(v);
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(raise[k]) : "f"(v));
      }
      if (WHOLE) down[1] = down[0], back[1] = back[0], raise[1] = raise[0];
    }
    look(n + 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(Sh::kStages - 2) : "memory");
    fetch(n + Sh::kStages - 1);       // into the slot of the step before, which this lane alone reads
    const unsigned int at_k = ring + slot * Sh::kStage + lane * 16, at_v = ring + slot * Sh::kStage + Sh::kKeys + lane * Sh::kValueWidth;
    slot = slot + 1 == Sh::kStages ? 0 : slot + 1;
    if (WHOLE && here[0] < 0) continue;
    // scores of tokens g (x[.][.][0, 1]) and g + 8 ([2, 3]); two sums, so that one product need not wait for the other
    float x[NR][4], x2[NR][4];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) x[r][k] = x2[r][k] = 0.f;
#pragma unroll
    for (int p = 0; p < Sh::kPerKey; ++p) {
      const uint4 u = from_shared16(at_k + p * 512), w = from_shared16(at_k + (Sh::kPerKey + p) * 512);
      const unsigned int uu[4] = {u.x, u.y, u.z, u.w}, ww[4] = {w.x, w.y, w.z, w.w};
      if constexpr (CODED) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          unsigned int y[4];
          e4m3_split(uu[t], y[0], y[2]);
          e4m3_split(ww[t], y[1], y[3]);
#pragma unroll
          for (int r = 0; r < NR; ++r) mma16<M>(t & 1 ? x2[r] : x[r], y, q[r][4 * p + t][0], q[r][4 * p + t][1]);
        }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const unsigned int y[4] = {uu[2 * t], ww[2 * t], uu[2 * t + 1], ww[2 * t + 1]};
#pragma unroll
          for (int r = 0; r < NR; ++r) mma16<M>(t & 1 ? x2[r] : x[r], y, q[r][2 * p + t][0], q[r][2 * p + t][1]);
        }
      }
    }
    const bool some_hidden = !WHOLE || j0 + 15 > all_see || (a.window && j0 < all_from && j0 + 15 >= a.sinks);
    bool grows = false;
    float top[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[r][k] = (x[r][k] + x2[r][k]) * (CODED ? unit[r][k & 1] * down[k >> 1] : unit[r][k & 1]);
      if (a.cap > 0.f) {
        tanh_chunk(x[r], 1.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[r][k] *= to_log2;
      }
      if (a.slopes)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = min(8 * r + 2 * (int)q4 + (k & 1), rows - 1);
          x[r][k] = fmaf(-a.slopes[head_of(i)] * kCacheLog2e, (float)(pos[r][k & 1] - j0 - (int)g - 8 * (k >> 1)), x[r][k]);
        }
      if constexpr (CODED)
#pragma unroll
        for (int k = 0; k < 4; ++k) x[r][k] += raise[k >> 1];
      if (some_hidden)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = j0 + (int)g + 8 * (k >> 1), at = pos[r][k & 1];
          const bool on = j <= at && j < end && (j >= cache_first(a, at) || j < a.sinks) && here[k >> 1] >= 0;
          x[r][k] = on ? x[r][k] : -INFINITY;
        }
      top[r][0] = fmaxf(x[r][0], x[r][2]);
      top[r][1] = fmaxf(x[r][1], x[r][3]);
      grows = grows || top[r][0] > m[r][0] + 8.f || top[r][1] > m[r][1] + 8.f;
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
      const float off0 = m[r][0] == -INFINITY ? 0.f : m[r][0] - kUp, off1 = m[r][1] == -INFINITY ? 0.f : m[r][1] - kUp;
      const float p0 = ex2(x[r][0] - off0), p1 = ex2(x[r][1] - off1), p2 = ex2(x[r][2] - off0), p3 = ex2(x[r][3] - off1);
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
        const unsigned int from = at_v + (k * Sh::kPerValue + piece) * 32 * Sh::kValueWidth;
        if constexpr (kWords == 4) {
          const uint4 v = from_shared16(from);
          y[k][0] = v.x; y[k][1] = v.y; y[k][2] = v.z; y[k][3] = v.w;
        } else {
          const uint2 v = from_shared8(from);
          y[k][0] = v.x; y[k][1] = v.y;
        }
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
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[r][k] += __shfl_xor_sync(0xffffffffu, l[r][k], d);
  __syncthreads();                    // the rings become the place where the warps meet
  float* join = (float*)dyn;
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
  float* parts = f.parts + (long long)blockIdx.x * R * W;
  // a warp takes every fourth row
  if (chunks > 1) {
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
    if (threadIdx.x == 0) last_block = atomicAdd(&f.tickets[first_unit], 1u) == chunks - 1u;
    __syncthreads();
    if (!last_block) return;
    if (threadIdx.x == 0) f.tickets[first_unit] = 0u;       // for the next run
    __threadfence();
  }
  const float* all = chunks > 1 ? f.parts + (long long)first_unit * R * W : join;
  const int n_parts = chunks > 1 ? (int)chunks : kCacheFewWarps;
  for (int i = (int)warp; i < rows; i += kCacheFewWarps) {
    float most, sum;
    few_weigh<DP>(all + i * W, n_parts, R * W, weights[warp], most, sum);
    bool fine = true;
    if (lane_e < DP) fine = cache_finish<T>(a, s.first + query_of(i), head_of(i), lane_e, few_gather(all + i * W, n_parts, R * W, weights[warp], lane_e, 0, 1), most, sum, kUp);
    if (attn_again(fine)) cache_attention_row<T, CODED>(a, b, head_of(i), s.first + query_of(i), s.pos0 + query_of(i), lane);
  }
}

}  // namespace b200
#endif
