// Attention of new tokens over a paged cache, 16-bit heads, the rows sixteen at a time: the next tokens of sequences, and ragged batches of them.
//
// The keys and values are read once and bound it.  The query heads that share a key head, and their tokens, are the 16 rows of a tile of mma.m16n8k16
// (tcgen05 has no tile of 16 rows).  A product does not care in which order its elements are added, so the order is chosen for the loads: with the
// 16 elements of a step dealt out as four neighbours to each of the four lanes that share a key, and the columns of the second product dealt out as
// neighbours to a lane too, every operand is read as whole 16-byte pieces of a row, by the lane that multiplies it.  A lane's cp.async ring is its
// own (no barrier between the lanes), codes of 8 bits become halves in registers, two to an instruction, and a transposed value pair is one byte
// permutation.  Codes are multiplied as they are: a page's scale of the keys goes onto its scores, the logarithm of its scale of the values onto the
// exponents of its weights, which the row's sum takes off again: out = sum w code / sum (w / scale), so that weights stay in the range of
// a half whatever the scales.  (bfloat16 queries beside codes become halves too, each row multiplied by the power of two that brings its largest to 2^14.)
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
  float* parts;            // [unit][16][DP + 4]: output (not divided), maximum, sum
  unsigned int* tickets;   // [unit], zero between runs
  long long target;        // chunks that fill the machine
  int least, most;         // tokens of a chunk at least; chunks of a tile at most
  Divisor by_group, by_key_heads;
};

constexpr int kCacheFewWarps = 4, kCacheFewThreads = 32 * kCacheFewWarps;
constexpr int kCacheChunk = 65536;     // tokens of a chunk at most, a quarter of them a warp's: its accumulators' cut-off sums lose 2^-13 (see kSumKeys)

template <int DP, bool CODED>
struct CacheFewShape {
  static constexpr int kPerKey = CODED ? DP / 64 : DP / 32;            // 16-byte pieces of a key that a lane has
  static constexpr int kValueBytes = CODED ? DP / 8 : DP / 4;          // bytes of a value that a lane has
  static constexpr int kValueWidth = kValueBytes < 16 ? kValueBytes : 16, kPerValue = kValueBytes / kValueWidth;
  static constexpr int kKeys = 2 * kPerKey * 512, kValues = 4 * kPerValue * 32 * kValueWidth, kScales = CODED ? 128 : 0;
  static constexpr int kStage = kKeys + kValues + kScales;             // bytes of a warp
  static constexpr int kStages = CODED ? 4 : DP == 64 ? 4 : 3;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kWidth = DP + 4;
  static constexpr int kJoin = kCacheFewWarps * 16 * kWidth * 4;
  static constexpr int smem() { return kCacheFewWarps * kRing > kJoin ? kCacheFewWarps * kRing : kJoin; }
};

template <int BYTES>
__device__ __forceinline__ void copy_in(unsigned int dst, const void* src, bool on) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(on ? BYTES : 0) : "memory");
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

// What a sequence's tiles look at: its rows of a key head, in tiles of 16, and no fewer tokens than any of them sees, as they are walked
struct CacheWalk {
  unsigned int tiles;
  long long tokens;
};
__device__ __forceinline__ CacheWalk cache_walk(const CacheAttnArgs& a, const CacheSeq& s) {
  CacheWalk w;
  w.tiles = (unsigned int)(((long long)s.count * a.group + 15) / 16);
  w.tokens = (long long)cache_last(a, s.pos0 + s.count - 1) + 1;
  if (a.window) w.tokens = min(w.tokens, (long long)a.window + ((a.sinks + 15ll) & ~15ll) + 16 / a.group + 17);
  w.tokens = max(w.tokens, 1ll);
  return w;
}
__device__ __forceinline__ unsigned int cache_chunks(const CacheFewArgs& f, long long tokens, long long size) {
  return (unsigned int)min((tokens + size - 1) / size, (long long)f.most);
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

template <class T, int DP, bool CODED>
__global__ void __launch_bounds__(kCacheFewThreads, 3) cache_attention_few(const __grid_constant__ CacheAttnArgs a, const __grid_constant__ CacheFewArgs f) {
  typedef CacheFewShape<DP, CODED> Sh;
  typedef typename std::conditional<CODED, __half, T>::type M;          // what is multiplied
  constexpr int KS = DP / 16, W = Sh::kWidth;
  constexpr float kUp = kLift<M>;
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ unsigned long long works[kCacheFewWarps];
  __shared__ unsigned int last_block;
  const CacheArgs& c = a.c;
  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, q4 = lane & 3u;
  grid_begin();

  // ---- this block's chunk
  unsigned long long work = 0;
  for (int i = (int)threadIdx.x; i < c.batch; i += kCacheFewThreads) {
    const CacheSeq s = cache_seq(c, i);
    if (s.count) {
      const CacheWalk w = cache_walk(a, s);
      work += (unsigned long long)w.tiles * (unsigned long long)w.tokens;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
  if (lane == 0) works[warp] = work;
  __syncthreads();
  work = 0;
#pragma unroll
  for (int i = 0; i < kCacheFewWarps; ++i) work += works[i];
  const long long size = min(max((long long)(work * (unsigned int)c.HK / (unsigned long long)f.target) + 1, (long long)f.least), (long long)kCacheChunk);
  int b;
  unsigned int nth;
  const bool found = find_unit<kCacheFewThreads>(
      c.batch, blockIdx.x,
      [&](int i) {
        const CacheSeq s = cache_seq(c, i);
        if (!s.count) return 0u;
        const CacheWalk w = cache_walk(a, s);
        return w.tiles * (unsigned int)c.HK * cache_chunks(f, w.tokens, size);
      },
      b, nth);
  if (!found) return;
  const CacheSeq s = cache_seq(c, b);
  const CacheWalk walk = cache_walk(a, s);
  const unsigned int chunks = cache_chunks(f, walk.tokens, size), pair = nth / chunks, chunk = nth - pair * chunks;
  const unsigned int tile = f.by_key_heads.of(pair), first_unit = blockIdx.x - chunk;
  const int hk = (int)(pair - tile * (unsigned int)c.HK);
  const int shared_rows = s.count * a.group, first_row = (int)tile * 16, rows = min(16, shared_rows - first_row);
  auto query_of = [&](int i) { return (int)f.by_group.of((unsigned int)(first_row + i)); };
  auto head_of = [&](int i) { return hk * a.group + first_row + i - query_of(i) * a.group; };

  // ---- what its rows see; this lane's two accumulator rows are g and g + 8
  int pos[2], last[2], first[2];
  float slope2[2] = {0.f, 0.f};
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int i = (int)g + 8 * w;
    pos[w] = -1;
    last[w] = -1;
    first[w] = 0;
    if (i < rows) {
      pos[w] = s.pos0 + query_of(i);
      last[w] = cache_last(a, pos[w]);
      first[w] = cache_first(a, pos[w]);
      if (a.slopes) slope2[w] = a.slopes[head_of(i)] * kCacheLog2e;
    }
  }
  const int least_pos = s.pos0 + query_of(0), most_pos = s.pos0 + query_of(rows - 1);
  const int end = cache_last(a, most_pos) + 1;                         // tokens that some row sees lie before it
  const int all_see = cache_last(a, least_pos), all_from = cache_first(a, most_pos);
  // the walk: tokens 0 .. sink_end - 1, then those from sink_end + shift on
  int sink_end = 0, shift = 0;
  if (a.window) {
    sink_end = (int)min(((long long)min(a.sinks, max(end, 0)) + 15) & ~15ll, 0x7ffffff0ll);
    shift = max((cache_first(a, least_pos) & ~15) - sink_end, 0);
  }
  const int n_tokens = shift ? max(end - shift, sink_end) : max(end, 0);       // (the window may lie behind the last page)
  const int per = (int)((((long long)n_tokens + chunks - 1) / chunks + 63) & ~63ll);
  const int v_begin = (int)min((long long)chunk * per, (long long)n_tokens), v_end = (int)min((long long)v_begin + per, (long long)n_tokens);

  // ---- the queries as the A operand, in the order of the keys' pieces
  unsigned int q[KS][4];
  float unit[2] = {1.f, 1.f};                        // what a row's products have to be multiplied by
  {
    constexpr int kRun = CODED ? 16 : 8;             // neighbouring elements of a lane
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int i = (int)g + 8 * w;
      const bool on = i < rows;
      const unsigned short* from = (const unsigned short*)a.q + (on ? ((long long)(s.first + query_of(i)) * a.H + head_of(i)) * c.D : 0);
      unsigned int most = 0;
#pragma unroll
      for (int p = 0; p < DP / (4 * kRun); ++p)
#pragma unroll
        for (int t = 0; t < kRun / 8; ++t) {
          const int e = p * 4 * kRun + (int)q4 * kRun + t * 8, ks = p * (kRun / 4) + 2 * t;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (on && e < c.D) v = *(const uint4*)(from + e);
          q[ks][w] = v.x;
          q[ks][2 + w] = v.y;
          q[ks + 1][w] = v.z;
          q[ks + 1][2 + w] = v.w;
        }
      if constexpr (CODED && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const unsigned int x = q[ks][2 * k + w];
            most = max(most, max(x & 0x7fffu, (x >> 16) & 0x7fffu));
          }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the exponent of the largest, which goes to 14 (none for zeros, and for what is infinite or undefined)
        const int e = (int)(most >> 7);
        const int up = e == 0 || e == 255 ? 0 : min(max(127 + 14 - e, -126), 126);
        const float by = power_of_two(up);
        unit[w] = power_of_two(-up);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = unpack2(q[ks][2 * k + w], __nv_bfloat16());
            q[ks][2 * k + w] = pack2(x.x * by, x.y * by, __half());
          }
      }
    }
  }
  const float to_log2 = a.cap > 0.f ? a.cap * kCacheLog2e : 1.f;
#pragma unroll
  for (int w = 0; w < 2; ++w) unit[w] *= a.cap > 0.f ? a.over : a.scale * kCacheLog2e;

  float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[i][k] = 0.f;

  // ---- the ring
  const unsigned int ring = b200_smem_addr(dyn) + warp * Sh::kRing;
  const int steps = v_end > v_begin ? (v_end - v_begin + 15) / 16 : 0;
  const int mine = steps > (int)warp ? (steps - (int)warp + kCacheFewWarps - 1) / kCacheFewWarps : 0;     // this warp's steps of 16 tokens
  const bool whole = (c.page & 15u) == 0;            // a step's tokens lie in one page
  auto token_of = [&](int n) {
    const int v = v_begin + ((int)warp + n * kCacheFewWarps) * 16;
    return v < sink_end ? v : v + shift;
  };
  auto page_of = [&](int j) { return cache_page_at(c, b, c.by_page.of((unsigned int)j)); };
  constexpr int kSize = CODED ? 1 : 2;
  const unsigned char *const keys = (const unsigned char*)c.k, *const values = (const unsigned char*)c.v;
  int ahead = 0 < mine ? page_of(token_of(0)) : -1;  // the page of the step that is fetched next
  unsigned int to = 0;                               // the slot that is filled next
  auto fetch = [&](int n) {
    if (n < mine) {
      const int j0 = token_of(n);
      const unsigned int at = ring + to * Sh::kStage;
      const int page = ahead;
      if (whole && n + 1 < mine) ahead = page_of(token_of(n + 1));
      const unsigned int slot0 = (unsigned int)j0 - c.by_page.of((unsigned int)j0) * c.page;
      const long long head0 = whole && page >= 0 ? cache_at(c, page, hk) + (long long)slot0 * c.D : 0;
      // byte of token j0 + i, -1: not there
      auto place = [&](int i) -> long long {
        if (j0 + i >= end) return -1;
        if (whole) return page < 0 ? -1 : (head0 + (long long)i * c.D) * kSize;
        const unsigned int index = c.by_page.of((unsigned int)(j0 + i));
        const int p = cache_page_at(c, b, index);
        return p < 0 ? -1 : (cache_at(c, p, hk) + (long long)((unsigned int)(j0 + i) - index * c.page) * c.D) * kSize;
      };
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const long long from = place((int)g + 8 * k);
#pragma unroll
        for (int p = 0; p < Sh::kPerKey; ++p) {
          const int e = (int)q4 * 16 + p * 64;       // bytes
          const bool on = from >= 0 && e < c.D * kSize;
          copy_in<16>(at + (k * Sh::kPerKey + p) * 512 + lane * 16, keys + (on ? from + e : 0), on);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long from = place((int)q4 * 2 + (k & 1) + 8 * (k >> 1));
#pragma unroll
        for (int p = 0; p < Sh::kPerValue; ++p) {
          const int e = (int)g * Sh::kValueBytes + p * 16;
          const bool on = from >= 0 && e < c.D * kSize;
          copy_in<Sh::kValueWidth>(at + Sh::kKeys + (k * Sh::kPerValue + p) * 32 * Sh::kValueWidth + lane * Sh::kValueWidth, values + (on ? from + e : 0), on);
        }
      }
      if constexpr (CODED) {
        // the scales of the step's keys, then those of its values
        const int j = j0 + (int)(lane & 15u), p = whole ? page : j < end ? page_of(j) : -1;
        copy_in<4>(at + Sh::kKeys + Sh::kValues + lane * 4, (lane < 16 ? c.k_scale : c.v_scale) + (p >= 0 ? (long long)p * c.HK + hk : 0), p >= 0);
      }
      to = to + 1 == Sh::kStages ? 0 : to + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < Sh::kStages - 1; ++i) fetch(i);

  unsigned int slot = 0;
  int there = 0 < mine ? page_of(token_of(0)) : -1;  // the page of the step at hand
  for (int n = 0; n < mine; ++n) {
    const int j0 = token_of(n), page = there;
    if (whole && n + 1 < mine) there = page_of(token_of(n + 1));
    asm volatile("cp.async.wait_group %0;" ::"n"(Sh::kStages - 2) : "memory");
    __syncwarp();                     // (the scales are other lanes' copies)
    fetch(n + Sh::kStages - 1);       // into the slot of the step before
    const unsigned int at = ring + slot * Sh::kStage;
    slot = slot + 1 == Sh::kStages ? 0 : slot + 1;
    if (whole && page < 0) continue;
    float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int p = 0; p < Sh::kPerKey; ++p) {
        const uint4 v = from_shared16(at + (k * Sh::kPerKey + p) * 512 + lane * 16);
        if constexpr (CODED) {
          mma16<M>(x[k], q[4 * p], e4m3_halves(v.x & 0xffffu), e4m3_halves(v.x >> 16));
          mma16<M>(x[k], q[4 * p + 1], e4m3_halves(v.y & 0xffffu), e4m3_halves(v.y >> 16));
          mma16<M>(x[k], q[4 * p + 2], e4m3_halves(v.z & 0xffffu), e4m3_halves(v.z >> 16));
          mma16<M>(x[k], q[4 * p + 3], e4m3_halves(v.w & 0xffffu), e4m3_halves(v.w >> 16));
        } else {
          mma16<M>(x[k], q[2 * p], v.x, v.y);
          mma16<M>(x[k], q[2 * p + 1], v.z, v.w);
        }
      }
    // the scales of this lane's four tokens, 2 q4, 2 q4 + 1, and 8 further
    float back[4] = {1.f, 1.f, 1.f, 1.f}, raise[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if constexpr (CODED) {
        const uint2 ks = from_shared8(at + Sh::kKeys + Sh::kValues + q4 * 8 + 32 * k), vs = from_shared8(at + Sh::kKeys + Sh::kValues + 64 + q4 * 8 + 32 * k);
        const float k0 = cache_scale(__uint_as_float(ks.x)), k1 = cache_scale(__uint_as_float(ks.y));
        const float v0 = cache_scale(__uint_as_float(vs.x)), v1 = cache_scale(__uint_as_float(vs.y));
        x[k][0] *= k0; x[k][1] *= k1; x[k][2] *= k0; x[k][3] *= k1;
        back[2 * k] = rcp(v0);
        back[2 * k + 1] = rcp(v1);
        raise[2 * k] = __log2f(v0);
        raise[2 * k + 1] = __log2f(v1);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[k][i] *= unit[i >> 1];
    }
    if (a.cap > 0.f) {
      tanh_chunk(x[0], 1.f);
      tanh_chunk(x[1], 1.f);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] *= to_log2;
    }
    if (a.slopes)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] = fmaf(-slope2[i >> 1], (float)(pos[i >> 1] - j0 - k * 8 - (int)q4 * 2 - (i & 1)), x[k][i]);
    if constexpr (CODED)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] += raise[2 * k + (i & 1)];
    if (!whole || j0 + 15 > all_see || (a.window && j0 < all_from && j0 + 15 >= a.sinks)) {
      bool here[4] = {true, true, true, true};
      if (!whole)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = j0 + (i >> 1) * 8 + (int)q4 * 2 + (i & 1);
          here[i] = j < end && page_of(j) >= 0;
        }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int w = i >> 1, j = j0 + k * 8 + (int)q4 * 2 + (i & 1);
          const bool on = j <= last[w] && (j >= first[w] || j < a.sinks) && here[2 * k + (i & 1)];
          x[k][i] = on ? x[k][i] : -INFINITY;
        }
    }
    // the maximum in use moves when a row has outgrown it by 2^8 (or has had none): hardly ever after the first steps
    float top[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) top[w] = fmaxf(fmaxf(x[0][2 * w], x[0][2 * w + 1]), fmaxf(x[1][2 * w], x[1][2 * w + 1]));
    if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 1));
        top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 2));
        const float next = fmaxf(m[w], top[w]);
        const float by = m[w] == next ? 1.f : m[w] == -INFINITY ? 0.f : ex2(m[w] - next);
        m[w] = next;
        l[w] *= by;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][2 * w] *= by;
          o[i][2 * w + 1] *= by;
        }
      }
    }
    const float off[2] = {m[0] == -INFINITY ? 0.f : m[0] - kUp, m[1] == -INFINITY ? 0.f : m[1] - kUp};
    // weights as the A operand: rows g, g + 8, tokens 0-7 and 8-15
    unsigned int p[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float p0 = ex2(x[k][0] - off[0]), p1 = ex2(x[k][1] - off[0]), p2 = ex2(x[k][2] - off[1]), p3 = ex2(x[k][3] - off[1]);
      if constexpr (CODED) {
        l[0] = fmaf(p0, back[2 * k], fmaf(p1, back[2 * k + 1], l[0]));
        l[1] = fmaf(p2, back[2 * k], fmaf(p3, back[2 * k + 1], l[1]));
      } else {
        l[0] += p0 + p1;
        l[1] += p2 + p3;
      }
      p[2 * k] = pack2(p0, p1, M());
      p[2 * k + 1] = pack2(p2, p3, M());
    }
    // values: element g * DP / 8 + i is column g of tile i
#pragma unroll
    for (int piece = 0; piece < Sh::kPerValue; ++piece) {
      constexpr int kWords = Sh::kValueWidth / 4;
      unsigned int y[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned int from = at + Sh::kKeys + (k * Sh::kPerValue + piece) * 32 * Sh::kValueWidth + lane * Sh::kValueWidth;
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
          const unsigned int a0 = __byte_perm(y[0][i], y[1][i], 0x5140), a1 = __byte_perm(y[0][i], y[1][i], 0x7362);
          const unsigned int b0 = __byte_perm(y[2][i], y[3][i], 0x5140), b1 = __byte_perm(y[2][i], y[3][i], 0x7362);
          const int tile0 = (piece * kWords + i) * 4;
          mma16<M>(o[tile0], p, e4m3_halves(a0 & 0xffffu), e4m3_halves(b0 & 0xffffu));
          mma16<M>(o[tile0 + 1], p, e4m3_halves(a0 >> 16), e4m3_halves(b0 >> 16));
          mma16<M>(o[tile0 + 2], p, e4m3_halves(a1 & 0xffffu), e4m3_halves(b1 & 0xffffu));
          mma16<M>(o[tile0 + 3], p, e4m3_halves(a1 >> 16), e4m3_halves(b1 >> 16));
        } else {
          const int tile0 = (piece * kWords + i) * 2;
          mma16<M>(o[tile0], p, __byte_perm(y[0][i], y[1][i], 0x5410), __byte_perm(y[2][i], y[3][i], 0x5410));
          mma16<M>(o[tile0 + 1], p, __byte_perm(y[0][i], y[1][i], 0x7632), __byte_perm(y[2][i], y[3][i], 0x7632));
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
  }
  __syncthreads();                    // the rings become the place where the warps meet
  float* join = (float*)dyn;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float* row = join + (warp * 16 + g + 8 * w) * W;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < DP / 8; i += 4)
        *(float4*)(row + (2 * q4 + h) * (DP / 8) + i) = make_float4(o[i][2 * w + h], o[i + 1][2 * w + h], o[i + 2][2 * w + h], o[i + 3][2 * w + h]);
    if (q4 == 0) {
      row[DP] = m[w];
      row[DP + 1] = l[w];
    }
  }
  __syncthreads();
  const int lane_e = 4 * (int)lane;
  __shared__ float weights[kCacheFewWarps][kFewMost];
  float* parts = f.parts + (long long)blockIdx.x * 16 * W;
  // a warp takes every fourth row
  if (chunks > 1) {
    for (int i = (int)warp; i < rows; i += kCacheFewWarps) {
      float top, sum;
      few_weigh<DP>(join + i * W, kCacheFewWarps, 16 * W, weights[warp], top, sum);
      if (lane_e < DP) *(float4*)(parts + i * W + lane_e) = few_gather(join + i * W, kCacheFewWarps, 16 * W, weights[warp], lane_e, 0, 1);
      if (lane == 0) {
        parts[i * W + DP] = top;
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
  const float* all = chunks > 1 ? f.parts + (long long)first_unit * 16 * W : join;
  const int n_parts = chunks > 1 ? (int)chunks : kCacheFewWarps;
  for (int i = (int)warp; i < rows; i += kCacheFewWarps) {
    float top, sum;
    few_weigh<DP>(all + i * W, n_parts, 16 * W, weights[warp], top, sum);
    bool fine = true;
    if (lane_e < DP) fine = cache_finish<T>(a, s.first + query_of(i), head_of(i), lane_e, few_gather(all + i * W, n_parts, 16 * W, weights[warp], lane_e, 0, 1), top, sum, kUp);
    if (attn_again(fine)) cache_attention_row<T, CODED>(a, b, head_of(i), s.first + query_of(i), s.pos0 + query_of(i), lane);
  }
}

}  // namespace b200
#endif
