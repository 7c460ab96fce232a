// New keys and values into a paged cache, with the rotary turn applied on the way, and queries turned beside them.
//
//   (a, b) -> m (a cos - b sin, a sin + b cos), once rounded;  in 8 bits: code = e4m3(x / 2^e), e the least with max|x| <= 448 * 2^e over the page's values
//
// Bound by memory: every new element is read and written once.  Angles are kept as 64-bit fractions of a turn, as the rotary operator has them.
// One launch with two kinds of blocks.  Rows that go where they lie, or to a cache of their own type, are taken a few tokens a block, all heads: one
// table of cosines and sines serves them.  Rows that become codes are taken a page of a sequence a block (keys and values apart), since a page's scale
// of a head needs all its values first: a warp (or a few) a head reads them twice, the second time from the caches, and no block has to wait for
// another.  Scales are powers of two, so that codes a page holds already lose nothing when its scale grows.
// Measured: prompts of 8192 tokens together, 32 heads over 8 of 128, codes, 59 to 65 us on several machines (floor 26): 37 million instructions of warps (keys turn
// twice, and a page makes its table) at half of the issue slots, with a third of the warps that an SM has room for, and with pieces that 80 registers a thread do not
// hold (524 bytes a thread go to memory and back); the same into a cache of 16 bits 40 us.  256 sequences' tokens, codes, 9.2 us: a chain of dependent
// accesses, of which the codes of a page whose scale grows, four bytes a lane one after another, are the longest.
#include <cmath>

#include "cache.hpp"

using namespace b200;

namespace {

struct AppendArgs {
  CacheArgs c;
  const void *k, *v, *q;
  void* q_out;
  const int* positions;
  const unsigned long long* turns;     // [pairs], of a turn per position, scaled by 2^64
  unsigned int heads, d, pairs;
  unsigned int turn_items, items, v_items;     // accesses of a head that turn, all of a head that turns, of a value head
  unsigned int per_block;              // tokens of a block of rows that need no scale
  unsigned int turned_rows, plain_items;       // of a token: rows that turn, and all accesses, of such a block
  unsigned int code_blocks, pages_each;        // blocks that make codes; pages that a sequence's tokens touch at most, without starts
  unsigned int tile;                   // tokens of a table, of a block that makes codes
  unsigned int per_head;               // warps of a head there
  unsigned int heads_each, groups;     // heads of such a block; blocks of a page's keys, or values
  Divisor by_pairs, by_items, by_v_items, by_plain, by_pages_each, by_groups;
  float magnitude;
};

constexpr int kAtOnce = 4;             // accesses of a thread under way together
constexpr int kThreads = 256, kWarps = kThreads / 32;

__device__ __forceinline__ float2 turn_of(const AppendArgs& a, int position, unsigned int pair) {
  const unsigned long long turn = (unsigned long long)(long long)position * a.turns[pair];
  // the nearest of 2^32 steps of a turn, as a signed number: the angle is step * 2 pi / 2^32
  const int step = (int)(unsigned int)((turn + 0x80000000ull) >> 32);
  float s, c;
  sincospif((float)step * 4.656612873077393e-10f, &s, &c);
  return make_float2(c * a.magnitude, s * a.magnitude);
}

// The table's pairs as an access takes them: kPairs of an item side by side, and 16 bytes between items where that keeps the 16-byte reads of eight lanes,
// each of an item of its own, out of one another's banks.
template <int VEC, bool INTERLEAVED>
struct Table {
  static constexpr int kPairs = VEC == 1 ? 1 : INTERLEAVED ? VEC / 2 : VEC, kPitch = kPairs >= 4 ? kPairs + 2 : kPairs;
  __host__ __device__ static constexpr unsigned int row(unsigned int pairs) { return pairs / kPairs * kPitch; }
  __device__ static unsigned int at(unsigned int pair) { return pair / kPairs * kPitch + pair % kPairs; }
};

// One access of a head: a vector, or with pairs that lie apart two (the second `far` elements behind the first)
template <class T, int VEC, bool INTERLEAVED>
struct Piece {
  static constexpr bool kSplit = !INTERLEAVED || VEC == 1;
  Raw<T, VEC> u, w;
  unsigned int item, at;               // at: the first element
  bool turns;
  __device__ __forceinline__ void load(const T* row, unsigned int i, unsigned int turn_items, unsigned int pairs) {
    item = i;
    turns = i < turn_items;
    if (!turns) at = (turn_items ? 2 * pairs : 0u) + (i - turn_items) * VEC;
    else at = INTERLEAVED && VEC == 1 ? 2 * i : i * VEC;
    u.load(row + at);
    if (kSplit && turns) w.load(row + at + far(pairs));
  }
  __device__ __forceinline__ unsigned int far(unsigned int pairs) const { return INTERLEAVED ? 1u : pairs; }
  typedef Table<VEC, INTERLEAVED> Tab;
  __device__ __forceinline__ void pairs_of(const float2* cs, float2 (&t)[Tab::kPairs]) const {
    const float2* from = cs + item * Tab::kPitch;
    if constexpr (Tab::kPairs == 1) {
      t[0] = from[0];
    } else {
#pragma unroll
      for (int q = 0; q < Tab::kPairs; q += 2) {
        const float4 v = *(const float4*)(from + q);
        t[q] = make_float2(v.x, v.y);
        t[q + 1] = make_float2(v.z, v.w);
      }
    }
  }
  // the values, turned; y only where pairs lie apart
  __device__ __forceinline__ void values(const float2* cs, float (&x)[VEC], float (&y)[VEC]) const {
    u.values(x);
    if (!turns) return;
    if constexpr (kSplit) {
      w.values(y);
      float2 t[VEC];
      pairs_of(cs, t);
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        const float x0 = x[q], y0 = y[q];
        x[q] = x0 * t[q].x - y0 * t[q].y;
        y[q] = x0 * t[q].y + y0 * t[q].x;
      }
    } else {
      float2 t[VEC / 2];
      pairs_of(cs, t);
#pragma unroll
      for (int q = 0; q < VEC / 2; ++q) {
        const float x0 = x[2 * q], y0 = x[2 * q + 1];
        x[2 * q] = x0 * t[q].x - y0 * t[q].y;
        x[2 * q + 1] = x0 * t[q].y + y0 * t[q].x;
      }
    }
  }
};

template <int VEC>
__device__ __forceinline__ void store_codes(unsigned char* to, const float (&x)[VEC], float by) {
  float v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = e4m3_has(x[i]) ? x[i] * by : __int_as_float(0x7fffffff);
  if constexpr (VEC == 1) *to = (unsigned char)e4m3_pack2(v[0], 0.f);
  else if constexpr (VEC == 4) *(unsigned int*)to = e4m3_pack2(v[0], v[1]) | e4m3_pack2(v[2], v[3]) << 16;
  else *(uint2*)to = make_uint2(e4m3_pack2(v[0], v[1]) | e4m3_pack2(v[2], v[3]) << 16, e4m3_pack2(v[4], v[5]) | e4m3_pack2(v[6], v[7]) << 16);
}

template <class T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void plain_rows(const AppendArgs& a, unsigned int block, float2* table, bool coded) {
  typedef Piece<T, VEC, INTERLEAVED> P;
  const CacheArgs& c = a.c;
  __shared__ int positions[kThreads];            // of the block's tokens
  __shared__ long long slots[kThreads];          // elements of the cache ahead of head 0 of a token's slot; -1: no slot, -2: no sequence
  const unsigned int first = block * a.per_block, n = min(a.per_block, (unsigned int)c.tokens - first), total = n * a.plain_items;
  const unsigned int turned = a.turned_rows * a.items;
  P it[kAtOnce];
  unsigned int tok[kAtOnce], row[kAtOnce];
  auto fetch = [&](unsigned int i, int k) {
    if (i >= total) return;
    tok[k] = a.by_plain.of(i);
    unsigned int j = i - tok[k] * a.plain_items;
    const unsigned long long t = first + tok[k];
    if (j < turned) {
      row[k] = a.by_items.of(j);
      const T* from = row[k] < a.heads ? (const T*)a.q + (t * a.heads + row[k]) * a.d : (const T*)a.k + (t * (unsigned int)c.HK + (row[k] - a.heads)) * a.d;
      it[k].load(from, j - row[k] * a.items, a.turn_items, a.pairs);
    } else {
      j -= turned;
      const unsigned int r = a.by_v_items.of(j);
      row[k] = a.turned_rows + r;
      it[k].load((const T*)a.v + (t * (unsigned int)c.HK + r) * a.d, j - r * a.v_items, 0u, 0u);
    }
  };
  // the first accesses are under way while places and table are made
#pragma unroll
  for (int k = 0; k < kAtOnce; ++k) fetch(threadIdx.x + kThreads * k, k);
  if (threadIdx.x < n) {
    const int t = (int)(first + threadIdx.x);
    int b;
    if (c.starts) {
      int lo = 0, hi = c.batch;                  // the last sequence that starts at the row or before it
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(c.starts + mid) <= t) lo = mid;
        else hi = mid;
      }
      b = lo;
    } else {
      b = t / c.each;
    }
    const CacheSeq s = cache_seq(c, b);
    const bool there = t >= s.first && t < s.first + s.count;
    const int pos = s.pos0 + (t - s.first);
    long long slot = there ? -1 : -2;
    if (there && pos >= 0 && !coded) {
      const unsigned int index = c.by_page.of((unsigned int)pos);
      const int page = cache_page_at(c, b, index);
      if (page >= 0) slot = cache_at(c, page, 0) + (long long)((unsigned int)pos - index * c.page) * c.D;
    }
    slots[threadIdx.x] = slot;
    positions[threadIdx.x] = a.positions ? a.positions[t] : pos;
  }
  __syncthreads();
  const unsigned int row_of_table = P::Tab::row(a.pairs);
  for (unsigned int i = threadIdx.x; i < n * a.pairs; i += kThreads) {
    const unsigned int t = a.by_pairs.of(i), pair = i - t * a.pairs;
    table[t * row_of_table + P::Tab::at(pair)] = turn_of(a, positions[t], pair);
  }
  __syncthreads();
  const long long head = (long long)c.page * c.D;      // from one head of a page to the next
  for (unsigned int base = 0; base < total; base += kThreads * kAtOnce) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (base + threadIdx.x + kThreads * k >= total) continue;
      const long long slot = slots[tok[k]];
      T* to;
      if (row[k] < a.heads) {
        if (slot == -2) continue;
        to = (T*)a.q_out + ((unsigned long long)(first + tok[k]) * a.heads + row[k]) * a.d;
      } else {
        if (slot < 0) continue;
        const bool value = row[k] >= a.turned_rows;
        to = (T*)(value ? c.v : c.k) + slot + (long long)(row[k] - (value ? a.turned_rows : a.heads)) * head;
      }
      float x[VEC], y[VEC];
      it[k].values(table + tok[k] * row_of_table, x, y);
      Vec<T, VEC>::store(to + it[k].at, x);
      if (P::kSplit && it[k].turns) Vec<T, VEC>::store(to + it[k].at + it[k].far(a.pairs), y);
    }
    if (base + kThreads * kAtOnce < total)
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) fetch(base + kThreads * (kAtOnce + k) + threadIdx.x, k);
  }
}

// A page of a sequence: its new keys, or values, become codes.
template <class T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void page_codes(const AppendArgs& a, float2* table) {
  typedef Piece<T, VEC, INTERLEAVED> P;
  const CacheArgs& c = a.c;
  __shared__ float largest[kWarps];
  const unsigned int block = a.by_groups.of(blockIdx.x), first_head = (blockIdx.x - block * a.groups) * a.heads_each, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const unsigned int unit = block >> 1;           // of pages
  const bool value = block & 1u;
  // pages that a sequence's new tokens touch
  auto pages_of = [&](const CacheSeq& s) -> unsigned int {
    const int end = s.pos0 + s.count, begin = max(s.pos0, 0);
    return s.count > 0 && end > begin ? c.by_page.of((unsigned int)(end - 1)) - c.by_page.of((unsigned int)begin) + 1u : 0u;
  };
  int b;
  unsigned int nth;
  if (c.starts) {
    if (!find_unit<kThreads>(c.batch, unit, [&](int i) { return pages_of(cache_seq(c, i)); }, b, nth)) return;
  } else {
    b = (int)a.by_pages_each.of(unit);
    nth = unit - (unsigned int)b * a.pages_each;
  }
  const CacheSeq s = cache_seq(c, b);
  if (nth >= pages_of(s)) return;
  const unsigned int begin0 = (unsigned int)max(s.pos0, 0), index = c.by_page.of(begin0) + nth;
  const int page = cache_page_at(c, b, index);
  if (page < 0) return;
  const unsigned int begin = max(begin0, index * c.page), end = (unsigned int)min((unsigned long long)(s.pos0 + s.count), (unsigned long long)(index + 1) * c.page);
  const unsigned int n = end - begin, slot = begin - index * c.page;       // new tokens of the page, and those that it holds
  const unsigned int row0 = (unsigned int)(s.first + ((int)begin - s.pos0));
  const T* from = (const T*)(value ? a.v : a.k);
  float* scales = (value ? c.v_scale : c.k_scale) + (long long)page * c.HK;
  unsigned char* codes = (unsigned char*)(value ? c.v : c.k);
  const unsigned int items = value ? a.v_items : a.items, turn_items = value ? 0u : a.turn_items;
  const Divisor by_items = value ? a.by_v_items : a.by_items;
  const unsigned int heads = min(first_head + a.heads_each, (unsigned int)c.HK), at_once = kWarps / a.per_head, share = warp % a.per_head;
  const bool one_table = n <= a.tile;
  const unsigned int row_of_table = P::Tab::row(a.pairs);
  auto make_table = [&](unsigned int t0) {
    if (!turn_items) return;
    __syncthreads();
    const unsigned int many = min(a.tile, n - t0) * a.pairs;
    for (unsigned int i = threadIdx.x; i < many; i += kThreads) {
      const unsigned int t = a.by_pairs.of(i), pair = i - t * a.pairs;
      table[t * row_of_table + P::Tab::at(pair)] = turn_of(a, a.positions ? a.positions[row0 + t0 + t] : (int)(begin + t0 + t), pair);
    }
    __syncthreads();
  };
  // A few tokens: a lane keeps its pieces, which are under way while the table is made; more are read twice.
  const bool kept = n * items <= 32 * a.per_head * kAtOnce;        // (no more than a table is for)
  P held[kAtOnce];
  auto hold = [&](unsigned int h0) {
    const unsigned int h = h0 + warp / a.per_head;
    if (h >= heads || warp >= at_once * a.per_head) return;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const unsigned int i = share * 32 + lane + 32 * a.per_head * k;
      if (i >= n * items) continue;
      const unsigned int t = by_items.of(i);
      held[k].load(from + ((unsigned long long)(row0 + t) * (unsigned int)c.HK + h) * a.d, i - t * items, turn_items, turn_items ? a.pairs : 0u);
    }
  };
  if (kept) hold(first_head);
  if (one_table) make_table(0);
  for (unsigned int h0 = first_head; h0 < heads; h0 += at_once) {
    const unsigned int h = h0 + warp / a.per_head;
    const bool mine = h < heads && warp < at_once * a.per_head;
    const float before = mine && slot ? scales[h] : 0.f;
    // all pieces of this warp's share: f(piece, token of the page's new ones, cosines and sines of its token)
    auto each = [&](auto&& f) {
      if (kept) {
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const unsigned int i = share * 32 + lane + 32 * a.per_head * k;
          if (!mine || i >= n * items) continue;
          const unsigned int t = by_items.of(i);
          f(held[k], t, table + t * row_of_table);
        }
        return;
      }
      for (unsigned int t0 = 0; t0 < n; t0 += a.tile) {
        if (!one_table) make_table(t0);
        const unsigned int many = mine ? min(a.tile, n - t0) * items : 0u;
        for (unsigned int i0 = share * 32 + lane; i0 < many; i0 += 32 * a.per_head * kAtOnce) {
          unsigned int tok[kAtOnce];
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) {
            const unsigned int i = i0 + 32 * a.per_head * k;
            if (i >= many) continue;
            tok[k] = by_items.of(i);
            held[k].load(from + ((unsigned long long)(row0 + t0 + tok[k]) * (unsigned int)c.HK + h) * a.d, i - tok[k] * items, turn_items, turn_items ? a.pairs : 0u);
          }
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k)
            if (i0 + 32 * a.per_head * k < many) f(held[k], t0 + tok[k], table + tok[k] * row_of_table);
        }
      }
    };
    float top = 0.f;
    each([&](const P& p, unsigned int, const float2* cs) {
      float x[VEC], y[VEC];
      p.values(cs, x, y);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (e4m3_has(x[i])) top = fmaxf(top, fabsf(x[i]));
        if (P::kSplit && p.turns && e4m3_has(y[i])) top = fmaxf(top, fabsf(y[i]));
      }
    });
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));       // (of numbers that are not negative)
    if (lane == 0) largest[warp] = top;
    __syncthreads();
    for (unsigned int i = 0; i < a.per_head; ++i) top = fmaxf(top, largest[(warp - share + i) % kWarps]);
    const int e = e4m3_exponent(top);
    float scale = power_of_two(e), by = power_of_two(-e);
    const bool grows = !(before >= scale);
    if (!grows) {
      scale = before;
      by = 1.f / before;               // (exact: a power of two, where this operator wrote it)
    }
    const long long at = mine ? cache_at(c, page, (int)h) : 0;
    if (mine && slot && grows) {
      // what the page holds, in units of the new scale
      const float back = before * by;
      const unsigned int held = slot * a.d;
      if constexpr (VEC > 1) {
        for (unsigned int i = (share * 32 + lane) * 4; i < held; i += 128 * a.per_head) {
          unsigned int* p = (unsigned int*)(codes + at + i);
          const float2 lo = e4m3_unpack2(*p & 0xffffu), hi = e4m3_unpack2(*p >> 16);
          *p = e4m3_pack2(lo.x * back, lo.y * back) | e4m3_pack2(hi.x * back, hi.y * back) << 16;
        }
      } else {
        for (unsigned int i = share * 32 + lane; i < held; i += 32 * a.per_head) codes[at + i] = (unsigned char)e4m3_pack2(e4m3_value(codes[at + i]) * back, 0.f);
      }
    }
    each([&](const P& p, unsigned int t, const float2* cs) {
      float x[VEC], y[VEC];
      p.values(cs, x, y);
      unsigned char* to = codes + at + (unsigned long long)(slot + t) * a.d + p.at;
      store_codes<VEC>(to, x, by);
      if (P::kSplit && p.turns) store_codes<VEC>(to + p.far(a.pairs), y, by);
    });
    if (mine && share == 0 && lane == 0 && (grows || !slot)) scales[h] = scale;
    if (kept && h0 + at_once < heads) hold(h0 + at_once);
    __syncthreads();                   // (`largest` is written again)
  }
}

template <class T, int VEC, bool INTERLEAVED, bool CODED>
__global__ void __launch_bounds__(kThreads, 3) cache_append(const __grid_constant__ AppendArgs a) {
  extern __shared__ __align__(16) float2 table[];    // [token][pair]: cosine, sine, times the magnitude
  grid_begin();
  // (pages first: they take longer)
  if (CODED && blockIdx.x < a.code_blocks) page_codes<T, VEC, INTERLEAVED>(a, table);
  else plain_rows<T, VEC, INTERLEAVED>(a, blockIdx.x - a.code_blocks, table, CODED);
}

typedef void (*AppendKernel)(const AppendArgs);

template <class T>
AppendKernel kernel_of(bool vec, bool interleaved, bool coded) {
  constexpr int V = 16 / (int)sizeof(T);
  if (coded) {
    if (vec) return interleaved ? cache_append<T, V, true, true> : cache_append<T, V, false, true>;
    return interleaved ? cache_append<T, 1, true, true> : cache_append<T, 1, false, true>;
  }
  if (vec) return interleaved ? cache_append<T, V, true, false> : cache_append<T, V, false, false>;
  return interleaved ? cache_append<T, 1, true, false> : cache_append<T, 1, false, false>;
}

struct AppendOperator : b200_operator {
  AppendArgs a = {};
  AppendKernel kernel = nullptr;
  unsigned int grid = 0;
  size_t smem = 0;
  void run(cudaStream_t s) override {
    if (grid) launch(kernel, dim3(grid), kThreads, smem, s, a);
  }
};

}  // namespace

extern "C" int b200_cache_append_link(b200_dev* dev, const b200_cache_append* p, b200_operator** out) {
  return link_operator<AppendOperator>(dev, p, out, [&](AppendOperator* op) {
    Operands ops(op, "cache_append");
    ops.dtype(p->dtype);
    const b200_cache& pc = p->cache;
    AppendArgs& a = op->a;
    a.c = bind_cache(ops, pc, p->dtype, true);
    if (pc.d > 1024) ops.refuse("heads of more than 1024 elements", B200_E_UNSUPPORTED);
    if (p->heads < 0 || p->heads > 65535) ops.refuse("heads must be between 0 and 65535");
    if (p->pairs < 0 || 2ll * p->pairs > pc.d) ops.refuse("2 * pairs must not exceed d");
    if (p->pairs && !p->frequencies) ops.refuse("'frequencies' is required");
    if (!std::isfinite(p->magnitude)) ops.refuse("the magnitude must be finite");
    for (int i = 0; i < p->pairs; ++i)
      if (!std::isfinite(p->frequencies[i])) ops.refuse("a frequency is not finite");
    const bool coded = pc.dtype == B200_E4M3;
    const size_t size = dtype_bytes(p->dtype);
    const unsigned long long rows = extent_product({pc.tokens, pc.kv_heads, pc.d}, "cache_append"), q_rows = extent_product({pc.tokens, p->heads, pc.d}, "cache_append");
    a.k = (const void*)ops.in(p->k, "k", rows, size);
    a.v = (const void*)ops.in(p->v, "v", rows, size);
    if (p->heads) {
      a.q = (const void*)ops.in(p->q, "q", q_rows, size);
      a.q_out = (void*)ops.out(p->q_out, "q_out", q_rows, size);
    }
    a.positions = (const int*)ops.in(p->positions, "positions", (unsigned long long)pc.tokens, 4, false);
    ops.check_overlaps({{"q_out", "q"}});
    const unsigned int V = 16 / (unsigned int)size;
    a.heads = (unsigned int)p->heads;
    a.d = (unsigned int)pc.d;
    a.pairs = (unsigned int)p->pairs;
    a.magnitude = p->magnitude;
    bool vec = a.d % V == 0 && (p->interleaved ? 2 * a.pairs % V == 0 : a.pairs % V == 0);
    for (const void* n : {a.k, a.v, a.q, (const void*)a.q_out, (const void*)a.c.k, (const void*)a.c.v}) vec &= ((size_t)n & 15) == 0;
    const unsigned int v = vec ? V : 1;
    a.turn_items = p->interleaved ? (vec ? 2 * a.pairs / v : a.pairs) : a.pairs / v;
    a.items = a.turn_items + (a.d - 2 * a.pairs) / v;
    a.v_items = a.d / v;
    a.turned_rows = a.heads + (coded ? 0u : (unsigned int)pc.kv_heads);
    const unsigned long long per_token = (unsigned long long)a.turned_rows * a.items + (coded ? 0ull : (unsigned long long)pc.kv_heads * a.v_items);
    a.by_pairs = Divisor(std::max(1u, a.pairs));
    a.by_items = Divisor(a.items);
    a.by_v_items = Divisor(a.v_items);
    // (Table: pairs of an item, and the floats between items)
    const unsigned int of_item = !vec ? 1 : p->interleaved ? V / 2 : V, row_of_table = a.pairs / of_item * (of_item >= 4 ? of_item + 2 : of_item);
    unsigned long long plain = 0, codes = 0;
    size_t table = 0;
    if (pc.tokens && pc.batch && per_token) {
      // About four accesses a thread, while that leaves the machine enough blocks; a table of at most 4096 pairs (32 KB, and the gaps between
      // items: 40 KB in 16 bits, 48 in single precision, where pairs lie apart)
      unsigned long long tok = std::max(1ull, 1024ull / per_token);
      tok = std::min(tok, std::max(1ull, (unsigned long long)pc.tokens / (2ull * (unsigned)dev->sm_count)));
      if (a.pairs) tok = std::min(tok, std::max(1ull, 4096ull / a.pairs));
      tok = std::min(tok, (unsigned long long)kThreads);
      if (tok * per_token >> 31) ops.refuse("a token has too many elements", B200_E_UNSUPPORTED);
      a.per_block = (unsigned int)tok;
      a.plain_items = (unsigned int)per_token;
      a.by_plain = Divisor(a.plain_items);
      plain = ((unsigned long long)pc.tokens + tok - 1) / tok;
      table = (size_t)tok * row_of_table * 8;
    }
    if (coded && pc.tokens && pc.batch) {
      // Of n >= 1 tokens a sequence touches at most (n - 2) / page + 2 pages (rounded down, 1 of one token)
      const long long some = std::min<long long>(pc.batch, pc.tokens), page = pc.page;
      codes = (unsigned long long)std::min<long long>(pc.tokens, (pc.tokens + some * (page - 2)) / page + some);
      if (!a.c.starts) {
        a.pages_each = (unsigned int)((a.c.each + page - 2) / page + 1);
        codes = (unsigned long long)a.pages_each * (unsigned long long)pc.batch;
      }
      a.by_pages_each = Divisor(std::max(1u, a.pages_each));
      // A table of at most 8192 pairs, 64 to 96 KB (two blocks an SM then; three where pages of 64 tokens of 64 pairs need 40 KB), and no fewer tokens than lanes
      // keep the pieces of, all of which look into one table.
      a.tile = (unsigned int)std::min<long long>(page, a.pairs ? std::max(8192u / a.pairs, std::max(1u, (unsigned int)(kThreads * kAtOnce) / a.items)) : page);
      table = std::max(table, (size_t)std::min<long long>(a.tile, pc.tokens) * row_of_table * 8);
      // Warps of a head: no fewer than hold what a page receives of it, as many as there are where heads are few.  (A block a page and all its heads, each read
      // twice by one warp: 75 us for 8192 tokens of 8 heads, pages of 64.)
      const long long fill = std::min<long long>(page, pc.tokens / some) * a.v_items;
      a.per_head = 1;
      while (a.per_head < (unsigned int)kWarps && ((long long)a.per_head * 32 * kAtOnce < fill || (long long)kWarps / a.per_head >= 2ll * pc.kv_heads)) a.per_head *= 2;
      a.heads_each = std::max(2u, (unsigned int)kWarps / a.per_head);
      a.groups = ((unsigned int)pc.kv_heads + a.heads_each - 1) / a.heads_each;
      a.by_groups = Divisor(a.groups);
    }
    codes *= 2 * a.groups;
    if ((plain + codes) >> 31) ops.refuse("too many tokens", B200_E_UNSUPPORTED);
    a.code_blocks = (unsigned int)codes;
    op->grid = (unsigned int)(plain + codes);
    op->smem = table;
    op->kernel = p->dtype == B200_F32 ? kernel_of<float>(vec, p->interleaved, coded) : p->dtype == B200_BF16 ? kernel_of<__nv_bfloat16>(vec, p->interleaved, coded)
                                                                                                            : kernel_of<__half>(vec, p->interleaved, coded);
    ready(op->kernel, table);
    if (!a.pairs) return;
    op->take_workspace((size_t)a.pairs * 8);
    write_turns(op, op->workspace, p->frequencies, p->pairs);
    a.turns = (const unsigned long long*)op->workspace;
  });
}
