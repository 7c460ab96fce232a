// Attention for 16-bit heads on the tensor cores, any number of keys: softmax with a running maximum and sum.
//
// A CTA takes NQ tiles of 128 queries of one (sequence, head).  Roles: a warp that copies (TMA: the queries once, then tiles of
// 64 or 128 keys and values through rings), a warp that issues tcgen05.mma, and four warps per query tile that do the softmax, a thread
// a row.  Scores of a tile lie in tensor memory (128 columns: one tile of 128 keys, or two of 64, of which the next one's scores are formed
// during the softmax of this); the thread loads its row, 32 scores at a time, applies cap, bias and mask, takes
// the maximum, writes the weights exp2(s - m) in 16 bits over the scores, and they are the A operand of the second product, which adds
// to the output accumulators in tensor memory.  The accumulators are only multiplied by 2^(m_old - m_new) when a row's maximum has
// grown by more than 2^8 (weights stay below that, sums and accumulators are single precision, so nothing is lost): after the
// first tiles hardly ever.  With NQ = 2 the two tiles take turns on the tensor cores and on the arithmetic; with NQ = 1 two CTAs of an SM do.
//
// Over more than kSumKeys keys (SUMS) the accumulators are added to sums in the workspace every so many tiles, and cleared.  (In all
// kernels, never taken, the branch cost 5 % of the shorter rows' time.)
//
// Key tiles that no query of a tile sees are skipped, and those that all see take no mask: known from the rows' last keys alone, or, with
// documents, from classes made first for all key tiles from the range of document numbers in each.
//
// Short sequences are bound by the chain from a CTA's start to its end (64 sequences of 256 positions, 8 heads of 64: 9600 cycles, of which
// 1200 were the classes, 1800 the wait for the first operands, 1800 the way out): so the copies start before anything else, and every
// warp sends its own 32 rows out.
#ifndef B200_ATTN_FWD_SM100_CUH
#define B200_ATTN_FWD_SM100_CUH
#include "attn_terms.cuh"
#ifndef B200_ELEM_BYTES
#define B200_ELEM_BYTES 2
#endif
#include "tc_sm100.cuh"
#include <type_traits>

namespace b200 {

constexpr unsigned int kTileBytes64 = 128 * 128;   // 128 rows x 64 elements of 16 bits: one swizzled panel

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh x = 1 - 2 / (e^2x + 1), of which 2 x log2(e) is given; off by a few 2^-24 (absolute), which a cap multiplies
__device__ __forceinline__ float tanh_of(float two_x_log2e) { return fmaf(-2.f, rcp(ex2(two_x_log2e) + 1.f), 1.f); }

// x = tanh(x scale) of N scores of each lane.  The exponential and the reciprocal of tanh_of pass through the unit that also has to make
// the weights, at an eighth of the multiply-adds' rate, and would bound the kernel: where all of a warp's scores are at most the cap in
// size, tanh y = y + y^3 Q(y^2) instead, with Q the polynomial of degree 5 whose largest error on [0, 1] is least (3.0e-8, 8e-8 in single
// precision, 1.6e-7 relative; fitted by iterated weighted least squares).  2 x 4096 positions, 16 heads of 128, causal: 301 us without,
// 226 with it and tiles of 64 keys.
template <int N>
__device__ __forceinline__ void tanh_chunk(float (&x)[N], float scale) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(x[j]));
  if (__any_sync(0xffffffffu, top * scale > 1.f)) {
    const float s = 2.f * kLog2e * scale;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = tanh_of(x[j] * s);
    return;
  }
  const Pair s(scale, scale);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const Pair y = mul2(Pair(x[j], x[j + 1]), s), z = mul2(y, y);
    Pair p = fma2(z, Pair(0.0010059071937575936f, 0.0010059071937575936f), Pair(-0.00609551602974534f, -0.00609551602974534f));
    p = fma2(p, z, Pair(0.020165905356407166f, 0.020165905356407166f));
    p = fma2(p, z, Pair(-0.053391970694065094f, -0.053391970694065094f));
    p = fma2(p, z, Pair(0.13323739171028137f, 0.13323739171028137f));
    p = fma2(p, z, Pair(-0.3333275318145752f, -0.3333275318145752f));
    fma2(mul2(y, z), p, y).get(x[j], x[j + 1]);
  }
}

// Weights are at most 2^8 (the maximum in use may lag by that).  Half ones are multiplied by 2^7 more, which the row's sum has too: those
// down to 2^-21 of the largest are then normal numbers.  (Many keys of 2^-20 beside one of 1 kept four bits: outputs were 3 % off.)
template <class T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;

// A from tensor memory: 16-bit elements, two to a column
__device__ __forceinline__ void umma_ts(unsigned int d, unsigned int a, unsigned long long b, unsigned int idesc, unsigned int accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(unsigned int taddr, const unsigned int* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// The next kernel in the stream may be placed from here on, and not before this block has its tensor memory: one that took it first would
// wait for this kernel's end, and this block for the memory.
__device__ __forceinline__ void tmem_taken() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class T>
__host__ __device__ constexpr unsigned int idesc_of(int m, int n, bool a_mn, bool b_mn) {
  const unsigned int f = sizeof(T) == 2 ? (std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((unsigned int)(n / 8) << 17) | ((unsigned int)(m / 16) << 24);
}

// what a tile of rows sees: the least and the greatest last key, the range of documents
struct AttnSpan {
  int last_min, last_max, doc_min, doc_max;
};
// of rows r0 .. r0 + n - 1, without documents
__device__ __forceinline__ AttnSpan plain_span(const AttnArgs& a, const AttnSeq& q, int r0, int n) {
  AttnSpan s;
  s.last_min = r0 < a.S ? attn_last(a, q, r0) : 0x7fffffff;
  s.last_max = r0 < a.S ? attn_last(a, q, min(r0 + n, a.S) - 1) : -1;
  s.doc_min = s.doc_max = 0;
  return s;
}
__device__ __forceinline__ AttnSpan span_of(bool ok, const AttnRow& w) {
  AttnSpan s;
  s.last_min = __reduce_min_sync(0xffffffffu, ok ? w.last : 0x7fffffff);
  s.last_max = __reduce_max_sync(0xffffffffu, ok ? w.last : -1);
  s.doc_min = __reduce_min_sync(0xffffffffu, ok ? w.doc : 0x7fffffff);
  s.doc_max = __reduce_max_sync(0xffffffffu, ok ? w.doc : -0x7fffffff - 1);
  return s;
}
// 0: no row sees a key of the tile, 1: every row sees every key, 2: some
__device__ __forceinline__ unsigned int tile_class(const AttnSpan& s, int j0, int width, bool docs, int kmin, int kmax, bool negative) {
  if (j0 > s.last_max) return 0u;
  if (!docs) return j0 + width - 1 <= s.last_min ? 1u : 2u;
  if (kmax < s.doc_min || kmin > s.doc_max) return 0u;
  return (j0 + width - 1 <= s.last_min && !negative && kmin == kmax && s.doc_min == s.doc_max && s.doc_min == kmin) ? 1u : 2u;
}
// Ranges of the non-negative documents of the W keys of each of N tiles from tile t on, `step` apart (a warp); `negative`: some are
// padding.  All loads are under way before the first is used.
template <int W, int N>
__device__ __forceinline__ void key_documents(const AttnArgs& a, int b, int t, int step, unsigned int lane, int (&kmin)[N], int (&kmax)[N], bool (&negative)[N]) {
  int d[N][W / 32];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < W / 32; ++i) {
      const long long j = (long long)(t + n * step) * W + lane + 32 * i;
      d[n][i] = j < a.T ? __ldg(a.kdoc + (long long)b * a.T + j) : -0x7fffffff - 1;      // (no key: neither a document nor padding)
    }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int lo = 0x7fffffff, hi = -1, bad = 0;
#pragma unroll
    for (int i = 0; i < W / 32; ++i) {
      if (d[n][i] < 0) bad |= d[n][i] != -0x7fffffff - 1;
      else { lo = min(lo, d[n][i]); hi = max(hi, d[n][i]); }
    }
    kmin[n] = __reduce_min_sync(0xffffffffu, lo);
    kmax[n] = __reduce_max_sync(0xffffffffu, hi);
    negative[n] = __any_sync(0xffffffffu, bad);
  }
}
// Which of 32 N keys from j0 the lane's row sees, a bit each.  The rows of a warp belong to one document or a few: one round each.
template <int N>
__device__ __forceinline__ void visible_words(const AttnArgs& a, int b, int j0, const AttnRow& w, unsigned int lane, unsigned int (&bits)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int n = w.last + 1 - (j0 + 32 * i);       // keys of this word up to the last one
    bits[i] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
  }
  if (!a.kdoc) return;
  int d[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = j0 + (int)lane + 32 * i;
    d[i] = j < a.T ? a.kdoc[(long long)b * a.T + j] : -1;
  }
  unsigned int todo = 0xffffffffu;
  while (todo) {
    const int doc = __shfl_sync(0xffffffffu, w.doc, __ffs(todo) - 1);
    const bool mine = w.doc == doc;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned int same = __ballot_sync(0xffffffffu, d[i] == doc);
      if (mine) bits[i] &= same;
    }
    todo &= ~__ballot_sync(0xffffffffu, mine);
  }
}

// KW: keys of a tile.  With 64 the scores have two places in tensor memory, and those of the next tile are formed while the softmax of
// this one runs; with 128 one, and they wait for its weights.
template <int DP, int NQ, int KW>
struct FwdShape {
  static constexpr int kPanels = DP / 64, kScores = 128 / KW;
  static constexpr unsigned int kTile = kPanels * kTileBytes64;              // queries
  static constexpr unsigned int kPanel = KW * 128, kKeys = kPanels * kPanel; // keys or values
  // slots for keys and for values: 64 KB together with two query tiles or two CTAs an SM
  static constexpr int kSlots = (DP == 128 && NQ == 1) ? 128 / KW : 2 * 128 / KW;
  static constexpr unsigned int kThreads = NQ * 128 + 64;
  static constexpr unsigned int kBytes = NQ * kTile + 2 * kSlots * kKeys;
  static constexpr unsigned int kColumns = NQ * (128 + DP) <= 256 ? 256 : 512;
  static constexpr size_t smem(int tiles) { return 1024 + kBytes + 512 + (size_t)tiles; }
};

template <class T, int DP, int NQ, int KW, bool CAP, bool BIAS, bool SUMS>
__global__ void __launch_bounds__(NQ * 128 + 64, NQ == 1 ? 2 : 1)
attn_forward_tc(const __grid_constant__ b200_tmap map_q, const __grid_constant__ b200_tmap map_k, const __grid_constant__ b200_tmap map_v,
                const __grid_constant__ b200_tmap map_o, const __grid_constant__ AttnArgs a) {
  typedef FwdShape<DP, NQ, KW> Sh;
  extern __shared__ __align__(128) unsigned char dyn[];
  const unsigned int base = (b200_smem_addr(dyn) + 1023u) & ~1023u;
  unsigned char* const gen = dyn + (base - b200_smem_addr(dyn));
  const unsigned int q_at = base, k_at = base + NQ * Sh::kTile, v_at = k_at + Sh::kSlots * Sh::kKeys;
  unsigned long long* bars = (unsigned long long*)(gen + Sh::kBytes);
  const unsigned int bar0 = b200_smem_addr(bars);
  const unsigned int bar_q = bar0, bar_kf = bar0 + 8, bar_ke = bar0 + 40, bar_vf = bar0 + 72, bar_ve = bar0 + 104;   // four slots each but bar_q
  const unsigned int bar_s = bar0 + 136, bar_p = bar0 + 168, bar_o = bar0 + 200, bar_f = bar0 + 216;      // a query tile each; bar_s, bar_p: two places each
  volatile unsigned int* tmem_slot = (volatile unsigned int*)(bars + 29);
  volatile unsigned int* abort_flag = tmem_slot + 1;
  AttnSpan* spans = (AttnSpan*)(bars + 32);           // [2], 16 bytes each
  unsigned char* classes = (unsigned char*)(gen + Sh::kBytes + 512);

  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const unsigned int kLoad = NQ * 4, kMma = NQ * 4 + 1;
  // this CTA's queries: the last ones first, which under a causal mask see the most keys
  const unsigned int tiles_q = (a.S + 128 * NQ - 1) / (128 * NQ), from_last = a.all_heads.of(blockIdx.x);
  const int r0 = (int)(tiles_q - 1 - from_last) * 128 * NQ;
  const unsigned int bh = blockIdx.x - from_last * a.all_heads.d;
  const int b = (int)a.heads.of(bh), h = (int)bh - b * a.H, hk = (int)a.per_key_head.of((unsigned int)h);
  const bool docs = a.kdoc != nullptr;

  auto load_keys = [&](int t, unsigned int slot) {
    b200_mbar_expect_tx(bar_kf + 8 * slot, Sh::kKeys);
#pragma unroll
    for (int p = 0; p < Sh::kPanels; ++p) b200_tma_load_4d(k_at + slot * Sh::kKeys + p * Sh::kPanel, &map_k, bar_kf + 8 * slot, p * 64, t * KW, hk, b);
  };
  auto load_values = [&](int t, unsigned int slot) {
    b200_mbar_expect_tx(bar_vf + 8 * slot, Sh::kKeys);
#pragma unroll
    for (int p = 0; p < Sh::kPanels; ++p) b200_tma_load_4d(v_at + slot * Sh::kKeys + p * Sh::kPanel, &map_v, bar_vf + 8 * slot, p * 64, t * KW, hk, b);
  };
  // (a barrier a lane: one thread would take some 600 cycles for all of them, ahead of the first copies)
  if (warp == kLoad) {
    constexpr unsigned int kBarriers = 29, kFirstP = 21, kLastP = 24;
    if (lane < kBarriers) b200_mbar_init(bar0 + 8 * lane, lane >= kFirstP && lane <= kLastP ? 128 : 1);
    if (lane < 2) {
      spans[lane].last_min = spans[lane].doc_min = 0x7fffffff;
      spans[lane].last_max = -1;
      spans[lane].doc_max = -0x7fffffff - 1;
    }
    if (lane == 2) *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(b200_smem_addr((const void*)tmem_slot)), "r"(Sh::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tmem_taken();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const AttnSeq seq = attn_seq(a, b);
  AttnSpan span[NQ];
  int n_tiles = 0;
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    span[i] = plain_span(a, seq, r0 + 128 * i, 128);
    n_tiles = max(n_tiles, (span[i].last_max + KW) / KW);
  }
  // the queries, and without documents the first keys and values, are on their way from here
  if (threadIdx.x == kLoad * 32) {
    b200_mbar_expect_tx(bar_q, NQ * Sh::kTile);
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int p = 0; p < Sh::kPanels; ++p) b200_tma_load_4d(q_at + i * Sh::kTile + p * kTileBytes64, &map_q, bar_q, p * 64, r0 + 128 * i, h, b);
    if (!docs && n_tiles) {
      load_keys(0, 0);
      load_values(0, 0);
    }
  }
  const unsigned int g = warp >> 2;                        // query tile of a softmax warp
  const int r = r0 + (int)threadIdx.x;                     // row of a softmax thread
  AttnRow row;
  row.pos = 0; row.last = -1; row.doc = 0;
  if (warp < kLoad && r < a.S) row = attn_row(a, b, r);
  tc_before();
  __syncthreads();
  tc_after();
  if (docs) {
    if (warp < kLoad) {
      const AttnSpan s = span_of(r < a.S, row);
      if (lane == 0) {
        atomicMin(&spans[g].last_min, s.last_min);
        atomicMax(&spans[g].last_max, s.last_max);
        atomicMin(&spans[g].doc_min, s.doc_min);
        atomicMax(&spans[g].doc_max, s.doc_max);
      }
    }
    __syncthreads();
    n_tiles = 0;
#pragma unroll
    for (int i = 0; i < NQ; ++i) n_tiles = max(n_tiles, (spans[i].last_max + KW) / KW);
    constexpr int kWarps = Sh::kThreads / 32, kAhead = 4;
    for (int t0 = (int)warp; t0 < n_tiles; t0 += kAhead * kWarps) {
      int kmin[kAhead], kmax[kAhead];
      bool negative[kAhead];
      key_documents<KW, kAhead>(a, b, t0, kWarps, lane, kmin, kmax, negative);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int t = t0 + n * kWarps;
        unsigned int c = 0;
#pragma unroll
        for (int i = 0; i < NQ; ++i) c |= tile_class(spans[i], t * KW, KW, true, kmin[n], kmax[n], negative[n]) << (2 * i);
        if (lane == 0 && t < n_tiles) classes[t] = (unsigned char)c;
      }
    }
    __syncthreads();
  }
  // what query tile i sees of key tile t; what any does
  auto class_of = [&](int t, int i) { return docs ? (classes[t] >> (2 * i)) & 3u : tile_class(span[i], t * KW, KW, false, 0, 0, false); };
  auto seen_at = [&](int t) { return !docs || classes[t] != 0; };      // (without documents every tile up to the last one)
  const unsigned int tmem = *tmem_slot;
  const unsigned int acc_o = tmem + NQ * 128;              // output accumulators behind the scores

  if (warp == kLoad) {
    if (lane == 0) {
      unsigned int n = 0;
      bool live = true;
      for (int t = 0; t < n_tiles && live; ++t) {
        if (!seen_at(t)) continue;
        const unsigned int slot = n % Sh::kSlots, use = n / Sh::kSlots;
        if (docs || n) {
          if (use) live = b200_wait(bar_ke + 8 * slot, (use - 1) & 1u, abort_flag, a.status, 21u);
          if (!live) break;
          load_keys(t, slot);
          if (use) live = b200_wait(bar_ve + 8 * slot, (use - 1) & 1u, abort_flag, a.status, 22u);
          if (!live) break;
          load_values(t, slot);
        }
        ++n;
      }
      // the copies under way land before shared memory is given up, whatever happened to the others
      if (*abort_flag) {
        for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bar_q, 0u); ++tries) {}
        for (unsigned int i = 0; i < Sh::kSlots && i < n; ++i) {
          const unsigned int last = (n - 1 - i) / Sh::kSlots, slot = (n - 1 - i) % Sh::kSlots;
          for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bar_kf + 8 * slot, last & 1u); ++tries) {}
          for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bar_vf + 8 * slot, last & 1u); ++tries) {}
        }
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    if (b200_elect()) {
      constexpr unsigned int idesc_s = idesc_of<T>(128, KW, false, false), idesc_o = idesc_of<T>(128, DP, false, true);
      bool live = b200_wait(bar_q, 0u, abort_flag, a.status, 23u);
      unsigned int scored[NQ], done[NQ];         // tiles whose scores are queued, whose weights have been multiplied
      int last[NQ];                              // the last tile of keys that a query tile sees: its product is awaited
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        scored[i] = done[i] = 0;
        for (last[i] = n_tiles - 1; last[i] >= 0 && !class_of(last[i], i); --last[i]) {}
      }
      auto scores = [&](int i, unsigned int slot) {
        const unsigned int place = scored[i]++ % Sh::kScores;
#pragma unroll
        for (int p = 0; p < Sh::kPanels; ++p) {
          const unsigned long long dq = b200_smem_desc(q_at + i * Sh::kTile + p * kTileBytes64, 16u, 1024u);
          const unsigned long long dk = b200_smem_desc(k_at + slot * Sh::kKeys + p * Sh::kPanel, 16u, 1024u);
#pragma unroll
          for (unsigned int ks = 0; ks < 4; ++ks) b200_umma(tmem + i * 128 + place * KW, dq + ks * 2, dk + ks * 2, idesc_s, (p || ks) ? 1u : 0u);
        }
        b200_umma_commit(bar_s + 16 * i + 8 * place);
      };
      int t = 0, next = 0;
      unsigned int n = 0;
      while (next < n_tiles && !seen_at(next)) ++next;
      if (live && next < n_tiles) {
        live = b200_wait(bar_kf, 0u, abort_flag, a.status, 24u);
        tc_after();
        if (live) {
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (class_of(next, i)) scores(i, 0);
          b200_umma_commit(bar_ke);
        }
      }
      while (live && next < n_tiles) {
        t = next;
        for (++next; next < n_tiles && !seen_at(next); ++next) {}
        const unsigned int slot = n % Sh::kSlots, ph = (n / Sh::kSlots) & 1u, slot1 = (n + 1) % Sh::kSlots, ph1 = ((n + 1) / Sh::kSlots) & 1u;
        if (next < n_tiles) live = b200_wait(bar_kf + 8 * slot1, ph1, abort_flag, a.status, 26u);
        if (!live) break;
        tc_after();
        // With two places the next tile's scores go ahead of this one's products (their place was given up with the weights before);
        // with one they follow them, query tile by query tile.
        if (Sh::kScores == 2 && next < n_tiles) {
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (class_of(next, i)) scores(i, slot1);
          b200_umma_commit(bar_ke + 8 * slot1);
        }
        live = b200_wait(bar_vf + 8 * slot, ph, abort_flag, a.status, 25u);
        tc_after();
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          if (!live) break;
          if (class_of(t, i)) {
            live = b200_wait(bar_p + 16 * i + 8 * (done[i] % Sh::kScores), done[i] / Sh::kScores & 1u, abort_flag, a.status, 27u);
            tc_after();
            if (!live) break;
            const unsigned int weights = tmem + i * 128 + done[i] % Sh::kScores * KW;
            const unsigned long long dv = b200_smem_desc(v_at + slot * Sh::kKeys, Sh::kPanel, 1024u);
#pragma unroll
            for (unsigned int ks = 0; ks < KW / 16; ++ks) umma_ts(acc_o + i * DP, weights + ks * 8, dv + ks * 128, idesc_o, (done[i] || ks) ? 1u : 0u);
            // the last product has a barrier of its own: the others' may be two phases behind when it is waited for
            if (t == last[i]) b200_umma_commit(bar_f + 8 * i);
            else if (Sh::kScores == 2) b200_umma_commit(bar_o + 8 * i);
            ++done[i];
          }
          if (i == NQ - 1) b200_umma_commit(bar_ve + 8 * slot);
          if (Sh::kScores == 1 && next < n_tiles && class_of(next, i)) scores(i, slot1);
        }
        if (!live) break;
        if (Sh::kScores == 1 && next < n_tiles) b200_umma_commit(bar_ke + 8 * slot1);
        ++n;
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax: a thread a row
    const unsigned int mine = tmem + g * 128 + ((warp & 3u) << 21), mine_o = acc_o + g * DP + ((warp & 3u) << 21);
    const float c = CAP ? a.cap * kLog2e : a.scale * kLog2e;
    const float to_tanh = CAP ? a.over : 0.f;
    const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;
    const AttnSpan mine_span = NQ == 2 && g == 1u ? span[NQ - 1] : span[0];
    float m = -INFINITY, l = 0.f;      // m: in log 2 units without bias or cap scaled by c, see `unit`
    const float unit = BIAS ? 1.f : c;
    unsigned int seen = 0;
    bool live = true;
    // the sums in memory: the maximum that they are relative to, and what they have to be multiplied by
    constexpr unsigned int kSumTiles = kSumKeys / KW;
    [[maybe_unused]] float m_sum = -INFINITY;
    [[maybe_unused]] auto sums_at = [&](int e) { return (float4*)(a.sums + (((long long)b * a.H + h) * a.S + r) * DP + e); };
    [[maybe_unused]] auto since = [&]() { return m_sum == m ? 1.f : m_sum == -INFINITY ? 0.f : ex2(m_sum - m); };
    for (int t = 0; t < n_tiles && live; ++t) {
      const unsigned int cls = docs ? (classes[t] >> (2 * g)) & 3u : tile_class(mine_span, t * KW, KW, false, 0, 0, false);
      if (!cls) continue;
      const unsigned int place = seen % Sh::kScores, at = mine + place * KW;
      unsigned int bits[KW / 32];
      if (cls == 2u) visible_words<KW / 32>(a, b, t * KW, row, lane, bits);     // (its loads pass while the scores are formed)
      live = b200_wait(bar_s + 16 * g + 8 * place, seen / Sh::kScores & 1u, abort_flag, a.status, 28u);
      if (!live) break;
      tc_after();
      // first pass: the row's maximum, 32 scores at a time; what cap, bias or mask have changed goes back
      float x[2][32], top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      b200_tmem_ld32(at, (unsigned int*)x[0]);
#pragma unroll
      for (int k = 0; k < KW / 32; ++k) {
        float* y = x[k & 1];
        tmem_wait_ld();
        if (k < KW / 32 - 1) b200_tmem_ld32(at + 32 * (k + 1), (unsigned int*)x[(k + 1) & 1]);
        if constexpr (CAP) tanh_chunk(x[k & 1], to_tanh);
        if constexpr (BIAS) {
          const float from = (float)(row.pos - t * KW - 32 * k);
#pragma unroll
          for (int j = 0; j < 32; ++j) y[j] = fmaf(-slope2, fabsf(from - (float)j), y[j] * c);
        }
        if (cls == 2u) {
#pragma unroll
          for (int j = 0; j < 32; ++j) y[j] = (bits[k] >> j) & 1u ? y[j] : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], y[j]);
        if (CAP || BIAS || cls == 2u) b200_tmem_st32(at + 32 * k, (const unsigned int*)y);
      }
      if (CAP || BIAS || cls == 2u) tmem_wait_st();
      b200_tmem_ld32(at, (unsigned int*)x[0]);
      const float m_tile = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * unit;
      if constexpr (SUMS)
        if (seen && seen % kSumTiles == 0) {
          // (the product before is waited for as below)
          if (Sh::kScores == 2) {
            live = b200_wait(bar_o + 8 * g, (seen - 1) & 1u, abort_flag, a.status, 49u);
            tc_after();
          }
          const float by = since();
#pragma unroll
          for (int e = 0; e < DP; e += 32) {
            float o[32];
            b200_tmem_ld32(mine_o + e, (unsigned int*)o);
            tmem_wait_ld();
            if (r < a.S)
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                float4* to = sums_at(e + j);
                const float4 w = seen > kSumTiles && by != 0.f ? *to : make_float4(0.f, 0.f, 0.f, 0.f);
                *to = make_float4(fmaf(w.x, by, o[j]), fmaf(w.y, by, o[j + 1]), fmaf(w.z, by, o[j + 2]), fmaf(w.w, by, o[j + 3]));
              }
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0.f;
            b200_tmem_st32(mine_o + e, (unsigned int*)o);
          }
          m_sum = m;
        }
      // the maximum in use moves when some row of the warp has outgrown it (or has had none)
      if (__any_sync(0xffffffffu, m_tile > m + 8.f || (m == -INFINITY && m_tile != -INFINITY))) {
        const float m_new = fmaxf(m, m_tile);
        const float by = m == -INFINITY ? 0.f : ex2(m - m_new);
        if (seen) {
          // (with one place the scores came behind the product before; with two it may still run, but not the one before it, which the
          // scores came behind: the barrier is in this phase or past it)
          if (Sh::kScores == 2) {
            live = b200_wait(bar_o + 8 * g, (seen - 1) & 1u, abort_flag, a.status, 30u);
            tc_after();
          }
#pragma unroll
          for (int e = 0; e < DP; e += 32) {
            float o[32];
            b200_tmem_ld32(mine_o + e, (unsigned int*)o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = by == 0.f ? 0.f : o[j] * by;
            b200_tmem_st32(mine_o + e, (unsigned int*)o);
          }
        }
        l *= by;
        m = m_new;
      }
      const float off = m == -INFINITY ? 0.f : kLift<T> - m;
      Pair part[2] = {Pair(0.f, 0.f), Pair(0.f, 0.f)};
      const Pair unit2(unit, unit), off2(off, off);
      // second pass: the weights, over the scores that have been read
#pragma unroll
      for (int k = 0; k < KW / 32; ++k) {
        const float* y = x[k & 1];
        tmem_wait_ld();
        if (k < KW / 32 - 1) b200_tmem_ld32(at + 32 * (k + 1), (unsigned int*)x[(k + 1) & 1]);
        unsigned int w[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float p0, p1;
          fma2(Pair(y[j], y[j + 1]), unit2, off2).get(p0, p1);
          p0 = ex2(p0);
          p1 = ex2(p1);
          part[j >> 1 & 1] = add2(part[j >> 1 & 1], Pair(p0, p1));
          w[j / 2] = pack2(p0, p1, T());
        }
        tmem_st16(at + 16 * k, w);
      }
      float l0, l1;
      add2(part[0], part[1]).get(l0, l1);
      l += l0 + l1;
      tmem_wait_st();
      tc_before();
      // (a barrier a place: with two of them a warp may be a tile ahead of another)
      b200_mbar_arrive(bar_p + 16 * g + 8 * place);
      ++seen;
    }
    // ---------------------------------------------------------------- output
    // (the output goes through the queries' tile, which has to have arrived even where nobody reads it)
    if (live) live = b200_wait(seen ? bar_f + 8 * g : bar_q, 0u, abort_flag, a.status, 29u);
    tc_after();
    const float by = l > 0.f || l != l ? 1.f / l : 0.f;
    // (of scores beyond 2^23 the product with `unit`, which is not rounded, and the maximum, which is, may lie far apart: such rows are done again)
    float bad = !BIAS && fabsf(m) > 8388608.f && seen && m != -INFINITY ? 1.f : 0.f;
    unsigned char* tile = gen + g * Sh::kTile;     // the queries' tile: its last product is done
    const unsigned int in = (warp & 3u) * 32 + lane;
#pragma unroll
    for (int e = 0; e < DP; e += 32) {
      float o[32];
      if (live && seen) {
        b200_tmem_ld32(mine_o + e, (unsigned int*)o);
        tmem_wait_ld();
      }
      if constexpr (SUMS)
        if (seen > kSumTiles && r < a.S) {
          const float before = since();
          if (before != 0.f)
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 w = *sums_at(e + j);
              o[j] = fmaf(w.x, before, o[j]);
              o[j + 1] = fmaf(w.y, before, o[j + 1]);
              o[j + 2] = fmaf(w.z, before, o[j + 2]);
              o[j + 3] = fmaf(w.w, before, o[j + 3]);
            }
        }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        o[j] = by == 0.f ? 0.f : o[j] * by;
        bad = fmaf(o[j], 0.f, bad);
      }
      unsigned char* line = tile + (e >> 6) * kTileBytes64 + in * 128;
      const unsigned int piece0 = (e & 63) >> 3;
#pragma unroll
      for (int p = 0; p < 4; ++p)
        *(uint4*)(line + (((piece0 + p) ^ (in & 7u)) << 4)) =
            make_uint4(pack2(o[8 * p], o[8 * p + 1], T()), pack2(o[8 * p + 2], o[8 * p + 3], T()), pack2(o[8 * p + 4], o[8 * p + 5], T()), pack2(o[8 * p + 6], o[8 * p + 7], T()));
    }
    if (live && r < a.S && a.lse) a.lse[((long long)b * a.H + h) * a.S + r] = l > 0.f || l != l ? (m - kLift<T> + log2f(l)) * kLn2 : -INFINITY;
    // every warp sends its 32 rows; those with a value that is infinite or undefined are done again, one by one
    const int first = r0 + (int)warp * 32;
    const unsigned int mend = __ballot_sync(0xffffffffu, live && r < a.S && bad != 0.f);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0 && live && first < a.S) {
#pragma unroll
      for (int p = 0; p < Sh::kPanels; ++p)
        if (p * 64 < a.D) b200_tma_store_4d(&map_o, b200_smem_addr(tile) + p * kTileBytes64 + (warp & 3u) * 4096, p * 64, first, h, b);
      if (mend) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      else b200_tma_store_read_wait<0>();
    }
    __syncwarp();
    for (unsigned int todo = mend; todo; todo &= todo - 1) attn_forward_row<T>(a, b, h, first + __ffs(todo) - 1, lane);
  }
  // ------------------------------------------------------------------ teardown
  __syncwarp();
  if (*abort_flag) {
    const unsigned long long t0 = b200_now_ns();
    while (b200_now_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_before();
  __syncthreads();
  if (warp == kMma) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::kColumns) : "memory");
  }
}

}  // namespace b200
#endif
