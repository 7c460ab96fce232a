// The gradients of attention for 16-bit heads on the tensor cores.
//
// Two kinds of CTAs in one launch, each of which owns its outputs and adds to them in a fixed order (no atomic additions: the same bits every time), at
// the price of forming the scores and their gradients twice: seven products a pair of tiles instead of five.  (As two launches
// few rows left most SMs idle twice.)
//
//   keys     a CTA has 128 keys of one key head and walks the tiles of 128 queries that see them, of all query heads it
//            serves.  s^T = k q^T and dp^T = v do^T have a thread per key; p^T and ds^T go back to tensor memory in 16 bits, as the
//            A operand of dv += p^T do and dk += ds^T q.
//   queries  a CTA has 128 queries of one head and walks the tiles of keys they see: s = q k^T, dp = do v^T, dq += ds k.
//
// A thread does 64 columns of a row; half score gradients are scaled, see unit_of; one warp copies, one issues the products.  Weights are formed while the second product runs, the
// score gradients while the next tile's scores are.  Heads of more than 64 elements take tiles of 128 columns, two threads a row, and
// all of tensor memory; those of up to 64 tiles of 64 columns, a thread a row, and half of it, so that two CTAs share an SM (short
// sequences are bound by the chain from a CTA's start to its end).  Copies start before anything else.
#ifndef B200_ATTN_BWD_SM100_CUH
#define B200_ATTN_BWD_SM100_CUH
#include "attn_fwd_sm100.cuh"

namespace b200 {

// CW: columns of a tile, that is queries (or keys) of one step; 64 a thread.
template <int DP, int CW>
struct BwdShape {
  static constexpr int kPanels = DP / 64, kGroups = CW / 64;                 // groups of four warps
  static constexpr unsigned int kTile = kPanels * kTileBytes64;              // the CTA's own rows
  static constexpr unsigned int kPanel = CW * 128, kStep = kPanels * kPanel; // a tile of the others
  static constexpr unsigned int kThreads = kGroups * 128 + 64, kWarps = kThreads / 32;
  static constexpr unsigned int kStage = 2 * kStep + 1024;                   // two tiles, and the queries' statistics (8 bytes each)
  static constexpr unsigned int kBytes = 2 * kTile + 2 * kStage;
  static constexpr unsigned int kColumns = 2 * CW + 2 * DP <= 256 && 3 * CW + DP <= 256 ? 256 : 512;
  static constexpr size_t smem(int tiles) { return 1024 + kBytes + 256 + (size_t)tiles; }
};

// Half gradients of scores are multiplied by a power of two before they are rounded, a row's own: ds = p <d_out, v - out> is at most
// |d_out| |v| + |d_out| |out|, and the power brings that bound between 2^13 and 2^14.  A query's row has its own |d_out| and the largest
// |v| that its tile of queries sees; a key's its own |v| and the largest |d_out| and |d_out| |out| of the tiles that see it.  So p may be 2^-20 before the first
// bits are lost, whatever the sizes of d_out and v, and other rows, heads and sequences have no say in it.
// (One power for the whole call, of the largest |d_out|, left 3 % of a gradient wrong beside a row 10^4 times as large.)
__device__ __forceinline__ float unit_of(float bound) {
  return bound > 0.f && bound < INFINITY ? exp2f(fminf(fmaxf(floorf(14.f - log2f(bound)), -60.f), 60.f)) : 1.f;
}
// the largest of each of N values of the softmax threads; `sh`: N floats a warp, used once
template <int WARPS, int N>
__device__ __forceinline__ void largest(float (&v)[N], float* sh) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] = fmaxf(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
    if ((threadIdx.x & 31u) == 0) sh[n * WARPS + (threadIdx.x >> 5)] = v[n];
  }
  named_barrier(5, WARPS * 32);
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < WARPS; ++i) v[n] = fmaxf(v[n], sh[n * WARPS + i]);
}

__device__ __forceinline__ void bulk_load(unsigned int dst, const void* src, unsigned int bytes, unsigned int bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Which of the 64 queries from r0 see key j, a bit each (bits of queries behind the last one are of no account: their weights are zero).
// Without documents a key is seen from one query on.
__device__ __forceinline__ void visible_queries(const AttnArgs& a, const AttnSeq& seq, int b, int r0, int j, unsigned int lane, unsigned int (&bits)[2]) {
  int first = 0;
  if (j >= seq.len) first = 0x7fffffff;
  else if (a.mask == B200_MASK_CAUSAL || (a.mask == B200_MASK_PREFIX && j >= seq.prefix)) first = max(0, j - (seq.len - a.S));
  int doc = 0;
  if (a.kdoc) {
    doc = j < a.T ? a.kdoc[(long long)b * a.T + j] : -1;
    if (doc < 0) first = 0x7fffffff;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = first - (r0 + 32 * i);     // queries of this word before the first
    bits[i] = n <= 0 ? 0xffffffffu : n >= 32 ? 0u : 0xffffffffu << n;
  }
  if (!a.kdoc) return;
  const AttnQueryDocs theirs(a, seq, b);
  int d[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + (int)lane + 32 * i;
    d[i] = r < a.S ? theirs.of(r) : -1;
  }
  unsigned int todo = 0xffffffffu;
  while (todo) {
    const int k = __shfl_sync(0xffffffffu, doc, __ffs(todo) - 1);
    const bool mine = doc == k;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned int same = __ballot_sync(0xffffffffu, d[i] == k);
      if (mine) bits[i] &= same;
    }
    todo &= ~__ballot_sync(0xffffffffu, mine);
  }
}

// 32 accumulator columns of a row into the swizzled 16-bit tile that leaves by TMA; false where a value is infinite or undefined
template <class T>
__device__ __forceinline__ bool store_columns(unsigned char* tile, unsigned int in, int e, const float* o) {
  float bad = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) bad = fmaf(o[j], 0.f, bad);
  unsigned char* line = tile + (e >> 6) * kTileBytes64 + in * 128;
  const unsigned int piece0 = (e & 63) >> 3;
#pragma unroll
  for (int p = 0; p < 4; ++p)
    *(uint4*)(line + (((piece0 + p) ^ (in & 7u)) << 4)) =
        make_uint4(pack2(o[8 * p], o[8 * p + 1], T()), pack2(o[8 * p + 2], o[8 * p + 3], T()), pack2(o[8 * p + 4], o[8 * p + 5], T()), pack2(o[8 * p + 6], o[8 * p + 7], T()));
  return bad == 0.f;
}

// Score of one pair in units of log 2, from tanh(x / cap) or x
template <bool BIAS>
__device__ __forceinline__ float pair_score(float x, float c, float slope2, float far) {
  x *= c;
  if constexpr (BIAS) x = fmaf(-slope2, fabsf(far), x);
  return x;
}

// ------------------------------------------------------------------ keys
template <class T, int DP, int CW, bool CAP, bool BIAS>
__device__ __forceinline__ void attn_grad_keys(const b200_tmap& map_q, const b200_tmap& map_k, const b200_tmap& map_v, const b200_tmap& map_do,
                                               const b200_tmap& map_dk, const b200_tmap& map_dv, const AttnArgs& a, unsigned int block) {
  typedef BwdShape<DP, CW> Sh;
  extern __shared__ __align__(128) unsigned char dyn[];
  const unsigned int base = (b200_smem_addr(dyn) + 1023u) & ~1023u;
  unsigned char* const gen = dyn + (base - b200_smem_addr(dyn));
  const unsigned int k_at = base, v_at = base + Sh::kTile, ring = base + 2 * Sh::kTile;
  unsigned long long* bars = (unsigned long long*)(gen + Sh::kBytes);
  const unsigned int bar0 = b200_smem_addr(bars);
  const unsigned int bar_kv = bar0, bar_full = bar0 + 8, bar_empty = bar0 + 24;      // two each
  const unsigned int bar_s = bar0 + 40, bar_dp = bar0 + 48, bar_p = bar0 + 56, bar_ds = bar0 + 64, bar_done = bar0 + 72;
  volatile unsigned int* tmem_slot = (volatile unsigned int*)(bars + 10);
  volatile unsigned int* abort_flag = tmem_slot + 1;
  float* scratch = (float*)(bars + 12);                   // [16]
  unsigned char* classes = (unsigned char*)(gen + Sh::kBytes + 256);

  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  constexpr unsigned int kLoad = Sh::kWarps - 2, kMma = Sh::kWarps - 1;
  // this CTA's keys: the first ones first, which under a causal mask are seen by the most queries
  // (blocks that share a key tile, each for some of the query heads, lie one behind the other)
  const unsigned int share_of = a.all_key_heads.of(block), bh = block - share_of * a.all_key_heads.d;
  const unsigned int tile_of = a.parts_of.of(share_of);
  const int j0 = (int)tile_of * 128, b = (int)a.key_heads.of(bh), hk = (int)bh - b * a.HK;
  const int part = (int)(share_of - tile_of * a.parts_of.d), first_head = hk * a.group + part * a.part_heads;
  const int tiles = (a.S + CW - 1) / CW, stat_tiles = (a.S + 127) / 128;
  const bool docs = a.kdoc != nullptr;
  if (warp == kLoad) {
    if (lane < 10) b200_mbar_init(bar0 + 8 * lane, lane == 7 || lane == 8 ? Sh::kGroups * 128 : 1);      // (bar_p, bar_ds)
    if (lane == 10) *abort_flag = 0u;
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
  if (threadIdx.x == kLoad * 32) {
    b200_mbar_expect_tx(bar_kv, 2 * Sh::kTile);
#pragma unroll
    for (int p = 0; p < Sh::kPanels; ++p) {
      b200_tma_load_4d(k_at + p * kTileBytes64, &map_k, bar_kv, p * 64, j0, hk, b);
      b200_tma_load_4d(v_at + p * kTileBytes64, &map_v, bar_kv, p * 64, j0, hk, b);
    }
  }
  // queries: a tile of CW; `n`: tiles taken so far
  auto load = [&](int h, int t, unsigned int n) {
    const unsigned int slot = n & 1u, at = ring + slot * Sh::kStage, bar = bar_full + 8 * slot;
    b200_mbar_expect_tx(bar, 2 * Sh::kStep + CW * 8);
#pragma unroll
    for (int p = 0; p < Sh::kPanels; ++p) {
      b200_tma_load_4d(at + p * Sh::kPanel, &map_q, bar, p * 64, t * CW, h, b);
      b200_tma_load_4d(at + Sh::kStep + p * Sh::kPanel, &map_do, bar, p * 64, t * CW, h, b);
    }
    const float* stat = a.stat + (((long long)b * a.H + h) * stat_tiles + t * CW / 128) * 256 + t * CW % 128;
    bulk_load(at + 2 * Sh::kStep, stat, CW * 4, bar);
    bulk_load(at + 2 * Sh::kStep + CW * 4, stat + 128, CW * 4, bar);
  };
  auto class_without = [&](int t) { return tile_class(plain_span(a, seq, t * CW, CW), j0, 128, false, 0, 0, false); };
  int early = -1;             // the tile that is on its way before the others are known
  if (!docs)
    for (early = 0; early < tiles && !class_without(early); ++early) {}
  if (threadIdx.x == kLoad * 32 && early >= 0 && early < tiles) load(first_head, early, 0);
  tc_before();
  __syncthreads();
  tc_after();
  if (docs) {
    int kmin[1], kmax[1];
    bool negative[1];
    key_documents<128, 1>(a, b, j0 / 128, 0, lane, kmin, kmax, negative);
    const AttnQueryDocs theirs(a, seq, b);
    constexpr int kAhead = 4;
    for (int t0 = (int)warp; t0 < tiles; t0 += kAhead * (int)Sh::kWarps) {
      int d[kAhead][CW / 32];
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
#pragma unroll
        for (int i = 0; i < CW / 32; ++i) {
          const long long r = (long long)(t0 + n * (int)Sh::kWarps) * CW + 32 * i + lane;
          d[n][i] = r < a.S ? theirs.of((int)r) : -1;
        }
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int t = t0 + n * (int)Sh::kWarps;
        AttnSpan s;
        s.last_min = s.doc_min = 0x7fffffff;
        s.last_max = -1;
        s.doc_max = -0x7fffffff - 1;
#pragma unroll
        for (int i = 0; i < CW / 32; ++i) {
          const int r = t * CW + 32 * i + (int)lane;
          AttnRow w;
          w.doc = d[n][i];
          w.last = w.doc < 0 ? -1 : attn_last(a, seq, r);
          const AttnSpan p = span_of(t < tiles && r < a.S, w);
          s.last_min = min(s.last_min, p.last_min);
          s.last_max = max(s.last_max, p.last_max);
          s.doc_min = min(s.doc_min, p.doc_min);
          s.doc_max = max(s.doc_max, p.doc_max);
        }
        if (lane == 0 && t < tiles) classes[t] = (unsigned char)tile_class(s, j0, 128, true, kmin[0], kmax[0], negative[0]);
      }
    }
    __syncthreads();
  }
  auto class_of = [&](int t) { return docs ? (unsigned int)classes[t] : class_without(t); };
  const int begin = docs ? 0 : early;       // (without documents the tiles that see the keys are the last ones)
  const unsigned int tmem = *tmem_slot;
  const unsigned int t_s = tmem, t_dp = tmem + CW, t_dv = tmem + 2 * CW, t_dk = tmem + 2 * CW + DP;

  if (warp == kLoad) {
    if (lane == 0) {
      unsigned int n = 0;
      bool live = true;
      for (int h = first_head; h < first_head + a.part_heads && live; ++h)
        for (int t = begin; t < tiles; ++t) {
          if (!class_of(t)) continue;
          if (docs || n) {
            if (n > 1) live = b200_wait(bar_empty + 8 * (n & 1u), ((n >> 1) - 1) & 1u, abort_flag, a.status, 31u);
            if (!live) break;
            load(h, t, n);
          }
          ++n;
        }
      // the copies under way land before shared memory is given up, whatever happened to the others
      if (*abort_flag) {
        for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bar_kv, 0u); ++tries) {}
        for (unsigned int i = 0; i < 2 && i < n; ++i)
          for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bar_full + 8 * ((n - 1 - i) & 1u), ((n - 1 - i) >> 1) & 1u); ++tries) {}
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    if (b200_elect()) {
      constexpr unsigned int idesc_s = idesc_of<T>(128, CW, false, false), idesc_g = idesc_of<T>(128, DP, false, true);
      // 128 x CW of two k-major tiles
      auto square = [&](unsigned int d, unsigned int x, unsigned int y) {
#pragma unroll
        for (int p = 0; p < Sh::kPanels; ++p) {
          const unsigned long long dx = b200_smem_desc(x + p * kTileBytes64, 16u, 1024u), dy = b200_smem_desc(y + p * Sh::kPanel, 16u, 1024u);
#pragma unroll
          for (unsigned int ks = 0; ks < 4; ++ks) b200_umma(d, dx + ks * 2, dy + ks * 2, idesc_s, (p || ks) ? 1u : 0u);
        }
      };
      // += (16-bit rows in tensor memory, 64 columns of the tile in each 64) x (tile read along its rows)
      auto product = [&](unsigned int d, unsigned int x, unsigned int y, bool add) {
        const unsigned long long dy = b200_smem_desc(y, Sh::kPanel, 1024u);
#pragma unroll
        for (unsigned int ks = 0; ks < CW / 16; ++ks) umma_ts(d, x + (ks >> 2) * 64 + (ks & 3u) * 8, dy + ks * 128, idesc_g, (add || ks) ? 1u : 0u);
      };
      int total = 0;
      for (int t = begin; t < tiles; ++t) total += class_of(t) != 0;
      total *= a.part_heads;
      bool live = b200_wait(bar_kv, 0u, abort_flag, a.status, 32u);
      if (live && total) {
        live = b200_wait(bar_full, 0u, abort_flag, a.status, 33u);
        tc_after();
        if (live) {
          square(t_s, k_at, ring);
          b200_umma_commit(bar_s);
          square(t_dp, v_at, ring + Sh::kStep);
          b200_umma_commit(bar_dp);
        }
      }
      for (int n = 0; live && n < total; ++n) {
        const unsigned int at = ring + (n & 1) * Sh::kStage, next = ring + ((n + 1) & 1) * Sh::kStage;
        live = b200_wait(bar_p, n & 1, abort_flag, a.status, 34u);
        if (!live) break;
        tc_after();
        product(t_dv, t_s, at + Sh::kStep, n != 0);
        if (n + 1 < total) {
          live = b200_wait(bar_full + 8 * ((n + 1) & 1), ((n + 1) >> 1) & 1, abort_flag, a.status, 35u);
          if (!live) break;
          tc_after();
          square(t_s, k_at, next);
          b200_umma_commit(bar_s);
        }
        live = b200_wait(bar_ds, n & 1, abort_flag, a.status, 36u);
        if (!live) break;
        tc_after();
        product(t_dk, t_dp, at, n != 0);
        b200_umma_commit(bar_empty + 8 * (n & 1));
        if (n + 1 < total) {
          square(t_dp, v_at, next + Sh::kStep);
          b200_umma_commit(bar_dp);
        } else {
          b200_umma_commit(bar_done);
        }
      }
    }
    __syncwarp();
  } else {
    const unsigned int half = warp >> 2, in = (warp & 3u) * 32 + lane, lanes = (warp & 3u) << 21;
    const unsigned int my_s = t_s + 64 * half + lanes, my_dp = t_dp + 64 * half + lanes;
    const float c = CAP ? a.cap * kLog2e : a.scale * kLog2e, to_tanh = CAP ? a.over : 0.f;
    const int j = j0 + (int)in;
    float grad_unit = 1.f;
    if constexpr (std::is_same<T, __half>::value) {
      float most[2] = {0.f, 0.f};
      for (int h = first_head; h < first_head + a.part_heads; ++h) {
        const float2* sizes = a.row_sizes + ((long long)b * a.H + h) * stat_tiles * 128;
#pragma unroll 8
        for (int r = begin * CW + (int)threadIdx.x; r < tiles * CW; r += Sh::kGroups * 128)
          if (!docs || classes[r / CW]) {
            const float2 s = sizes[r];
            most[0] = fmaxf(most[0], s.x);
            most[1] = fmaxf(most[1], s.y);
          }
      }
      const float of_v = j < a.T ? a.value_sizes[((long long)b * a.T + j) * a.HK + hk] : 0.f;
      largest<Sh::kGroups * 4>(most, scratch);
      grad_unit = unit_of(fmaf(most[0], of_v, most[1]));
    }
    const float to_unit = grad_unit * kWeightBack<T>;
    unsigned int n = 0;
    bool live = true;
    for (int h = first_head; h < first_head + a.part_heads && live; ++h) {
      const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;
      for (int t = begin; t < tiles; ++t) {
        const unsigned int cls = class_of(t);
        if (!cls) continue;
        const float* stat = (const float*)(gen + 2 * Sh::kTile + (n & 1u) * Sh::kStage + 2 * Sh::kStep) + 64 * half;
        unsigned int bits[2] = {0xffffffffu, 0xffffffffu};
        const int r0 = t * CW + 64 * (int)half;
        if (cls == 2u) visible_queries(a, seq, b, r0, j, lane, bits);
        live = b200_wait(bar_full + 8 * (n & 1u), (n >> 1) & 1u, abort_flag, a.status, 37u) && b200_wait(bar_s, n & 1u, abort_flag, a.status, 38u);
        if (!live) break;
        tc_after();
        float w[64];            // weights, times 1 - tanh^2 with a cap
        // (two forms: the mask costs three instructions an element)
        auto weights = [&](auto masked) {
          constexpr bool M = decltype(masked)::value;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x[32];
            unsigned int u[16];
            b200_tmem_ld32(my_s + 32 * k, (unsigned int*)x);
            [[maybe_unused]] const float far = BIAS ? (float)(seq.len - a.S + r0 + 32 * k - j) : 0.f;
            tmem_wait_ld();
            if constexpr (CAP) tanh_chunk(x, to_tanh);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 l = *(const float4*)(stat + 32 * k + i);
              const float lse2[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float p;
                if constexpr (!BIAS) p = ex2(fmaf(x[i + q], c, -lse2[q]));
                else p = ex2(pair_score<BIAS>(x[i + q], c, slope2, far + (float)(i + q)) - lse2[q]);
                if constexpr (M) p = (bits[k] >> (i + q)) & 1u ? p : 0.f;
                w[32 * k + i + q] = CAP ? p * fmaf(-x[i + q], x[i + q], 1.f) : p;
                x[i + q] = p;
              }
              u[i / 2] = pack2(x[i], x[i + 1], T());
              u[i / 2 + 1] = pack2(x[i + 2], x[i + 3], T());
            }
            tmem_st16(my_s + 16 * k, u);
          }
        };
        if (cls == 2u) weights(std::true_type());
        else weights(std::false_type());
        tmem_wait_st();
        tc_before();
        b200_mbar_arrive(bar_p);
        live = b200_wait(bar_dp, n & 1u, abort_flag, a.status, 39u);
        if (!live) break;
        tc_after();
        auto gradients = [&](auto masked) {
          constexpr bool M = decltype(masked)::value;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x[32];
            unsigned int u[16];
            b200_tmem_ld32(my_dp + 32 * k, (unsigned int*)x);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 l = *(const float4*)(stat + CW + 32 * k + i);
              const float delta[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float ds = w[32 * k + i + q] * (x[i + q] - delta[q]);
                if constexpr (std::is_same<T, __half>::value) ds *= to_unit;
                if constexpr (M) ds = (bits[k] >> (i + q)) & 1u ? ds : 0.f;
                x[i + q] = ds;
              }
              u[i / 2] = pack2(x[i], x[i + 1], T());
              u[i / 2 + 1] = pack2(x[i + 2], x[i + 3], T());
            }
            tmem_st16(my_dp + 16 * k, u);
          }
        };
        if (cls == 2u) gradients(std::true_type());
        else gradients(std::false_type());
        tmem_wait_st();
        tc_before();
        b200_mbar_arrive(bar_ds);
        ++n;
      }
    }
    // ---- dv and dk, 32 rows a warp, through the tiles of v and k: by the first four warps and the others, or one after the other
    if (live) live = b200_wait(n ? bar_done : bar_kv, 0u, abort_flag, a.status, 40u);
    tc_after();
    const int first = j0 + (int)(warp & 3u) * 32;
    unsigned int mend[2] = {0u, 0u};           // rows of dv, of dk that are to be done again
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (Sh::kGroups == 2 && which != (int)half) continue;
      const unsigned int from = (which ? t_dk : t_dv) + lanes;
      unsigned char* tile = gen + (which ? 0 : Sh::kTile);
      const float by = which ? a.scale / grad_unit : kWeightBack<T>;
      bool fine = true;
#pragma unroll
      for (int e = 0; e < DP; e += 32) {
        float o[32];
        if (live && n) {
          b200_tmem_ld32(from + e, (unsigned int*)o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = n ? o[i] * by : 0.f;
        if (a.n_parts > 1) {         // joined with the other blocks' by a kernel of its own
          float* to = a.parts + ((((long long)(2 * part + 1 - which) * a.B + b) * a.T + j) * a.HK + hk) * DP + e;
          if (live && j < a.T)
#pragma unroll
            for (int i = 0; i < 32; i += 4) *(float4*)(to + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else {
          fine &= store_columns<T>(tile, in, e, o);
        }
      }
      if (a.n_parts > 1) continue;
      mend[which] = __ballot_sync(0xffffffffu, live && j < a.T && !fine);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0 && live && first < a.T) {
#pragma unroll
        for (int p = 0; p < Sh::kPanels; ++p)
          if (p * 64 < a.D) b200_tma_store_4d(which ? &map_dk : &map_dv, b200_smem_addr(tile) + p * kTileBytes64 + (warp & 3u) * 4096, p * 64, first, hk, b);
      }
    }
    if (lane == 0 && live) {
      if (mend[0] | mend[1]) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      else b200_tma_store_read_wait<0>();
    }
    __syncwarp();
#pragma unroll
    for (int which = 0; which < 2; ++which)
      for (unsigned int todo = mend[which]; todo; todo &= todo - 1) attn_dkv_row<T>(a, b, hk, first + __ffs(todo) - 1, lane, which ? 1 : 2);
  }
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

// ------------------------------------------------------------------ queries
template <class T, int DP, int CW, bool CAP, bool BIAS>
__device__ __forceinline__ void attn_grad_queries(const b200_tmap& map_q, const b200_tmap& map_k, const b200_tmap& map_v, const b200_tmap& map_do,
                                                  const b200_tmap& map_dq, const AttnArgs& a, unsigned int block) {
  typedef BwdShape<DP, CW> Sh;
  extern __shared__ __align__(128) unsigned char dyn[];
  const unsigned int base = (b200_smem_addr(dyn) + 1023u) & ~1023u;
  unsigned char* const gen = dyn + (base - b200_smem_addr(dyn));
  const unsigned int q_at = base, do_at = base + Sh::kTile, ring = base + 2 * Sh::kTile;
  unsigned long long* bars = (unsigned long long*)(gen + Sh::kBytes);
  const unsigned int bar0 = b200_smem_addr(bars);
  const unsigned int bar_q = bar0, bar_full = bar0 + 8, bar_empty = bar0 + 24, bar_s = bar0 + 40;      // two each but bar_q
  const unsigned int bar_dp = bar0 + 56, bar_ds = bar0 + 64, bar_done = bar0 + 72;
  volatile unsigned int* tmem_slot = (volatile unsigned int*)(bars + 10);
  volatile unsigned int* abort_flag = tmem_slot + 1;
  float* scratch = (float*)(bars + 12);                   // [8]
  AttnSpan* span = (AttnSpan*)(bars + 18);
  unsigned char* classes = (unsigned char*)(gen + Sh::kBytes + 256);

  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  constexpr unsigned int kLoad = Sh::kWarps - 2, kMma = Sh::kWarps - 1;
  const unsigned int from_last = a.all_heads.of(block), bh = block - from_last * a.all_heads.d;
  const int tiles_q = (a.S + 127) / 128, t_q = tiles_q - 1 - (int)from_last, r0 = t_q * 128;
  const int b = (int)a.heads.of(bh), h = (int)bh - b * a.H, hk = (int)a.per_key_head.of((unsigned int)h);
  const bool docs = a.kdoc != nullptr;
  if (warp == kLoad) {
    if (lane < 10) b200_mbar_init(bar0 + 8 * lane, lane == 8 ? Sh::kGroups * 128 : 1);      // (bar_ds)
    if (lane == 10) {
      span->last_min = span->doc_min = 0x7fffffff;
      span->last_max = -1;
      span->doc_max = -0x7fffffff - 1;
      *abort_flag = 0u;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(b200_smem_addr((const void*)tmem_slot)), "r"(Sh::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tmem_taken();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const AttnSpan plain = plain_span(a, attn_seq(a, b), r0, 128);
  int tiles = (plain.last_max + CW) / CW;
  auto load = [&](int t, unsigned int n) {
    const unsigned int slot = n & 1u, at = ring + slot * Sh::kStage, bar = bar_full + 8 * slot;
    b200_mbar_expect_tx(bar, 2 * Sh::kStep);
#pragma unroll
    for (int p = 0; p < Sh::kPanels; ++p) {
      b200_tma_load_4d(at + p * Sh::kPanel, &map_k, bar, p * 64, t * CW, hk, b);
      b200_tma_load_4d(at + Sh::kStep + p * Sh::kPanel, &map_v, bar, p * 64, t * CW, hk, b);
    }
  };
  if (threadIdx.x == kLoad * 32) {
    b200_mbar_expect_tx(bar_q, 2 * Sh::kTile);
#pragma unroll
    for (int p = 0; p < Sh::kPanels; ++p) {
      b200_tma_load_4d(q_at + p * kTileBytes64, &map_q, bar_q, p * 64, r0, h, b);
      b200_tma_load_4d(do_at + p * kTileBytes64, &map_do, bar_q, p * 64, r0, h, b);
    }
    if (!docs && tiles) load(0, 0);
  }
  const unsigned int half = warp >> 2, in = (warp & 3u) * 32 + lane;
  const int r = r0 + (int)in;
  AttnRow row;
  row.pos = 0; row.last = -1; row.doc = 0;
  if (warp < kLoad && r < a.S) row = attn_row(a, b, r);
  tc_before();
  __syncthreads();
  tc_after();
  if (docs) {
    if (warp < 4) {
      const AttnSpan s = span_of(r < a.S, row);
      if (lane == 0) {
        atomicMin(&span->last_min, s.last_min);
        atomicMax(&span->last_max, s.last_max);
        atomicMin(&span->doc_min, s.doc_min);
        atomicMax(&span->doc_max, s.doc_max);
      }
    }
    __syncthreads();
    tiles = (span->last_max + CW) / CW;
    constexpr int kAhead = 4;
    for (int t0 = (int)warp; t0 < tiles; t0 += kAhead * (int)Sh::kWarps) {
      int kmin[kAhead], kmax[kAhead];
      bool negative[kAhead];
      key_documents<CW, kAhead>(a, b, t0, Sh::kWarps, lane, kmin, kmax, negative);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int t = t0 + n * (int)Sh::kWarps;
        const unsigned int cls = tile_class(*span, t * CW, CW, true, kmin[n], kmax[n], negative[n]);
        if (lane == 0 && t < tiles) classes[t] = (unsigned char)cls;
      }
    }
    __syncthreads();
  }
  auto class_of = [&](int t) { return docs ? (unsigned int)classes[t] : tile_class(plain, t * CW, CW, false, 0, 0, false); };
  const unsigned int tmem = *tmem_slot;
  const unsigned int t_dp = tmem + 2 * CW, t_dq = tmem + 3 * CW;     // two tiles of scores ahead of them

  if (warp == kLoad) {
    if (lane == 0) {
      unsigned int n = 0;
      bool live = true;
      for (int t = 0; t < tiles; ++t) {
        if (!class_of(t)) continue;
        if (docs || n) {
          if (n > 1) live = b200_wait(bar_empty + 8 * (n & 1u), ((n >> 1) - 1) & 1u, abort_flag, a.status, 41u);
          if (!live) break;
          load(t, n);
        }
        ++n;
      }
      if (*abort_flag) {
        for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bar_q, 0u); ++tries) {}
        for (unsigned int i = 0; i < 2 && i < n; ++i)
          for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bar_full + 8 * ((n - 1 - i) & 1u), ((n - 1 - i) >> 1) & 1u); ++tries) {}
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    if (b200_elect()) {
      constexpr unsigned int idesc_s = idesc_of<T>(128, CW, false, false), idesc_g = idesc_of<T>(128, DP, false, true);
      auto square = [&](unsigned int d, unsigned int x, unsigned int y) {
#pragma unroll
        for (int p = 0; p < Sh::kPanels; ++p) {
          const unsigned long long dx = b200_smem_desc(x + p * kTileBytes64, 16u, 1024u), dy = b200_smem_desc(y + p * Sh::kPanel, 16u, 1024u);
#pragma unroll
          for (unsigned int ks = 0; ks < 4; ++ks) b200_umma(d, dx + ks * 2, dy + ks * 2, idesc_s, (p || ks) ? 1u : 0u);
        }
      };
      int total = 0;
      for (int t = 0; t < tiles; ++t) total += class_of(t) != 0;
      bool live = b200_wait(bar_q, 0u, abort_flag, a.status, 42u);
      if (live && total) {
        live = b200_wait(bar_full, 0u, abort_flag, a.status, 43u);
        tc_after();
        if (live) {
          square(tmem, q_at, ring);
          b200_umma_commit(bar_s);
          square(t_dp, do_at, ring + Sh::kStep);
          b200_umma_commit(bar_dp);
        }
      }
      for (int n = 0; live && n < total; ++n) {
        const unsigned int at = ring + (n & 1) * Sh::kStage, next = ring + ((n + 1) & 1) * Sh::kStage;
        if (n + 1 < total) {
          live = b200_wait(bar_full + 8 * ((n + 1) & 1), ((n + 1) >> 1) & 1, abort_flag, a.status, 44u);
          if (!live) break;
          tc_after();
          square(tmem + CW * ((n + 1) & 1), q_at, next);
          b200_umma_commit(bar_s + 8 * ((n + 1) & 1));
        }
        live = b200_wait(bar_ds, n & 1, abort_flag, a.status, 45u);
        if (!live) break;
        tc_after();
        const unsigned long long dk = b200_smem_desc(at, Sh::kPanel, 1024u);
#pragma unroll
        for (unsigned int ks = 0; ks < CW / 16; ++ks) umma_ts(t_dq, t_dp + (ks >> 2) * 64 + (ks & 3u) * 8, dk + ks * 128, idesc_g, (n || ks) ? 1u : 0u);
        b200_umma_commit(bar_empty + 8 * (n & 1));
        if (n + 1 < total) {
          square(t_dp, do_at, next + Sh::kStep);
          b200_umma_commit(bar_dp);
        } else {
          b200_umma_commit(bar_done);
        }
      }
    }
    __syncwarp();
  } else {
    const unsigned int lanes = (warp & 3u) << 21;
    const unsigned int my_dp = t_dp + 64 * half + lanes;
    const float c = CAP ? a.cap * kLog2e : a.scale * kLog2e, to_tanh = CAP ? a.over : 0.f;
    const float slope2 = BIAS ? a.slopes[h] * kLog2e : 0.f;
    const float* stat = a.stat + (((long long)b * a.H + h) * tiles_q + t_q) * 256 + in;
    const float lse2 = stat[0], delta = stat[128];
    float grad_unit = 1.f;
    if constexpr (std::is_same<T, __half>::value) {
      // (of keys that some row of the tile sees)
      float of_v[1] = {0.f};
      const float* sizes = a.value_sizes + (long long)b * a.T * a.HK + hk;
      if (!docs) {
#pragma unroll 8
        for (int j = (int)threadIdx.x; j <= plain.last_max; j += Sh::kGroups * 128) of_v[0] = fmaxf(of_v[0], sizes[(long long)j * a.HK]);
      } else {
        // tiles of which all is seen are shared out; of the others a warp takes what its own rows see
        for (int t = 0; t < tiles; ++t) {
          const unsigned int cls = classes[t];
          if (!cls || (cls == 1u && (t & 3) != (int)(warp & 3u))) continue;
          const int first = t * CW + 64 * (int)half;
          unsigned int seen[2] = {0xffffffffu, 0xffffffffu};
          if (cls == 2u) visible_words<2>(a, b, first, row, lane, seen);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (__reduce_or_sync(0xffffffffu, seen[i]) >> lane & 1u) of_v[0] = fmaxf(of_v[0], sizes[(long long)(first + 32 * i + (int)lane) * a.HK]);
        }
      }
      const float2 s = a.row_sizes[(((long long)b * a.H + h) * tiles_q + t_q) * 128 + in];
      largest<Sh::kGroups * 4>(of_v, scratch);
      grad_unit = unit_of(fmaf(s.x, of_v[0], s.y));
    }
    const float to_unit = grad_unit * kWeightBack<T>;
    unsigned int n = 0;
    bool live = true;
    for (int t = 0; t < tiles; ++t) {
      const unsigned int cls = class_of(t);
      if (!cls) continue;
      unsigned int bits[2] = {0xffffffffu, 0xffffffffu};
      if (cls == 2u) visible_words<2>(a, b, t * CW + 64 * (int)half, row, lane, bits);
      live = b200_wait(bar_s + 8 * (n & 1u), (n >> 1) & 1u, abort_flag, a.status, 46u);
      if (!live) break;
      tc_after();
      float w[64];
      const unsigned int my_s = tmem + CW * (n & 1u) + 64 * half + lanes;
      auto weights = [&](auto masked) {
        constexpr bool M = decltype(masked)::value;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float x[32];
          b200_tmem_ld32(my_s + 32 * k, (unsigned int*)x);
          [[maybe_unused]] const float far = BIAS ? (float)(row.pos - t * CW - 64 * (int)half - 32 * k) : 0.f;
          tmem_wait_ld();
          if constexpr (CAP) tanh_chunk(x, to_tanh);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float p;
            if constexpr (!BIAS) p = ex2(fmaf(x[i], c, -lse2));
            else p = ex2(pair_score<BIAS>(x[i], c, slope2, far - (float)i) - lse2);
            if constexpr (M) p = (bits[k] >> i) & 1u ? p : 0.f;
            if constexpr (std::is_same<T, __half>::value) p *= to_unit;
            w[32 * k + i] = CAP ? p * fmaf(-x[i], x[i], 1.f) : p;
          }
        }
      };
      if (cls == 2u) weights(std::true_type());
      else weights(std::false_type());
      live = b200_wait(bar_dp, n & 1u, abort_flag, a.status, 47u);
      if (!live) break;
      tc_after();
      auto gradients = [&](auto masked) {
        constexpr bool M = decltype(masked)::value;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float x[32];
          unsigned int u[16];
          b200_tmem_ld32(my_dp + 32 * k, (unsigned int*)x);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            x[i] = w[32 * k + i] * (x[i] - delta);
            if constexpr (M) x[i] = (bits[k] >> i) & 1u ? x[i] : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) u[i / 2] = pack2(x[i], x[i + 1], T());
          tmem_st16(my_dp + 16 * k, u);
        }
      };
      if (cls == 2u) gradients(std::true_type());
      else gradients(std::false_type());
      tmem_wait_st();
      tc_before();
      b200_mbar_arrive(bar_ds);
      ++n;
    }
    // ---- dq through the queries' tile: 32 rows a warp, half of a row's elements where two threads share it
    if (live) live = b200_wait(n ? bar_done : bar_q, 0u, abort_flag, a.status, 48u);
    tc_after();
    const float by = a.scale / grad_unit;
    const int first = r0 + (int)(warp & 3u) * 32;
    constexpr int kMine = DP / Sh::kGroups;
    bool fine = true;
#pragma unroll
    for (int e = 0; e < kMine; e += 32) {
      float o[32];
      const int col = (int)half * kMine + e;
      if (live && n) {
        b200_tmem_ld32(t_dq + lanes + col, (unsigned int*)o);
        tmem_wait_ld();
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = n ? o[i] * by : 0.f;
      fine &= store_columns<T>(gen, in, col, o);
    }
    unsigned int mend = __ballot_sync(0xffffffffu, live && r < a.S && !fine);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0 && live && first < a.S) {
#pragma unroll
      for (int p = (int)half * kMine / 64; p < ((int)half + 1) * kMine / 64; ++p)
        if (p * 64 < a.D) b200_tma_store_4d(&map_dq, q_at + p * kTileBytes64 + (warp & 3u) * 4096, p * 64, first, h, b);
    }
    bool all_out = mend != 0u;         // whether the copies have to be complete, not only read
    if (Sh::kGroups == 2) {
      // two warps share their rows: a row to be done again is done by the first, when both halves are out
      volatile unsigned int* mends = (volatile unsigned int*)(bars + 22);
      if (lane == 0) mends[warp] = mend;
      named_barrier(1 + (int)(warp & 3u), 64);
      mend |= mends[warp ^ 4u];
      all_out = mend != 0u;
    }
    if (lane == 0 && live) {
      if (all_out) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      else b200_tma_store_read_wait<0>();
    }
    __syncwarp();
    if (Sh::kGroups == 2 && all_out) {
      named_barrier(1 + (int)(warp & 3u), 64);
      if (half) mend = 0u;
    }
    for (unsigned int todo = mend; todo; todo &= todo - 1) attn_dq_row<T>(a, b, h, first + __ffs(todo) - 1, lane);
  }
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

// Adds the parts of every key's gradients in their order, a warp a row; DP: 64 or 128
template <class T, int DP>
__global__ void __launch_bounds__(256) attn_join_parts(const __grid_constant__ AttnArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const unsigned int lane = threadIdx.x & 31u;
  const long long rows = (long long)a.B * a.T * a.HK;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows; i += (long long)gridDim.x * 8) {
    int again = 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {          // dk, dv
      float v[DP / 32];
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) v[k] = 0.f;
      for (int p = 0; p < a.n_parts; ++p) {
        const float* from = a.parts + ((2 * p + which) * rows + i) * DP;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k) v[k] += from[lane + 32 * k];
      }
      bool fine = true;
      T* to = (T*)(which ? a.dv : a.dk) + i * a.ld;
#pragma unroll
      for (int k = 0; k < DP / 32; ++k)
        if ((int)lane + 32 * k < a.D) {
          from_float(v[k], to[lane + 32 * k]);
          fine = fine && v[k] * 0.f == 0.f;
        }
      if (attn_again(fine)) again |= 1 << which;
    }
    if (again) {
      const long long bt = i / a.HK;
      attn_dkv_row<T>(a, (int)(bt / a.T), (int)(i - bt * a.HK), (int)(bt % a.T), lane, again);
    }
  }
}

// What both kinds of CTAs are given: a tensor map for the rows a CTA owns and one for the tiles it walks
struct GradMaps {
  b200_tmap q, k, v, d_out, own_q, own_k, own_v, own_d_out, dq, dk, dv;
};

// The keys' CTAs come first: theirs are the longer walks.
template <class T, int DP, int CW, bool CAP, bool BIAS>
__global__ void __launch_bounds__(BwdShape<DP, CW>::kThreads, CW == 64 ? 2 : 1)
attn_grad_tc(const __grid_constant__ GradMaps m, const __grid_constant__ AttnArgs a, unsigned int keys_grid) {
  if (blockIdx.x < keys_grid) attn_grad_keys<T, DP, CW, CAP, BIAS>(m.q, m.own_k, m.own_v, m.d_out, m.dk, m.dv, a, blockIdx.x);
  else attn_grad_queries<T, DP, CW, CAP, BIAS>(m.own_q, m.k, m.v, m.own_d_out, m.dq, a, blockIdx.x - keys_grid);
}

}  // namespace b200
#endif
