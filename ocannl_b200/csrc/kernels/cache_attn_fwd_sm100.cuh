// Attention of many new tokens over a paged cache on the tensor cores (tcgen05), 16-bit heads: prompts, and parts of them.
//
// A CTA takes NQ tiles of 128 rows of one (sequence, key head): the query heads that share the keys lie beside each other, token by token, so that a tile is 128 /
// group tokens.  Roles: a warp that copies (TMA: the queries once, then tiles of 64 tokens, each in as many boxes as it has pages; a page that is not there is
// a box outside the cache, which arrives as zeros), a warp that issues tcgen05.mma, and four warps a row tile that do the softmax, a thread a row, as in
// attention over whole sequences: two places of 64 scores in tensor memory, so that the next scores are formed during the softmax of these, weights written
// over them as the second product's operand, accumulators in tensor memory that are multiplied only when a row's maximum has grown by 2^8.
//
// Codes of 8 bits arrive as they are and two more warps make halves of them, in the layout the tensor cores read: 128 x 2 conversions a tile of 64 tokens
// for each of their threads, beside the 1000 cycles that its products take.  Scales stay outside, as with few rows: a page's scale of the keys
// multiplies its scores, that of the values raises its weights' exponents and is taken off the sum.  (bfloat16 queries beside codes are made halves in
// shared memory by the softmax's threads, each row brought to 2^14.)
//
// Bound by the chain product, weights, product of a tile: 4096 new tokens of sequences of 8192, 32 heads over 8 of 128, codes, take 364 to 428 us on several machines
// (958 to 815 TFLOP/s), tensor pipe and exponential unit 41 % busy each over a grid of 3.6 uneven rounds.  (3000 half tokens, a window of 700, 16 heads over 4, capped:
// 52 to 73 us, 254 in tiles of 8 rows.)
//
// Over more than kSumKeys tokens the accumulators are added to sums in tensor memory of their own every so many tiles (NQ = 1, which has room for them).
#ifndef B200_CACHE_ATTN_FWD_SM100_CUH
#define B200_CACHE_ATTN_FWD_SM100_CUH
#include "attn_fwd_sm100.cuh"
#include "cache_attn_terms.cuh"

namespace b200 {

struct CacheTileArgs {
  Divisor by_group, by_key_heads;
  int tokens;              // of a tile of 128 rows
  int box;                 // rows of a TMA box of the cache
  int sums;                // more than kSumKeys tokens may be walked
};

template <int DP, int NQ, bool CODED>
struct CacheTileShape {
  static constexpr int kPanels = DP / 64;
  static constexpr unsigned int kTile = kPanels * kTileBytes64;              // queries
  static constexpr unsigned int kPanel = 64 * 128, kKeys = kPanels * kPanel; // 64 keys or values
  static constexpr int kSlots = CODED ? 2 : NQ == 2 ? 4 : 2;
  static constexpr unsigned int kRaw = 64 * DP;                              // codes of 64 tokens
  static constexpr int kRawSlots = CODED ? 4 : 1;                            // keys and values in turn
  static constexpr unsigned int kBytes = NQ * kTile + 2 * kSlots * kKeys + (CODED ? kRawSlots * kRaw : 0);
  static constexpr unsigned int kThreads = NQ * 128 + 64 + (CODED ? 64 : 0);
  static constexpr int kMeta = 8;                                            // tiles whose scales are kept: no fewer than two rings of the keys
  static constexpr size_t kSmem = 1024 + kBytes + 512 + kMeta * 64;
  static constexpr int kBlocks = NQ == 1 && DP == 64 && !CODED ? 2 : 1;
};

// of a group of 16 tokens: the scale of the keys, the logarithm and the inverse of that of the values, and whether its page is there
struct CacheMeta {
  float down, raise, back, there;
};

__device__ __forceinline__ unsigned int low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

template <class T, int DP, int NQ, bool CODED>
__global__ void __launch_bounds__((CacheTileShape<DP, NQ, CODED>::kThreads), (CacheTileShape<DP, NQ, CODED>::kBlocks))
cache_attention_tc(const __grid_constant__ b200_tmap map_q, const __grid_constant__ b200_tmap map_k, const __grid_constant__ b200_tmap map_v,
                   const __grid_constant__ CacheAttnArgs a, const __grid_constant__ CacheTileArgs f) {
  typedef CacheTileShape<DP, NQ, CODED> Sh;
  typedef typename std::conditional<CODED, __half, T>::type M;               // what is multiplied
  constexpr bool kConvert = CODED && std::is_same<T, __nv_bfloat16>::value;  // queries become halves
  constexpr unsigned int kLoad = NQ * 4, kMma = NQ * 4 + 1, kColumns = NQ == 1 && DP == 64 ? 256 : 512;
  extern __shared__ __align__(128) unsigned char dyn[];
  const unsigned int base = (b200_smem_addr(dyn) + 1023u) & ~1023u;
  unsigned char* const gen = dyn + (base - b200_smem_addr(dyn));
  const unsigned int q_at = base, k_at = base + NQ * Sh::kTile, v_at = k_at + Sh::kSlots * Sh::kKeys, raw_at = v_at + Sh::kSlots * Sh::kKeys;
  unsigned long long* bars = (unsigned long long*)(gen + Sh::kBytes);
  const unsigned int bar0 = b200_smem_addr(bars);
  // queries, and their halves; four slots each: keys full, empty, values full, empty; codes full, empty; scores and weights: two places a row tile
  const unsigned int bar_q = bar0, bar_h = bar0 + 8, bar_kf = bar0 + 16, bar_ke = bar0 + 48, bar_vf = bar0 + 80, bar_ve = bar0 + 112, bar_rf = bar0 + 144, bar_re = bar0 + 176;
  const unsigned int bar_s = bar0 + 208, bar_p = bar0 + 240, bar_o = bar0 + 272, bar_f = bar0 + 288;
  constexpr unsigned int kBarriers = 38;
  volatile unsigned int* tmem_slot = (volatile unsigned int*)(bars + kBarriers);
  volatile unsigned int* abort_flag = tmem_slot + 1;
  CacheMeta* meta = (CacheMeta*)(gen + Sh::kBytes + 512);                    // [kMeta][4]

  const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const CacheArgs& c = a.c;
  if (warp == kLoad) {
    for (unsigned int i = lane; i < kBarriers; i += 32) {
      const unsigned int at = bar0 + 8 * i;
      unsigned int many = 1;
      if (at == bar_h) many = NQ * 128;
      if (at >= bar_p && at < bar_o) many = 128;
      if (CODED && ((at >= bar_kf && at < bar_ke) || (at >= bar_vf && at < bar_ve) || (at >= bar_re && at < bar_s))) many = 64;
      b200_mbar_init(at, many);
    }
    if (lane == 0) *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(b200_smem_addr((const void*)tmem_slot)), "r"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tmem_taken();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // ---- this CTA's rows: a sequence's last ones first, which see the most tokens
  const int per_cta = NQ * f.tokens;
  int b = 0;
  unsigned int nth = 0;
  const bool found = find_unit<Sh::kThreads>(
      c.batch, blockIdx.x, [&](int i) { return ((unsigned int)cache_seq(c, i).count + per_cta - 1) / per_cta * (unsigned int)c.HK; }, b, nth);
  CacheSeq s = {0, 0, 0};
  if (found) s = cache_seq(c, b);
  const unsigned int tiles = ((unsigned int)s.count + per_cta - 1) / per_cta, tile = tiles - 1 - f.by_key_heads.of(nth);
  const int hk = (int)(nth % (unsigned int)c.HK);
  const int token0 = found ? (int)tile * per_cta : 0;                        // of the sequence's new ones
  const int n_new = found ? min(per_cta, s.count - token0) : 0;
  const int least_pos = s.pos0 + token0, most_pos = least_pos + n_new - 1;
  const int end = n_new ? cache_last(a, most_pos) + 1 : 0;
  // the walk: tokens 0 .. sink_end - 1, then those from sink_end + shift on
  int sink_end = 0, shift = 0;
  if (a.window) {
    sink_end = (int)min(((long long)min(a.sinks, max(end, 0)) + 63) & ~63ll, 0x7fffffc0ll);
    shift = max((cache_first(a, least_pos) & ~63) - sink_end, 0);
  }
  const int n_tokens = shift ? max(end - shift, sink_end) : max(end, 0), n_tiles = n_new ? n_tokens / 64 + (n_tokens % 64 != 0) : 0;
  auto token_of = [&](int t) { return t * 64 < sink_end ? t * 64 : t * 64 + shift; };
  // what row tile i sees of a tile of tokens: 0 nothing, 1 everything (pages aside), 2 some
  auto class_of = [&](int t, int i) -> unsigned int {
    const int from = i * f.tokens, to = min(n_new, from + f.tokens) - 1, j0 = token_of(t);
    if (to < from) return 0u;
    const int lo = least_pos + from, hi = least_pos + to;
    if (j0 > cache_last(a, hi) || (a.window && j0 >= a.sinks && j0 + 63 < cache_first(a, lo))) return 0u;
    return j0 + 63 <= cache_last(a, lo) && (!a.window || j0 >= cache_first(a, hi) || j0 + 63 < a.sinks) ? 1u : 2u;
  };
  tc_before();
  __syncthreads();
  tc_after();
  const unsigned int tmem = *tmem_slot;
  const unsigned int acc_o = tmem + NQ * 128;              // output accumulators behind the scores, and behind them (NQ = 1) sums of them

  if (warp == kLoad) {
    // ---------------------------------------------------------------- copies
    bool live = true;
    if (lane == 0 && n_tiles) {
      b200_mbar_expect_tx(bar_q, NQ * Sh::kPanels * (unsigned int)(a.group * f.tokens) * 128u);
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int p = 0; p < Sh::kPanels; ++p) b200_tma_load_4d(q_at + i * Sh::kTile + p * kTileBytes64, &map_q, bar_q, p * 64, 0, hk, s.first + token0 + i * f.tokens);
    }
    const int boxes = 64 / f.box, per_group = f.box / 16;
    int page = -1;
    CacheMeta of_group = {1.f, 0.f, 1.f, 0.f};
    unsigned int filled[2] = {0, 0};
    for (int t = 0; t < n_tiles && live; ++t) {
      if ((t & 7) == 0) {
        // the pages and scales of eight tiles, a group of 16 tokens a lane
        const int mine = t + (int)(lane >> 2), j = token_of(mine) + (int)(lane & 3u) * 16;
        page = mine < n_tiles && j < end ? cache_page_at(c, b, c.by_page.of((unsigned int)j)) : -1;
        of_group.there = page >= 0 ? 1.f : 0.f;
        if constexpr (CODED) {
          of_group.down = of_group.back = 1.f;
          of_group.raise = 0.f;
          if (page >= 0) {
            of_group.down = cache_scale(__ldg(c.k_scale + (long long)page * c.HK + hk));
            const float v = cache_scale(__ldg(c.v_scale + (long long)page * c.HK + hk));
            of_group.back = rcp(v);
            asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(of_group.raise) : "f"(v));
          }
        }
      }
      const int j0 = token_of(t);
      const unsigned int tile_at = (unsigned int)t;
#pragma unroll
      for (int which = 0; which < 2; ++which) {              // keys, then values; codes of both go through one ring
        const unsigned int item = CODED ? 2 * tile_at + which : tile_at;
        constexpr unsigned int kRing = CODED ? 4 : Sh::kSlots;
        const unsigned int slot = item % kRing, use = item / kRing;
        const unsigned int full = (CODED ? bar_rf : which ? bar_vf : bar_kf) + 8 * slot, empty = (CODED ? bar_re : which ? bar_ve : bar_ke) + 8 * slot;
        const unsigned int to = CODED ? raw_at + slot * Sh::kRaw : (which ? v_at : k_at) + slot * Sh::kKeys;
        if (lane == 0 && live && use) live = b200_wait(empty, (use - 1) & 1u, abort_flag, a.status, 61u);
        live = __shfl_sync(0xffffffffu, (int)live, 0) != 0;
        if (live) {
          if (which == 0 && (int)(lane >> 2) == (t & 7)) meta[(tile_at % Sh::kMeta) * 4 + (lane & 3u)] = of_group;
          __syncwarp();
          if (lane == 0) b200_mbar_expect_tx(full, CODED ? Sh::kRaw : Sh::kKeys);
          ++filled[which];
          for (int i = 0; i < boxes; ++i) {
            const int p = __shfl_sync(0xffffffffu, page, (t & 7) * 4 + i * per_group), j = j0 + i * f.box;
            const int at = (int)((unsigned int)j - c.by_page.of((unsigned int)j) * c.page);
            if (lane == 0) {
              if (CODED)
                b200_tma_load_4d(to + i * f.box * DP, which ? &map_v : &map_k, full, 0, at, hk, p < 0 ? (int)c.n_pages : p);
              else
#pragma unroll
                for (int k = 0; k < Sh::kPanels; ++k)
                  b200_tma_load_4d(to + k * Sh::kPanel + i * f.box * 128, which ? &map_v : &map_k, full, k * 64, at, hk, p < 0 ? (int)c.n_pages : p);
            }
          }
        }
      }
    }
    // the copies under way land before shared memory is given up, whatever happened to the others
    if (lane == 0 && *abort_flag && n_tiles) {
      auto landed = [&](unsigned int bars_at, unsigned int ring, unsigned int many) {
        for (unsigned int k = 0; k < ring && k < many; ++k)
          for (int tries = 0; tries < 1 << 20 && !b200_mbar_try(bars_at + 8 * ((many - 1 - k) % ring), ((many - 1 - k) / ring) & 1u); ++tries) {}
      };
      landed(bar_q, 1, 1);
      if (CODED) {
        landed(bar_rf, 4, filled[0] + filled[1]);
      } else {
        landed(bar_kf, Sh::kSlots, filled[0]);
        landed(bar_vf, Sh::kSlots, filled[1]);
      }
    }
    __syncwarp();
  } else if (warp == kMma) {
    // ---------------------------------------------------------------- products
    if (b200_elect() && n_tiles) {
      constexpr unsigned int idesc_s = idesc_of<M>(128, 64, false, false), idesc_o = idesc_of<M>(128, DP, false, true);
      bool live = b200_wait(kConvert ? bar_h : bar_q, 0u, abort_flag, a.status, 63u);
      unsigned int scored[NQ], done[NQ];         // tiles whose scores are queued, whose weights have been multiplied
      int last[NQ];                              // the last tile of tokens that a row tile sees: its product is awaited
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        scored[i] = done[i] = 0;
        for (last[i] = n_tiles - 1; last[i] >= 0 && !class_of(last[i], i); --last[i]) {}
      }
      auto scores = [&](int i, unsigned int slot) {
        const unsigned int place = scored[i]++ & 1u;
#pragma unroll
        for (int p = 0; p < Sh::kPanels; ++p) {
          const unsigned long long dq = b200_smem_desc(q_at + i * Sh::kTile + p * kTileBytes64, 16u, 1024u);
          const unsigned long long dk = b200_smem_desc(k_at + slot * Sh::kKeys + p * Sh::kPanel, 16u, 1024u);
#pragma unroll
          for (unsigned int ks = 0; ks < 4; ++ks) b200_umma(tmem + i * 128 + place * 64, dq + ks * 2, dk + ks * 2, idesc_s, (p || ks) ? 1u : 0u);
        }
        b200_umma_commit(bar_s + 16 * i + 8 * place);
      };
      if (live) {
        live = b200_wait(bar_kf, 0u, abort_flag, a.status, 64u);
        tc_after();
        if (live) {
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (class_of(0, i)) scores(i, 0);
          b200_umma_commit(bar_ke);
        }
      }
      for (int t = 0; live && t < n_tiles; ++t) {
        const unsigned int slot = t % Sh::kSlots, ph = (t / Sh::kSlots) & 1u, slot1 = (t + 1) % Sh::kSlots, ph1 = ((t + 1) / Sh::kSlots) & 1u;
        if (t + 1 < n_tiles) {
          live = b200_wait(bar_kf + 8 * slot1, ph1, abort_flag, a.status, 65u);
          if (!live) break;
          tc_after();
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (class_of(t + 1, i)) scores(i, slot1);
          b200_umma_commit(bar_ke + 8 * slot1);
        }
        live = b200_wait(bar_vf + 8 * slot, ph, abort_flag, a.status, 66u);
        if (!live) break;
        tc_after();
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          if (!class_of(t, i)) continue;
          live = b200_wait(bar_p + 16 * i + 8 * (done[i] & 1u), done[i] >> 1 & 1u, abort_flag, a.status, 67u);
          if (!live) break;
          tc_after();
          const unsigned int weights = tmem + i * 128 + (done[i] & 1u) * 64;
          const unsigned long long dv = b200_smem_desc(v_at + slot * Sh::kKeys, Sh::kPanel, 1024u);
#pragma unroll
          for (unsigned int ks = 0; ks < 4; ++ks) umma_ts(acc_o + i * DP, weights + ks * 8, dv + ks * 128, idesc_o, (done[i] || ks) ? 1u : 0u);
          // the last product has a barrier of its own: the others' may be two phases behind when it is waited for
          if (t == last[i]) b200_umma_commit(bar_f + 8 * i);
          else b200_umma_commit(bar_o + 8 * i);
          ++done[i];
        }
        if (!live) break;
        b200_umma_commit(bar_ve + 8 * slot);
      }
    }
    __syncwarp();
  } else if (warp > kMma) {
    // ---------------------------------------------------------------- codes become halves
    if constexpr (CODED) {
      const unsigned int me = threadIdx.x - (kMma + 1) * 32;                 // of 64
      constexpr int kPieces = DP / 16;                                       // of a token: 16 codes each
      bool live = true;
      for (unsigned int item = 0; live && item < 2u * (unsigned int)n_tiles; ++item) {
        const unsigned int raw = item % Sh::kRawSlots, n = item >> 1, slot = n % Sh::kSlots, use = n / Sh::kSlots, value = item & 1u;
        live = b200_wait(bar_rf + 8 * raw, (item / Sh::kRawSlots) & 1u, abort_flag, a.status, 68u);
        if (live && use) live = b200_wait((value ? bar_ve : bar_ke) + 8 * slot, (use - 1) & 1u, abort_flag, a.status, 69u);
        if (!live) break;
        const unsigned char* from = gen + (raw_at - base) + raw * Sh::kRaw;
        unsigned char* to = gen + ((value ? v_at : k_at) - base) + slot * Sh::kKeys;
#pragma unroll 4
        for (int i = 0; i < kPieces; ++i) {
          const unsigned int piece = me + 64 * i, row = piece / kPieces, p = piece % kPieces;
          const uint4 w = *(const uint4*)(from + row * DP + p * 16);
          uint4 lo, hi;
          e4m3_split(w.x, lo.x, lo.y);
          e4m3_split(w.y, lo.z, lo.w);
          e4m3_split(w.z, hi.x, hi.y);
          e4m3_split(w.w, hi.z, hi.w);
          unsigned char* line = to + (p >> 2) * Sh::kPanel + row * 128;
          const unsigned int chunk = (p & 3u) * 2;
          *(uint4*)(line + ((chunk ^ (row & 7u)) << 4)) = lo;
          *(uint4*)(line + (((chunk + 1) ^ (row & 7u)) << 4)) = hi;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        b200_mbar_arrive((value ? bar_vf : bar_kf) + 8 * slot);
        b200_mbar_arrive(bar_re + 8 * raw);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax: a thread a row
    const unsigned int g = warp >> 2;                                        // its row tile
    const int in_tile = (int)(threadIdx.x & 127u);
    const unsigned int mine = tmem + g * 128 + ((warp & 3u) << 21), mine_o = acc_o + g * DP + ((warp & 3u) << 21), mine_sum = mine_o + DP;
    const int of_token = (int)f.by_group.of((unsigned int)in_tile), token = (int)g * f.tokens + of_token, h = hk * a.group + in_tile - of_token * a.group;
    const bool on = of_token < f.tokens && token < n_new;                    // a row of a token
    const int pos = on ? least_pos + token : -1, last = on ? cache_last(a, pos) : -1, first = cache_first(a, pos);
    const float slope2 = a.slopes && on ? a.slopes[h] * kCacheLog2e : 0.f;
    float unit = a.cap > 0.f ? a.over : a.scale * kCacheLog2e;
    bool live = true;
    if (kConvert && n_tiles) {
      live = b200_wait(bar_q, 0u, abort_flag, a.status, 70u);
      // this row's queries in halves, the largest at 2^14 (none for zeros, and for what is infinite or undefined)
      unsigned char* row = gen + g * Sh::kTile + in_tile * 128;
      unsigned int most = 0;
#pragma unroll 4
      for (int i = 0; i < DP / 8; ++i) {
        const uint4 w = *(const uint4*)(row + (i >> 3) * kTileBytes64 + (((i & 7) ^ (in_tile & 7)) << 4));
        const unsigned int u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max(most, max(u[k] & 0x7fffu, (u[k] >> 16) & 0x7fffu));
      }
      const int e = (int)(most >> 7), up = e == 0 || e == 255 ? 0 : min(max(127 + 14 - e, -126), 126);
      const float by = power_of_two(up);
      unit *= power_of_two(-up);
#pragma unroll 4
      for (int i = 0; i < DP / 8; ++i) {
        uint4* at = (uint4*)(row + (i >> 3) * kTileBytes64 + (((i & 7) ^ (in_tile & 7)) << 4));
        const uint4 w = *at;
        unsigned int u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = unpack2(u[k], __nv_bfloat16());
          u[k] = pack2(x.x * by, x.y * by, __half());
        }
        *at = make_uint4(u[0], u[1], u[2], u[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      b200_mbar_arrive(bar_h);
    }
    const float to_log2 = a.cap * kCacheLog2e;
    float m = -INFINITY, l = 0.f;
    unsigned int seen = 0;
    constexpr unsigned int kSumTiles = kSumKeys / 64;
    bool summed = false;
    for (int t = 0; t < n_tiles && live; ++t) {
      const unsigned int cls = class_of(t, (int)g);
      if (!cls) continue;
      const unsigned int place = seen & 1u, at = mine + place * 64;
      live = b200_wait(bar_s + 16 * g + 8 * place, seen >> 1 & 1u, abort_flag, a.status, 71u);
      if (!live) break;
      tc_after();
      float x[64];
      b200_tmem_ld32(at, (unsigned int*)x);
      b200_tmem_ld32(at + 32, (unsigned int*)x + 32);
      const int j0 = token_of(t);
      // a multiplication and an addition for each group of 16 tokens
      float mul[4], add[4];
      [[maybe_unused]] float back[4];
      float there = 4.f;
      {
        const CacheMeta* w = meta + ((unsigned int)t % Sh::kMeta) * 4;
        there = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 z = *(const float4*)&w[k];
          mul[k] = CODED ? unit * z.x : unit;
          add[k] = CODED ? z.y : 0.f;
          back[k] = z.z;
          there += z.w;
        }
      }
      tmem_wait_ld();
      const bool plain = cls == 1u && there == 4.f;
      if (!plain || a.cap > 0.f || a.slopes) {
        if (a.cap > 0.f) {
#pragma unroll
          for (int j = 0; j < 64; ++j) x[j] *= mul[j >> 4];
          tanh_chunk(x, 1.f);
#pragma unroll
          for (int j = 0; j < 64; ++j) x[j] = fmaf(x[j], to_log2, add[j >> 4]);
        } else {
#pragma unroll
          for (int j = 0; j < 64; ++j) x[j] = fmaf(x[j], mul[j >> 4], add[j >> 4]);
        }
        if (a.slopes) {
          const float from = (float)(pos - j0);
#pragma unroll
          for (int j = 0; j < 64; ++j) x[j] = fmaf(-slope2, from - (float)j, x[j]);
        }
        if (!plain) {
          const CacheMeta* w = meta + ((unsigned int)t % Sh::kMeta) * 4;
          unsigned int bits[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int j = j0 + 32 * i;
            bits[i] = low_bits(last + 1 - j) & (~low_bits(first - j) | low_bits(a.window ? a.sinks - j : 0)) & ((w[2 * i].there != 0.f ? 0xffffu : 0u) | (w[2 * i + 1].there != 0.f ? 0xffff0000u : 0u));
          }
#pragma unroll
          for (int j = 0; j < 64; ++j) x[j] = (bits[j >> 5] >> (j & 31)) & 1u ? x[j] : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) mul[k] = 1.f, add[k] = 0.f;
      }
      float m_tile = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float top = x[16 * k], other = x[16 * k + 1];
#pragma unroll
        for (int j = 2; j < 16; j += 2) {
          top = fmaxf(top, x[16 * k + j]);
          other = fmaxf(other, x[16 * k + j + 1]);
        }
        m_tile = fmaxf(m_tile, fmaf(fmaxf(top, other), mul[k], add[k]));
      }
      if (!on) m_tile = -INFINITY;               // (what lies in a row of no token has no say in when the others' maxima move)
      if (NQ == 1 && f.sums && seen && seen % kSumTiles == 0) {
        // the accumulators are added to the sums (the product before is waited for as below)
        live = b200_wait(bar_o + 8 * g, (seen - 1) & 1u, abort_flag, a.status, 72u);
        tc_after();
#pragma unroll
        for (int e = 0; e < DP; e += 16) {
          float o[16], w[16];
          b200_tmem_ld16(mine_o + e, (unsigned int*)o);
          if (summed) b200_tmem_ld16(mine_sum + e, (unsigned int*)w);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            w[j] = summed ? w[j] + o[j] : o[j];
            o[j] = 0.f;
          }
          tmem_st16(mine_sum + e, (const unsigned int*)w);
          tmem_st16(mine_o + e, (const unsigned int*)o);
        }
        summed = true;
      }
      // the maximum in use moves when some row of the warp has outgrown it (or has had none)
      if (__any_sync(0xffffffffu, m_tile > m + 8.f || (m == -INFINITY && m_tile != -INFINITY))) {
        const float m_new = fmaxf(m, m_tile);
        const float by = m == -INFINITY ? 0.f : ex2(m - m_new);
        if (seen) {
          live = b200_wait(bar_o + 8 * g, (seen - 1) & 1u, abort_flag, a.status, 73u);
          tc_after();
#pragma unroll
          for (int e = 0; e < (NQ == 1 ? 2 * DP : DP); e += 16) {
            if (e >= DP && !summed) break;
            float o[16];
            b200_tmem_ld16(mine_o + e, (unsigned int*)o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = by == 0.f ? 0.f : o[j] * by;
            tmem_st16(mine_o + e, (const unsigned int*)o);
          }
        }
        l *= by;
        m = m_new;
      }
      const float off = m == -INFINITY ? 0.f : kLift<M> - m;
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        unsigned int w[16];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const Pair mul2_(mul[k + i], mul[k + i]), off2(add[k + i] + off, add[k + i] + off);
          Pair part(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            float p0, p1;
            fma2(Pair(x[16 * (k + i) + j], x[16 * (k + i) + j + 1]), mul2_, off2).get(p0, p1);
            p0 = ex2(p0);
            p1 = ex2(p1);
            part = add2(part, Pair(p0, p1));
            w[8 * i + j / 2] = pack2(p0, p1, M());
          }
          float l0, l1;
          part.get(l0, l1);
          l = CODED ? fmaf(l0 + l1, back[k + i], l) : l + (l0 + l1);
        }
        tmem_st16(at + 8 * k, w);
      }
      tmem_wait_st();
      tc_before();
      b200_mbar_arrive(bar_p + 16 * g + 8 * place);
      ++seen;
    }
    // ---------------------------------------------------------------- output
    // (it goes through the queries' tile, which has to have arrived even where nobody reads it)
    if (live && n_tiles) live = b200_wait(seen ? bar_f + 8 * g : bar_q, 0u, abort_flag, a.status, 74u);
    tc_after();
    const float by = l > 0.f || l != l ? 1.f / l : 0.f;
    // (of scores beyond 2^23 the product, which is not rounded, and the maximum, which is, may lie far apart: such rows are done again)
    float bad = fabsf(m) > 8388608.f && seen && m != -INFINITY ? 1.f : 0.f;
    unsigned char* tile_at = gen + g * Sh::kTile;  // its last product is done
#pragma unroll
    for (int e = 0; e < DP; e += 16) {
      float o[16], w[16];
      if (live && seen) {
        b200_tmem_ld16(mine_o + e, (unsigned int*)o);
        if (NQ == 1 && summed) b200_tmem_ld16(mine_sum + e, (unsigned int*)w);
        tmem_wait_ld();
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (NQ == 1 && summed) o[j] += w[j];
        o[j] = by == 0.f ? 0.f : o[j] * by;
        bad = fmaf(o[j], 0.f, bad);
      }
      unsigned char* line = tile_at + (e >> 6) * kTileBytes64 + in_tile * 128;
      const unsigned int piece0 = (e & 63) >> 3;
#pragma unroll
      for (int p = 0; p < 2; ++p)
        *(uint4*)(line + (((piece0 + p) ^ (in_tile & 7)) << 4)) =
            make_uint4(pack2(o[8 * p], o[8 * p + 1], T()), pack2(o[8 * p + 2], o[8 * p + 3], T()), pack2(o[8 * p + 4], o[8 * p + 5], T()), pack2(o[8 * p + 6], o[8 * p + 7], T()));
    }
    const long long row = (long long)(s.first + token0 + token);
    if (live && on && a.lse) a.lse[row * a.H + h] = l > 0.f || l != l ? (m - kLift<M> + log2f(l)) * kCacheLn2 : -INFINITY;
    const unsigned int store = __ballot_sync(0xffffffffu, live && on), mend = __ballot_sync(0xffffffffu, live && on && bad != 0.f);
    __syncwarp();
    // a warp's 32 rows leave as whole lines: 16 bytes a lane
    constexpr int kLanes = DP / 8;
    const int piece = (int)lane % kLanes;
    for (int i = (int)lane / kLanes; i < 32; i += 32 / kLanes) {
      const int r = (int)(warp & 3u) * 32 + i;
      const int tk = (int)f.by_group.of((unsigned int)r);
      const uint4 w = *(const uint4*)(tile_at + (piece >> 3) * kTileBytes64 + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
      if ((store >> i & 1u) && piece * 8 < c.D)
        *(uint4*)((T*)a.out + ((long long)(s.first + token0 + (int)g * f.tokens + tk) * a.H + hk * a.group + r - tk * a.group) * c.D + piece * 8) = w;
    }
    __syncwarp();
    for (unsigned int todo = mend; todo; todo &= todo - 1) {
      const int r = (int)(warp & 3u) * 32 + __ffs((int)todo) - 1, tk = (int)f.by_group.of((unsigned int)r), nth_token = (int)g * f.tokens + tk;
      cache_attention_row<T, CODED>(a, b, hk * a.group + r - tk * a.group, s.first + token0 + nth_token, least_pos + nth_token, lane);
    }
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
}

}  // namespace b200
#endif
