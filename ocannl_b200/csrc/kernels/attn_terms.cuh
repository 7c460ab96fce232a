// What the attention operators' kernels share: the arguments, which keys a query sees, the score, and the plain row by row
// forms.
//
// All masks come down to one number and one document a row: query r of sequence b sees key j when
//     j <= last   and, with documents,   key_documents[b, j] == doc,
// where last is -1 for a row that sees nothing.  Scores are kept in units of log 2, so that a weight is one exp2.
#ifndef B200_ATTN_TERMS_CUH
#define B200_ATTN_TERMS_CUH
#include "op_common.cuh"

namespace b200 {

struct AttnArgs {
  const void *q, *k, *v, *o, *d_out;     // o: the forward pass's output, read by the gradient
  void *out, *dq, *dk, *dv;
  float* lse;                            // [batch, heads, queries]
  float* stat;                           // gradient: a tile of 128 queries of a head: lse / log 2 of each, then <d_out, out>
  float* sums;                           // forward, over more than kSumKeys keys: [batch, heads, queries] rows of 64 or 128
  float* parts;                          // gradient, with `n_parts` > 1: a part's dk, then dv, of [batch, keys, kv_heads] rows of 64 or 128
  int n_parts, part_heads;               // blocks that share a key tile, query heads of each
  float2* row_sizes;                     // gradient, half, tiles of 128 queries of a head: |d_out|, then |d_out| |out|; zeros where nothing is seen
  float* value_sizes;                    // gradient, half, [batch, keys, kv_heads]: |v|
  const int *lengths, *prefix, *qdoc, *kdoc;   // (kdoc without qdoc: a query has the document of the key at its position)
  const float* slopes;
  unsigned int* status;
  int B, S, T, H, HK, D, group, mask;
  int ld;                                // elements from one head of a row to the next: D, or more in padded copies
  float scale, cap, over;                // over: scale / cap
  Divisor all_heads, heads, all_key_heads, key_heads, per_key_head, parts_of;    // of a block's number: B H, H, B HK, HK, H / HK, n_parts
};

// The tensor cores cut an accumulation off instead of rounding it: some 2^-22 for 16 keys, 0.7 % over a million of them where all
// products have one sign.  So after this many keys the accumulators are added to sums in memory and start again: 2^-13 at most.
constexpr int kSumKeys = 16384;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnRow {
  int pos, last, doc;
};

// a sequence's number of keys, and its prefix (0: none)
struct AttnSeq {
  int len, prefix;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, int b) {
  AttnSeq s;
  s.len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  s.prefix = a.mask == B200_MASK_PREFIX ? max(a.prefix[b], 0) : 0;
  return s;
}
// the last key that query r sees, documents aside: never less than that of the query before
__device__ __forceinline__ int attn_last(const AttnArgs& a, const AttnSeq& s, int r) {
  const int last = a.mask == B200_MASK_NONE ? s.len - 1 : min(s.len - 1, max(s.len - a.S + r, s.prefix - 1));
  return max(last, -1);
}
// a sequence's queries' documents: their entries, or those of the keys at their positions (none before the first position)
struct AttnQueryDocs {
  const int* at;
  int first;
  __device__ __forceinline__ AttnQueryDocs(const AttnArgs& a, const AttnSeq& s, int b)
      : at(a.qdoc ? a.qdoc + (long long)b * a.S : a.kdoc + ((long long)b * a.T + s.len - a.S)), first(a.qdoc ? 0 : a.S - s.len) {}
  __device__ __forceinline__ int of(int r) const { return r >= first ? __ldg(at + r) : -1; }
};
__device__ __forceinline__ AttnRow attn_row(const AttnArgs& a, int b, int r) {
  const AttnSeq s = attn_seq(a, b);
  AttnRow w;
  w.pos = s.len - a.S + r;
  w.last = attn_last(a, s, r);
  w.doc = 0;
  if (a.kdoc) {
    w.doc = AttnQueryDocs(a, s, b).of(r);
    if (w.doc < 0) w.last = -1;
  }
  return w;
}

__device__ __forceinline__ long long attn_q_at(const AttnArgs& a, int b, int r, int h) { return (((long long)b * a.S + r) * a.H + h) * a.ld; }
__device__ __forceinline__ long long attn_k_at(const AttnArgs& a, int b, int j, int hk) { return (((long long)b * a.T + j) * a.HK + hk) * a.ld; }

// The score in units of log 2, of x = <q, k> (not scaled yet); `th` receives tanh(x scale / cap).
__device__ __forceinline__ float attn_score(const AttnArgs& a, float x, float slope2, int pos, int j, float& th) {
  float s;
  if (a.cap > 0.f) {
    th = tanhf(x * a.over);
    s = th * (a.cap * kLog2e);
  } else {
    th = 0.f;
    s = x * (a.scale * kLog2e);
  }
  return fmaf(-slope2, fabsf((float)(pos - j)), s);
}

// Gradients of half heads have weights times 2^14, which their results give back: p is at most 1, and about 1 / keys in long rows (at a
// million keys a half has four bits of it, and dv was 1.4 % off).  The factor comes with the statistics: lse less 14.
template <class T>
constexpr float kWeightLog = std::is_same<T, __half>::value ? 14.f : 0.f;
template <class T>
constexpr float kWeightBack = std::is_same<T, __half>::value ? 1.f / 16384.f : 1.f;

// Where a row's statistics lie: its lse (of 16-bit heads in log 2 units, less kWeightLog; +infinity for a row that sees nothing: all weights are zero), 128 further <d_out, out>
__device__ __forceinline__ long long attn_stat_at(const AttnArgs& a, int b, int h, int r) {
  return (((long long)b * a.H + h) * ((a.S + 127) / 128) + (r >> 7)) * 256 + (r & 127);
}

// the lse of a row's statistics as it was given (or +infinity)
template <class T>
__device__ __forceinline__ float attn_lse_of(float stat) {
  if constexpr (std::is_same<T, float>::value) return stat;
  return (stat + kWeightLog<T>) * kLn2;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- one row by one warp.  Only what the row sees is read: these are right whatever the rest holds, and the tensor-core kernels
// hand them the rows that come out infinite or undefined (0 times infinity from a key that is not seen).  Elements lane,
// lane + 32, .. of a head, four at most.
template <class T>
__device__ __forceinline__ void attn_load_row(const AttnArgs& a, const void* p, long long at, unsigned int lane, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (int)lane + 32 * i < a.D ? to_float(((const T*)p)[at + lane + 32 * i]) : 0.f;
}
template <class T>
__device__ __forceinline__ void attn_store_row(const AttnArgs& a, void* p, long long at, unsigned int lane, const float (&v)[4], float by) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if ((int)lane + 32 * i < a.D) from_float(v[i] * by, ((T*)p)[at + lane + 32 * i]);
}
__device__ __forceinline__ float attn_dot(const float (&x)[4], const float (&y)[4]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(x[i], y[i], s);
  return warp_sum(s);
}

// Whether some lane's part of a row has to be done again; what the lanes have written of it lies behind (a vote alone orders no memory).
__device__ __forceinline__ bool attn_again(bool fine) {
  const bool again = __any_sync(0xffffffffu, !fine);
  __syncwarp();
  return again;
}

template <class T>
__device__ __noinline__ void attn_forward_row(const AttnArgs& a, int b, int h, int r, unsigned int lane) {
  const AttnRow w = attn_row(a, b, r);
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  const int hk = h / a.group;
  float q[4], k[4], v[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f, th;
  attn_load_row<T>(a, a.q, attn_q_at(a, b, r, h), lane, q);
  for (int j = 0; j <= w.last; ++j) {
    if (a.kdoc && a.kdoc[(long long)b * a.T + j] != w.doc) continue;
    const long long at = attn_k_at(a, b, j, hk);
    attn_load_row<T>(a, a.k, at, lane, k);
    attn_load_row<T>(a, a.v, at, lane, v);
    const float s = attn_score(a, attn_dot(q, k), slope2, w.pos, j, th);
    const float top = fmaxf(m, s);
    const float c = top == -INFINITY ? 1.f : exp2f(m - top), p = s == -INFINITY ? 0.f : exp2f(s - top);
    l = fmaf(l, c, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(o[i], c, p * v[i]);
    m = top;
  }
  attn_store_row<T>(a, a.out, attn_q_at(a, b, r, h), lane, o, l > 0.f || l != l ? 1.f / l : 0.f);
  if (a.lse && lane == 0) a.lse[((long long)b * a.H + h) * a.S + r] = (m + log2f(l)) * kLn2;
}

// p and dx of one pair, from the dot products <q, k> and <d_out, v>.  Score and lse meet in their own unit, where their difference is all but
// exact: each rounded in units of log 2 first, scores of 30 cost a third of p's accuracy in single precision.
__device__ __forceinline__ void attn_pair(const AttnArgs& a, float qk, float dov, float slope, int pos, int j, float lse, float delta, float& p, float& dx) {
  float th = 0.f, s;
  if (a.cap > 0.f) {
    th = tanhf(qk * a.over);
    s = th * a.cap;
  } else {
    s = qk * a.scale;
  }
  p = exp2f((fmaf(-slope, fabsf((float)(pos - j)), s) - lse) * kLog2e);
  dx = p * (dov - delta) * a.scale;
  if (a.cap > 0.f) dx *= 1.f - th * th;
}

template <class T>
__device__ __noinline__ void attn_dq_row(const AttnArgs& a, int b, int h, int r, unsigned int lane) {
  const AttnRow w = attn_row(a, b, r);
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  const int hk = h / a.group;
  const long long at = attn_q_at(a, b, r, h), stat = attn_stat_at(a, b, h, r);
  const float lse = attn_lse_of<T>(a.stat[stat]), delta = a.stat[stat + 128];
  float q[4], k[4], v[4], go[4], g[4] = {0.f, 0.f, 0.f, 0.f}, p, dx;
  attn_load_row<T>(a, a.q, at, lane, q);
  attn_load_row<T>(a, a.d_out, at, lane, go);
  for (int j = 0; j <= w.last; ++j) {
    if (a.kdoc && a.kdoc[(long long)b * a.T + j] != w.doc) continue;
    const long long kat = attn_k_at(a, b, j, hk);
    attn_load_row<T>(a, a.k, kat, lane, k);
    attn_load_row<T>(a, a.v, kat, lane, v);
    attn_pair(a, attn_dot(q, k), attn_dot(go, v), slope, w.pos, j, lse, delta, p, dx);
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = fmaf(dx, k[i], g[i]);
  }
  attn_store_row<T>(a, a.dq, at, lane, g, 1.f);
}

// which: 1 the key's gradient, 2 the value's, 3 both
template <class T>
__device__ __noinline__ void attn_dkv_row(const AttnArgs& a, int b, int hk, int j, unsigned int lane, int which) {
  const long long kat = attn_k_at(a, b, j, hk);
  const int doc = a.kdoc ? a.kdoc[(long long)b * a.T + j] : 0;
  float q[4], k[4], v[4], go[4], gk[4] = {0.f, 0.f, 0.f, 0.f}, gv[4] = {0.f, 0.f, 0.f, 0.f}, p, dx;
  attn_load_row<T>(a, a.k, kat, lane, k);
  attn_load_row<T>(a, a.v, kat, lane, v);
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    for (int r = 0; r < a.S; ++r) {
      const AttnRow w = attn_row(a, b, r);
      if (j > w.last || (a.kdoc && doc != w.doc)) continue;
      const long long at = attn_q_at(a, b, r, h), stat = attn_stat_at(a, b, h, r);
      attn_load_row<T>(a, a.q, at, lane, q);
      attn_load_row<T>(a, a.d_out, at, lane, go);
      attn_pair(a, attn_dot(q, k), attn_dot(go, v), slope, w.pos, j, attn_lse_of<T>(a.stat[stat]), a.stat[stat + 128], p, dx);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gk[i] = fmaf(dx, q[i], gk[i]);
        gv[i] = fmaf(p, go[i], gv[i]);
      }
    }
  }
  if (which & 1) attn_store_row<T>(a, a.dk, kat, lane, gk, 1.f);
  if (which & 2) attn_store_row<T>(a, a.dv, kat, lane, gv, 1.f);
}

}  // namespace b200
#endif
