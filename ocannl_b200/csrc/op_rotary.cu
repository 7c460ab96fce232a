// Rotary positions: pair i of a head at position p turns by the angle p * f_i.
//
//   (a, b) -> m (a cos - b sin, a sin + b cos);   inverse: the angle negated, which is also the gradient (the turn is orthogonal)
//
// Bound by memory: every element is read and written once.  The angle is kept as a 64-bit fraction of a turn: f_i / 2 pi as a
// fixed-point number, times the position in wrapping integer arithmetic, is the angle modulo a turn without any loss at far
// positions (2^31 positions: 2^-33 of a turn); its upper 32 bits go to sincospif.  A block takes a few tokens: their cosines and
// sines are made once, in shared memory, for all heads of both tensors.  (64 x 256 x 16 heads of 64, bf16: 14.4 us, 4.7 TB/s: 1024 blocks, of
// which 444 fit the machine at a time, so that three rounds are paid for 2.3, and each begins with its table and first loads.)
#include <cmath>

#include "kernels/op_common.cuh"
#include "operators.hpp"

using namespace b200;

namespace {

struct RotaryArgs {
  const void* x[2];
  void* y[2];
  const int* positions;
  const unsigned long long* turns;     // [pairs], of a turn per position, scaled by 2^64
  unsigned long long tokens, seq;
  long long first_position;
  unsigned int heads[2], d, pairs;
  unsigned int per_block;              // tokens
  unsigned int turn_items, items;      // of a head: accesses that turn, all accesses
  Divisor by_pairs, by_items, by_heads;
  float magnitude;
  int inverse;
};

constexpr int kAtOnce = 4;             // accesses of a thread under way together

template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary(const RotaryArgs a) {
  extern __shared__ float2 table[];    // [token][pair]: cosine, sine, times the magnitude
  grid_begin();
  const unsigned long long first = (unsigned long long)blockIdx.x * a.per_block;
  const unsigned int n = (unsigned int)min((unsigned long long)a.per_block, a.tokens - first);
  const unsigned int heads = a.heads[0] + a.heads[1], total = n * heads * a.items;
  // One access: where it lies, and its elements.  Half pairs have their second elements `pairs` further.
  struct Item {
    T* y;
    const T* x;
    unsigned int tok, item;
    Raw<T, VEC> u, v;
  } it[kAtOnce];
  auto fetch = [&](unsigned int i, Item& t) {
    if (i >= total) return;
    const unsigned int row = a.by_items.of(i), tok = a.by_heads.of(row), head = row - tok * heads;
    t.item = i - row * a.items;
    t.tok = tok;
    const bool second = head >= a.heads[0];
    const unsigned long long at = ((first + tok) * a.heads[second] + (second ? head - a.heads[0] : head)) * a.d;
    unsigned int e;
    if (t.item >= a.turn_items) e = 2 * a.pairs + (t.item - a.turn_items) * VEC;
    else e = INTERLEAVED && VEC == 1 ? 2 * t.item : t.item * VEC;
    t.x = (const T*)a.x[second] + at + e;
    t.y = (T*)a.y[second] + at + e;
    t.u.load(t.x);
    if (t.item < a.turn_items) {
      if constexpr (!INTERLEAVED) t.v.load(t.x + a.pairs);
      else if constexpr (VEC == 1) t.v.load(t.x + 1);
    }
  };
  // the first accesses are under way while the table is made
#pragma unroll
  for (int k = 0; k < kAtOnce; ++k) fetch(threadIdx.x + 256 * k, it[k]);
  for (unsigned int i = threadIdx.x; i < n * a.pairs; i += 256) {
    const unsigned int tok = a.by_pairs.of(i), pair = i - tok * a.pairs;
    const unsigned long long t = first + tok;
    const long long p = a.positions ? (long long)a.positions[t] : a.first_position + (long long)(t % a.seq);
    unsigned long long turn = (unsigned long long)p * a.turns[pair];
    if (a.inverse) turn = 0ull - turn;
    // the nearest of 2^32 steps of a turn, as a signed number: the angle is step * 2 pi / 2^32
    const int step = (int)(unsigned int)((turn + 0x80000000ull) >> 32);
    float s, c;
    sincospif((float)step * 4.656612873077393e-10f, &s, &c);
    table[i] = make_float2(c * a.magnitude, s * a.magnitude);
  }
  __syncthreads();
  for (unsigned int base = 0; base < total; base += 256 * kAtOnce) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const unsigned int i = base + threadIdx.x + 256 * k;
      if (i >= total) continue;
      const Item& t = it[k];
      if (t.item >= a.turn_items) {          // elements that do not turn
        if constexpr (VEC == 1) *t.y = t.u.r;
        else *(uint4*)t.y = t.u.r;
        continue;
      }
      const float2* cs = table + t.tok * a.pairs;
      float u[VEC], v[VEC];
      t.u.values(u);
      if constexpr (INTERLEAVED && VEC > 1) {
#pragma unroll
        for (int q = 0; q < VEC / 2; ++q) {
          const float2 w = cs[t.item * (VEC / 2) + q];
          v[2 * q] = u[2 * q] * w.x - u[2 * q + 1] * w.y;
          v[2 * q + 1] = u[2 * q] * w.y + u[2 * q + 1] * w.x;
        }
        Vec<T, VEC>::store(t.y, v);
      } else {
        t.v.values(v);
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const float2 w = cs[t.item * VEC + q];
          const float u0 = u[q], u1 = v[q];
          u[q] = u0 * w.x - u1 * w.y;
          v[q] = u0 * w.y + u1 * w.x;
        }
        Vec<T, VEC>::store(t.y, u);
        Vec<T, VEC>::store(INTERLEAVED ? t.y + 1 : t.y + a.pairs, v);
      }
    }
    if (base + 256 * kAtOnce < total)
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) fetch(base + 256 * (kAtOnce + k) + threadIdx.x, it[k]);
  }
}

typedef void (*RotaryKernel)(const RotaryArgs);

template <class T>
RotaryKernel kernel_of(bool vec, bool interleaved) {
  constexpr int V = 16 / (int)sizeof(T);
  if (vec) return interleaved ? rotary<T, V, true> : rotary<T, V, false>;
  return interleaved ? rotary<T, 1, true> : rotary<T, 1, false>;
}

struct RotaryOperator : b200_operator {
  RotaryArgs a = {};
  RotaryKernel kernel = nullptr;
  unsigned long long grid = 0;
  size_t smem = 0;
  void run(cudaStream_t s) override {
    if (grid) launch(kernel, dim3((unsigned int)grid), 256, smem, s, a);
  }
};

}  // namespace

extern "C" int b200_rotary_link(b200_dev* dev, const b200_rotary* p, b200_operator** out) {
  return link_operator<RotaryOperator>(dev, p, out, [&](RotaryOperator* op) {
    Operands ops(op, "rotary");
    ops.dtype(p->dtype);
    if (p->heads[0] < 1 || p->heads[1] < 0 || p->heads[0] > (1 << 20) || p->heads[1] > (1 << 20)) ops.refuse("heads must be between 1 and 2^20 (the second tensor's may be 0)");
    if (p->d < 1 || p->d > (1 << 16) || p->pairs < 0 || 2ll * p->pairs > p->d) ops.refuse("2 * pairs must not exceed d, d must be between 1 and 65536");
    if (p->pairs > 4096) ops.refuse("more than 4096 pairs", B200_E_UNSUPPORTED);
    if (p->pairs && !p->frequencies) ops.refuse("'frequencies' is required");
    if (!std::isfinite(p->magnitude)) ops.refuse("the magnitude must be finite");
    for (int i = 0; i < p->pairs; ++i)
      if (!std::isfinite(p->frequencies[i])) ops.refuse("a frequency is not finite");
    RotaryArgs& a = op->a;
    const size_t size = dtype_bytes(p->dtype);
    const unsigned long long tokens = extent_product({p->batch, p->seq}, "rotary");
    bool vec = (size_t)p->d * size % 16 == 0;
    for (int i = 0; i < 2; ++i) {
      a.heads[i] = (unsigned int)p->heads[i];
      if (!p->heads[i]) continue;
      const unsigned long long count = extent_product({p->batch, p->seq, p->heads[i], p->d}, "rotary");
      a.x[i] = (const void*)ops.in(p->x[i], i ? "x[1]" : "x[0]", count, size);
      a.y[i] = (void*)ops.out(p->y[i], i ? "y[1]" : "y[0]", count, size);
      vec &= ((size_t)a.x[i] & 15) == 0 && ((size_t)a.y[i] & 15) == 0;
    }
    a.positions = (const int*)ops.in(p->positions, "positions", tokens, 4, false);
    ops.check_overlaps({{"y[0]", "x[0]"}, {"y[1]", "x[1]"}});
    a.tokens = tokens;
    a.seq = (unsigned long long)p->seq;
    a.first_position = p->first_position;
    a.d = (unsigned int)p->d;
    a.pairs = (unsigned int)p->pairs;
    a.magnitude = p->magnitude;
    a.inverse = p->inverse != 0;
    const unsigned int V = 16 / (unsigned int)size;
    vec &= p->interleaved ? 2 * a.pairs % V == 0 : a.pairs % V == 0;
    const unsigned int v = vec ? V : 1;
    a.turn_items = p->interleaved ? (vec ? 2 * a.pairs / v : a.pairs) : a.pairs / v;
    a.items = a.turn_items + (a.d - 2 * a.pairs) / v;
    // About four accesses a thread, while that leaves the machine enough blocks; a table of at most 32 KB
    const unsigned long long per_token = (unsigned long long)(a.heads[0] + a.heads[1]) * a.items;
    unsigned long long tok = std::max(1ull, 1024ull / per_token);
    tok = std::min(tok, std::max(1ull, tokens / (2ull * (unsigned)dev->sm_count)));
    if (a.pairs) tok = std::min(tok, std::max(1ull, 4096ull / a.pairs));
    a.by_pairs = Divisor(std::max(1u, a.pairs));
    a.by_items = Divisor(a.items);
    a.by_heads = Divisor(a.heads[0] + a.heads[1]);
    if (tok * per_token >> 31) ops.refuse("a token has too many elements", B200_E_UNSUPPORTED);
    a.per_block = (unsigned int)tok;
    op->grid = (tokens + tok - 1) / tok;
    if (op->grid >> 31) ops.refuse("too many tokens", B200_E_UNSUPPORTED);
    op->smem = (size_t)tok * a.pairs * 8;
    op->kernel = p->dtype == B200_F32 ? kernel_of<float>(vec, p->interleaved) : p->dtype == B200_BF16 ? kernel_of<__nv_bfloat16>(vec, p->interleaved) : kernel_of<__half>(vec, p->interleaved);
    ready(op->kernel);
    if (!a.pairs) return;
    op->take_workspace((size_t)a.pairs * 8);
    write_turns(op, op->workspace, p->frequencies, p->pairs);
    a.turns = (const unsigned long long*)op->workspace;
  });
}
