// Element access shared by the operators' kernels: values travel as floats, 16-bit types are rounded once, to nearest, when
// they are stored.
#ifndef B200_OP_COMMON_CUH
#define B200_OP_COMMON_CUH
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace b200 {

__device__ __forceinline__ void grid_begin() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half_rn(v); }

// two values packed to 16 bits each, the first in the low half
__device__ __forceinline__ unsigned int pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *(const unsigned int*)&v;
}
__device__ __forceinline__ unsigned int pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *(const unsigned int*)&v;
}
__device__ __forceinline__ float2 unpack2(unsigned int w, __nv_bfloat16) { return __bfloat1622float2(*(const __nv_bfloat162*)&w); }
__device__ __forceinline__ float2 unpack2(unsigned int w, __half) { return __half22float2(*(const __half2*)&w); }

// VEC elements: one 16-byte access, or a single element
template <class T, int VEC>
struct Vec {
  static_assert(VEC == 1 || VEC * sizeof(T) == 16, "16 bytes or one element");
  static __device__ __forceinline__ void load(const T* p, float* v) {
    if constexpr (VEC == 1) {
      v[0] = to_float(*p);
    } else if constexpr (sizeof(T) == 4) {
      const float4 q = *(const float4*)p;
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const uint4 q = *(const uint4*)p;
      const unsigned int w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(w[i], T());
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float* v) {
    if constexpr (VEC == 1) {
      from_float(v[0], *p);
    } else if constexpr (sizeof(T) == 4) {
      *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      *(uint4*)p = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    }
  }
};

// Pairs of single-precision values in one instruction (the multiply-add pipe takes both in the issue slot of one).
struct Pair {
  unsigned long long v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Pair fma2(const Pair& a, const Pair& b, const Pair& c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair mul2(const Pair& a, const Pair& b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair add2(const Pair& a, const Pair& b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// The same access in two steps, so that a load can be under way while other work is done.
template <class T, int VEC>
struct Raw {
  typename std::conditional<VEC == 1, T, uint4>::type r;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) r = *p;
    else r = *(const uint4*)p;
  }
  __device__ __forceinline__ void clear() {
    if constexpr (VEC == 1) from_float(0.f, r);
    else r = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void values(float* v) const {
    if constexpr (VEC == 1) {
      v[0] = to_float(r);
    } else {
      const unsigned int w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          v[i] = __uint_as_float(w[i]);
        } else {
          const float2 f = unpack2(w[i], T());
          v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
      }
    }
  }
};

// Quotients by a number known at link (1 <= d < 2^31), for numerators below 2^31: one multiplication and a shift.
// With s = ceil(log2 d) and m = ceil(2^(31 + s) / d), floor(n m / 2^(31 + s)) is the quotient: m d exceeds 2^(31 + s) by less than 2^s.
struct Divisor {
  unsigned int d, m, s;
  Divisor() : d(1), m(0x80000000u), s(0) {}
  explicit Divisor(unsigned int by) : d(by), m(0), s(0) {
    while ((1ull << s) < by) ++s;
    m = (unsigned int)(((1ull << (31 + s)) + by - 1) / by);
  }
  __device__ __forceinline__ unsigned int of(unsigned int n) const { return (unsigned int)(((unsigned long long)n * m) >> (31 + s)); }
};

}  // namespace b200
#endif
