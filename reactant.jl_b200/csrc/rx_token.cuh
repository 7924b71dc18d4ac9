// Device-side pieces shared by the token-model kernels: eight elements at a time as 32-bit floats, and division by a
// row length known at launch.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "rx_device.cuh"

namespace rx {

// bf16 is handled as its 16-bit pattern throughout
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float2 widen_pair(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = bf16_bits(v); }

// Eight consecutive elements as they lie in memory, and as floats.  Loads and stores bypass or leave L1 early (.cs):
// every one of these operators touches its large operand once.
struct Raw8f { uint4 a, b; };
struct Raw8h { uint4 a; };
template <class T> struct Raw8T;
template <> struct Raw8T<float> { using type = Raw8f; };
template <> struct Raw8T<uint16_t> { using type = Raw8h; };
template <class T> using Raw8 = typename Raw8T<T>::type;

__device__ __forceinline__ Raw8f load8(const float* p) { return {__ldcs((const uint4*)p), __ldcs((const uint4*)p + 1)}; }
__device__ __forceinline__ Raw8h load8(const uint16_t* p) { return {__ldcs((const uint4*)p)}; }
__device__ __forceinline__ Raw8f load8_cached(const float* p) { return {__ldg((const uint4*)p), __ldg((const uint4*)p + 1)}; }
__device__ __forceinline__ Raw8h load8_cached(const uint16_t* p) { return {__ldg((const uint4*)p)}; }
__device__ __forceinline__ void widen8(const Raw8f& r, float (&v)[8]) {
  v[0] = u2f(r.a.x); v[1] = u2f(r.a.y); v[2] = u2f(r.a.z); v[3] = u2f(r.a.w);
  v[4] = u2f(r.b.x); v[5] = u2f(r.b.y); v[6] = u2f(r.b.z); v[7] = u2f(r.b.w);
}
__device__ __forceinline__ void widen8(const Raw8h& r, float (&v)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = __uint_as_float(w[k] << 16);
    v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  __stcs((uint4*)p, make_uint4(f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])));
  __stcs((uint4*)p + 1, make_uint4(f2u(v[4]), f2u(v[5]), f2u(v[6]), f2u(v[7])));
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  __stcs((uint4*)p, make_uint4(bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]), bf16x2_bits(v[4], v[5]), bf16x2_bits(v[6], v[7])));
}

// Eight consecutive elements from any element's boundary: the 16-byte lines that hold them, fetched first and shifted
// into place afterwards, so that several fetches can be in flight.  A line is read whole, up to 15 bytes in front of and
// behind the elements; where that would reach past `end` (of the memory behind the operand) they are read one by one.
template <class T>
struct Lines {
  uint4 w[sizeof(T) == 4 ? 3 : 2];
  int shift;  // elements
  __device__ __forceinline__ void fetch(const T* p, const T* end) {
    const uintptr_t a = (uintptr_t)p;
    shift = (int)(a % 16 / sizeof(T));
    const uint4* line = (const uint4*)(a - a % 16);
    constexpr int kWhole = sizeof(T) == 4 ? 2 : 1;
    if ((uintptr_t)(line + kWhole + (shift ? 1 : 0)) <= (uintptr_t)end) {
#pragma unroll
      for (int k = 0; k < kWhole; ++k) w[k] = __ldg(line + k);
      if (shift) w[kWhole] = __ldg(line + kWhole);
    } else {
      T one[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) one[k] = p + k < end ? __ldg(p + k) : T(0);
      shift = 0;
      if constexpr (sizeof(T) == 4) {
        w[0] = make_uint4(__float_as_uint(one[0]), __float_as_uint(one[1]), __float_as_uint(one[2]), __float_as_uint(one[3]));
        w[1] = make_uint4(__float_as_uint(one[4]), __float_as_uint(one[5]), __float_as_uint(one[6]), __float_as_uint(one[7]));
      } else {
        w[0] = make_uint4(one[0] | (uint32_t)one[1] << 16, one[2] | (uint32_t)one[3] << 16, one[4] | (uint32_t)one[5] << 16, one[6] | (uint32_t)one[7] << 16);
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    constexpr int kWords = sizeof(T) == 4 ? 12 : 8;
    uint32_t x[kWords];
#pragma unroll
    for (int k = 0; k < kWords / 4; ++k) {
      x[4 * k] = w[k].x;
      x[4 * k + 1] = w[k].y;
      x[4 * k + 2] = w[k].z;
      x[4 * k + 3] = w[k].w;
    }
    const int words = sizeof(T) == 4 ? shift : shift >> 1;
#pragma unroll
    for (int k = 0; k + 2 < kWords; ++k)
      if (words & 2) x[k] = x[k + 2];
#pragma unroll
    for (int k = 0; k + 1 < kWords; ++k)
      if (words & 1) x[k] = x[k + 1];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(x[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t y = shift & 1 ? __funnelshift_r(x[k], x[k + 1], 16) : x[k];
        v[2 * k] = __uint_as_float(y << 16);
        v[2 * k + 1] = __uint_as_float(y & 0xFFFF0000u);
      }
    }
  }
};

// The same where the eight elements start on their own size (32 bytes for floats): one store a lane, whole sectors.  Blocks
// of the pool start on 256 bytes, but memory taken over from another library on 16 only: launches ask `whole_stores` first.
__device__ __forceinline__ void store8_whole(float* p, const float (&v)[8]) {
  asm volatile("st.global.cs.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}
__device__ __forceinline__ void store8_whole(uint16_t* p, const float (&v)[8]) { store8(p, v); }

// Quotients of numbers below 2^31 by a fixed divisor with one multiplication (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994): with l = ceil(log2 d) and m = ceil(2^(31 + l) / d), which is below
// 2^32, n / d = (n m) >> (31 + l) for every n < 2^31.
struct Divisor {
  uint32_t d = 0, m = 0;
  int shift = 0;
  Divisor() = default;
  explicit Divisor(int64_t divisor) : d((uint32_t)divisor), m(0), shift(0) {
    if (divisor <= 0 || divisor >= (int64_t)1 << 31) return;  // not used
    int l = 0;
    while (((uint64_t)1 << l) < d) ++l;
    m = (uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d);
    shift = l - 1;
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> shift; }
};

inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
inline bool whole_stores(const void* out, size_t elem_bytes) { return (uintptr_t)out % (8 * elem_bytes) == 0; }

}  // namespace rx
