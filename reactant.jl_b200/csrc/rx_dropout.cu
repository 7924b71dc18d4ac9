// Dropout with a mask that is never stored: a kept element is scaled by 65536 / (65536 - threshold), the mask is a
// function of the key, the site and the element's index, and so the same call on a gradient is the gradient.
#include "rx_token.cuh"
#include "rx_token.h"

#include <algorithm>

namespace rx {

namespace {

constexpr int kBlock = 256;

// Philox4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror and D. Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011): four words of 32 random bits from a counter of four words and a key of two.
__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The bits of element i are half i % 2 of word i % 8 / 2 of the counter i / 8, low halves first.  Sixteen bits an
// element, not thirty-two: one evaluation of the generator (about 80 instructions) covers eight elements, a third of
// what the SMs can issue while the memory moves them; a word each would make bf16 instruction-bound.
__device__ __forceinline__ uint32_t bits_of(const uint4& r, int q) {
  const uint32_t w = q < 2 ? r.x : q < 4 ? r.y : q < 6 ? r.z : r.w;
  return q & 1 ? w >> 16 : w & 0xFFFFu;
}

struct DropoutArgs {
  int64_t n, first;  // elements, and the index of x[0] in the array all devices hold together
  uint32_t threshold, site;
  float scale;
};

template <class T, bool RES>
__device__ __forceinline__ void dropout_one(const T* x, const T* residual, T* out, int64_t i, const uint4& r, int q, const DropoutArgs& a) {
  const float v = widen(x[i]), add = RES ? widen(residual[i]) : 0.f;
  put(out + i, bits_of(r, q) >= a.threshold ? (RES ? fmaf(v, a.scale, add) : v * a.scale) : add);
}

// Bound by memory: 16384 x 4096 bf16 with a residual take 61.5 us, 403 MB at 6.55 TB/s, the rate of a plain copy (one
// element at a time: 202 us).  A thread takes kGroups groups of eight elements, a block apart, and asks for all of them before it
// computes: vectors are 16 bytes a lane.  VEC: the arrays start on 16 bytes and on a group; otherwise, and for a last
// group that is not whole, elements are read one by one.
template <class T, bool RES, bool VEC>
__global__ void __launch_bounds__(kBlock) k_dropout(const T* __restrict__ x, const uint32_t* __restrict__ key, const T* __restrict__ residual, T* __restrict__ out, DropoutArgs a) {
  constexpr int kGroups = RES ? 2 : 4;
  const uint32_t k0 = __ldg(key), k1 = __ldg(key + 1);
  const int64_t g0 = a.first >> 3, groups = ((a.first + a.n + 7) >> 3) - g0;
  const int64_t base = (int64_t)blockIdx.x * (kBlock * kGroups) + threadIdx.x;
  Raw8<T> rx_[kGroups], rr[kGroups];
  if (VEC) {
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      const int64_t g = base + k * kBlock;
      if ((g + 1) * 8 <= a.n) {
        rx_[k] = load8(x + g * 8);
        if (RES) rr[k] = load8(residual + g * 8);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const int64_t g = base + k * kBlock;
    if (g >= groups) break;
    const uint64_t counter = (uint64_t)(g0 + g);
    const uint4 r = philox((uint32_t)counter, (uint32_t)(counter >> 32), a.site, 0, k0, k1);
    if (VEC && (g + 1) * 8 <= a.n) {
      float v[8], add[8];
      widen8(rx_[k], v);
      if (RES) widen8(rr[k], add);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const bool keep = bits_of(r, q) >= a.threshold;
        v[q] = keep ? (RES ? fmaf(v[q], a.scale, add[q]) : v[q] * a.scale) : (RES ? add[q] : 0.f);
      }
      store8(out + g * 8, v);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int64_t i = (g0 + g) * 8 + q - a.first;
        if (i >= 0 && i < a.n) dropout_one<T, RES>(x, residual, out, i, r, q, a);
      }
    }
  }
}

template <class T>
void launch(const LaunchCtx& c, const void* x, const void* key, const void* residual, void* out, const DropoutArgs& a) {
  const bool vec = a.first % 8 == 0 && aligned16(x) && aligned16(out) && aligned16(residual);
  const int64_t groups = ((a.first + a.n + 7) >> 3) - (a.first >> 3), per = kBlock * (residual ? 2 : 4);
  const unsigned blocks = (unsigned)((groups + per - 1) / per);
  auto* f = residual ? (vec ? k_dropout<T, true, true> : k_dropout<T, true, false>) : (vec ? k_dropout<T, false, true> : k_dropout<T, false, false>);
  f<<<blocks, kBlock, 0, c.stream>>>((const T*)x, (const uint32_t*)key, (const T*)residual, (T*)out, a);
}

}  // namespace

cudaError_t launch_dropout(const LaunchCtx& c, const CallDesc& d, const void* x, const void* key, const void* residual, void* out, int64_t first) {
  DropoutArgs a;
  a.n = d.rows * d.cols;
  a.first = first;
  if (!a.n) return cudaSuccess;
  const int64_t threshold = dropout_threshold(d.rate);
  a.threshold = (uint32_t)threshold;
  a.site = (uint32_t)d.site;
  a.scale = (float)(65536.0 / (65536.0 - (double)threshold));
  if (d.in_dt == DT::BF16) launch<uint16_t>(c, x, key, residual, out, a);
  else launch<float>(c, x, key, residual, out, a);
  ++*c.launches;
  return cudaGetLastError();
}

}  // namespace rx
