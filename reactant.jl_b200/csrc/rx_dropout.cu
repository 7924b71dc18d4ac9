// Dropout with a mask that is never stored.
#include "rx_device.cuh"
#include "rx_token.h"

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

// Element i of the array has 16 bits: half i % 2 of word i % 8 / 2 of the counter i / 8; it stays when they reach the
// threshold.  `first`: the index of x[0] (a multiple of nothing in particular: a device's share of a sharded array).
template <bool BF16>
__global__ void __launch_bounds__(kBlock) k_dropout(const void* __restrict__ x, const uint32_t* __restrict__ key, const void* __restrict__ residual, void* __restrict__ out, int64_t n, int64_t first,
                                                    uint32_t threshold, float scale, uint32_t site) {
  const int elem = BF16 ? EL_BF16 : EL_F32;
  const uint32_t k0 = key[0], k1 = key[1];
  const int64_t g0 = first >> 3, groups = ((first + n + 7) >> 3) - g0, step = (int64_t)gridDim.x * kBlock;
  for (int64_t g = (int64_t)blockIdx.x * kBlock + threadIdx.x; g < groups; g += step) {
    const uint64_t counter = (uint64_t)(g0 + g);
    const uint4 r = philox((uint32_t)counter, (uint32_t)(counter >> 32), site, 0, k0, k1);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int64_t i = (g0 + g) * 8 + q - first;
      if (i < 0 || i >= n) continue;
      const uint32_t bits = (w[q / 2] >> (16 * (q & 1))) & 0xFFFFu;
      const float v = u2f(load_elem(x, i, elem)), add = residual ? u2f(load_elem(residual, i, elem)) : 0.f;
      const float y = bits >= threshold ? (residual ? fmaf(v, scale, add) : v * scale) : add;
      store_elem(out, i, elem, f2u(y));
    }
  }
}

}  // namespace

cudaError_t launch_dropout(const LaunchCtx& c, const CallDesc& d, const void* x, const void* key, const void* residual, void* out, int64_t first) {
  const int64_t n = d.rows * d.cols;
  if (!n) return cudaSuccess;
  const int64_t threshold = dropout_threshold(d.rate);
  const float scale = (float)(65536.0 / (65536.0 - (double)threshold));
  const int64_t blocks = std::min<int64_t>((n / 8 + 2 + kBlock - 1) / kBlock, (int64_t)c.sm_count * 8);
  auto* f = d.in_dt == DT::BF16 ? k_dropout<true> : k_dropout<false>;
  f<<<(unsigned)blocks, kBlock, 0, c.stream>>>(x, (const uint32_t*)key, residual, out, n, first, (uint32_t)threshold, scale, (uint32_t)d.site);
  ++*c.launches;
  return cudaGetLastError();
}

}  // namespace rx
