// Embedding lookup and its gradient.
#include "rx_device.cuh"
#include "rx_token.h"

namespace rx {

namespace {

constexpr int kBlock = 256;

template <class T>
__device__ __forceinline__ float as_float(T v) { return v; }
template <>
__device__ __forceinline__ float as_float<uint16_t>(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = bf16_bits(v); }

// out[t][c] = scale * table[ids[t]][c]; a token outside the table is a row of zeros
template <class In, class Out, class Id>
__global__ void __launch_bounds__(kBlock) k_embedding(const In* __restrict__ table, const Id* __restrict__ ids, Out* __restrict__ out, int64_t rows, int64_t cols, int64_t ld, int64_t vocab,
                                                      float scale) {
  const int64_t n = rows * cols, step = (int64_t)gridDim.x * kBlock;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += step) {
    const int64_t t = i / cols, c = i - t * cols;
    const int64_t id = ids[t];
    put(out + i, id >= 0 && id < vocab ? scale * as_float(table[id * ld + c]) : 0.f);
  }
}

// Stable counting of the tokens by id, 8 bits at a time: one CTA, each thread a contiguous piece of the tokens.
// keys/pos: two buffers of `rows` each; a token outside the table gets the key `vocab`.
template <class Id>
__global__ void __launch_bounds__(kBlock) k_sort_tokens(const Id* __restrict__ ids, int64_t rows, int64_t vocab, int passes, int32_t* keys0, int32_t* pos0, int32_t* keys1, int32_t* pos1) {
  __shared__ int32_t start[256];
  const int64_t per = (rows + kBlock - 1) / kBlock, lo = min(rows, per * threadIdx.x), hi = min(rows, lo + per);
  for (int64_t t = lo; t < hi; ++t) {
    const int64_t id = ids[t];
    keys0[t] = id >= 0 && id < vocab ? (int32_t)id : (int32_t)vocab;
    pos0[t] = (int32_t)t;
  }
  __syncthreads();
  int32_t *k0 = keys0, *p0 = pos0, *k1 = keys1, *p1 = pos1;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = 8 * pass;
    start[threadIdx.x] = 0;
    __syncthreads();
    for (int64_t t = lo; t < hi; ++t) atomicAdd(&start[(k0[t] >> shift) & 255], 1);
    __syncthreads();
    if (threadIdx.x == 0) {
      int32_t sum = 0;
      for (int b = 0; b < 256; ++b) {
        const int32_t n = start[b];
        start[b] = sum;
        sum += n;
      }
    }
    __syncthreads();
    for (int who = 0; who < kBlock; ++who) {  // in the order of the tokens
      if (threadIdx.x == who)
        for (int64_t t = lo; t < hi; ++t) {
          const int32_t at = start[(k0[t] >> shift) & 255]++;
          k1[at] = k0[t];
          p1[at] = p0[t];
        }
      __syncthreads();
    }
    int32_t* x = k0; k0 = k1; k1 = x;
    x = p0; p0 = p1; p1 = x;
  }
}

// One CTA per row of the table: its tokens by bisection, their gradients added in the order of the tokens.
template <class In, class Out>
__global__ void __launch_bounds__(kBlock) k_embedding_grad(const In* __restrict__ dy, const int32_t* __restrict__ keys, const int32_t* __restrict__ pos, Out* __restrict__ out, int64_t rows, int64_t cols,
                                                           int64_t ld, float scale) {
  const int32_t v = blockIdx.x;
  auto first = [&](int32_t key) {
    int64_t lo = 0, hi = rows;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (keys[mid] < key) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  const int64_t b = first(v), e = first(v + 1);
  for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
    float sum = 0;
    for (int64_t q = b; q < e; ++q) sum += as_float(dy[(int64_t)pos[q] * ld + c]);
    put(out + (int64_t)v * cols + c, scale * sum);
  }
}

int sort_passes(int64_t vocab) {
  int passes = 1;
  while (passes < 4 && (vocab >> (8 * passes))) ++passes;
  return passes;
}

// calls f with null pointers of the types that the three element types stand for
template <class F>
void with_types(DT in, DT out, DT ids, F f) {
  auto by_id = [&](auto* i, auto* o) {
    if (ids == DT::S64) f(i, o, (int64_t*)nullptr);
    else f(i, o, (int32_t*)nullptr);
  };
  auto by_out = [&](auto* i) {
    if (out == DT::BF16) by_id(i, (uint16_t*)nullptr);
    else by_id(i, (float*)nullptr);
  };
  if (in == DT::BF16) by_out((uint16_t*)nullptr);
  else by_out((float*)nullptr);
}

}  // namespace

cudaError_t launch_embedding(const LaunchCtx& c, const CallDesc& d, const void* table, const void* ids, void* out) {
  const int64_t n = d.rows * d.cols;
  if (!n) return cudaSuccess;
  const int64_t blocks = std::min<int64_t>((n + kBlock - 1) / kBlock, (int64_t)c.sm_count * 8);
  with_types(d.in_dt, d.out_dt, d.ids_dt, [&](auto* i, auto* o, auto* id) {
    k_embedding<<<(unsigned)blocks, kBlock, 0, c.stream>>>((decltype(i))table, (decltype(id))ids, (decltype(o))out, d.rows, d.cols, d.ld, d.vocab, (float)d.scale);
  });
  ++*c.launches;
  return cudaGetLastError();
}

int64_t embedding_grad_workspace(const CallDesc& d, int) { return 4 * d.rows * (int64_t)sizeof(int32_t); }

cudaError_t launch_embedding_grad(const LaunchCtx& c, const CallDesc& d, const void* dy, const void* ids, void* out, void* workspace) {
  if (d.vocab * d.cols == 0) return cudaSuccess;
  int32_t* w = (int32_t*)workspace;
  int32_t *k0 = w, *p0 = w + d.rows, *k1 = w + 2 * d.rows, *p1 = w + 3 * d.rows;
  const int passes = sort_passes(d.vocab);
  with_types(d.in_dt, d.out_dt, d.ids_dt, [&](auto* i, auto* o, auto* id) {
    if (d.rows) {
      k_sort_tokens<<<1, kBlock, 0, c.stream>>>((decltype(id))ids, d.rows, d.vocab, passes, k0, p0, k1, p1);
      ++*c.launches;
    }
    k_embedding_grad<<<(unsigned)d.vocab, kBlock, 0, c.stream>>>((decltype(i))dy, passes % 2 ? k1 : k0, passes % 2 ? p1 : p0, (decltype(o))out, d.rows, d.cols, d.ld, (float)d.scale);
  });
  ++*c.launches;
  return cudaGetLastError();
}

}  // namespace rx
