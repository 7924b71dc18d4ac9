// Embedding lookup and its gradient.
#include "rx_token.cuh"
#include "rx_token.h"

#include <algorithm>

namespace rx {

namespace {

constexpr int kBlock = 256;

// out[t][c] = scale * table[ids[t]][c]; a token outside the table is a row of zeros.
//
// Bound by memory: every distinct row is read, every row of the result written once.  The result is cut into units of
// eight consecutive elements; a thread takes kUnits of them, a block apart, and asks for the ids and then the rows of
// all of them before it stores.  VEC: rows of the table and of the result start on 16 bytes, so a unit is a vector of
// one row.  Otherwise (an odd row length) the elements of a unit are read one by one, from up to eight rows, and still
// leave as one vector.  65536 tokens of 2048 bf16 features: 72.9 us (one element a thread and a 64-bit division each: 361).
constexpr int kUnits = 4;

template <class Id>
__device__ __forceinline__ int64_t row_of(const Id* ids, int64_t t, int64_t vocab) {
  const int64_t id = (int64_t)__ldg(ids + t);
  return id >= 0 && id < vocab ? id : -1;
}

template <class In, class Out, class Id, bool VEC>
__global__ void __launch_bounds__(kBlock) k_embedding(const In* __restrict__ table, const Id* __restrict__ ids, Out* __restrict__ out, int64_t n, int64_t cols, Divisor by_row, bool small, int64_t ld,
                                                      int64_t vocab, float scale) {
  const int64_t units = (n + 7) >> 3;
  const int64_t base = (int64_t)blockIdx.x * (kBlock * kUnits) + threadIdx.x;
  if (VEC) {
    const int64_t per_row = cols >> 3;
    int64_t row[kUnits], col[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int64_t u = base + k * kBlock;
      row[k] = -2;
      if (u < units) {
        const int64_t t = small ? by_row.quotient((uint32_t)u) : u / per_row;
        col[k] = (u - t * per_row) << 3;
        row[k] = row_of(ids, t, vocab);
      }
    }
    Raw8<In> r[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
      if (row[k] >= 0) r[k] = load8_cached(table + row[k] * ld + col[k]);
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      if (row[k] == -2) break;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (row[k] >= 0) {
        widen8(r[k], v);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] *= scale;
      }
      store8(out + (base + k * kBlock) * 8, v);
    }
  } else {
#pragma unroll 1
    for (int k = 0; k < kUnits; ++k) {
      const int64_t u = base + k * kBlock;
      if (u >= units) break;
      int64_t t = small ? by_row.quotient((uint32_t)(u * 8)) : u * 8 / cols;
      int64_t c = u * 8 - t * cols;
      int64_t row = row_of(ids, t, vocab);
      const int m = (int)min((int64_t)8, n - u * 8);
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        v[q] = 0.f;
        if (q < m) {
          if (row >= 0) v[q] = scale * widen(__ldg(table + row * ld + c));
          if (++c == cols && q + 1 < m) {
            c = 0;
            row = row_of(ids, ++t, vocab);
          }
        }
      }
      if (m == 8) store8(out + u * 8, v);
      else
        for (int q = 0; q < m; ++q) put(out + u * 8 + q, v[q]);
    }
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
    for (int64_t q = b; q < e; ++q) sum += widen(dy[(int64_t)pos[q] * ld + c]);
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
  const int64_t in_bytes = (int64_t)dt_size(d.in_dt);
  const bool vec = d.cols % 8 == 0 && aligned16(table) && d.ld * in_bytes % 16 == 0;
  const bool small = n < (int64_t)1 << 31;
  const Divisor by_row(vec ? d.cols / 8 : d.cols);
  const unsigned blocks = (unsigned)((n + 8 * kBlock * kUnits - 1) / (8 * kBlock * kUnits));
  with_types(d.in_dt, d.out_dt, d.ids_dt, [&](auto* i, auto* o, auto* id) {
    using In = std::remove_pointer_t<decltype(i)>;
    using Out = std::remove_pointer_t<decltype(o)>;
    using Id = std::remove_pointer_t<decltype(id)>;
    auto* f = vec ? k_embedding<In, Out, Id, true> : k_embedding<In, Out, Id, false>;
    f<<<blocks, kBlock, 0, c.stream>>>((const In*)table, (const Id*)ids, (Out*)out, n, d.cols, by_row, small, d.ld, d.vocab, (float)d.scale);
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
