// Log probabilities of given tokens, with the entropy and the most likely tokens of every row, and their gradient.
#include "rx_token.cuh"
#include "rx_token.h"

#include <algorithm>
#include <type_traits>

namespace rx {

namespace {

constexpr int kBlock = 256;

// m = max z, s = sum exp(z - m), w = sum exp(z - m) (z - m) of some of a row's elements; m = -inf: nothing but -inf
struct RowSum {
  float m, s, w;
};
__device__ __forceinline__ void merge(RowSum& a, const RowSum& b) {
  const float m = nan_max(a.m, b.m);
  if (m == -INFINITY) return;
  const float da = a.m - m, db = b.m - m;
  const float fa = expf(da), fb = expf(db);
  // w was taken against the old maximum: sum e (z - m) = f (w + s (m_old - m))
  // (a part far below the maximum, a mask of the type's lowest value say, counts nothing: s (m_old - m) may be infinite there)
  const float wa = fa != 0.f ? fa * (a.w + a.s * da) : 0.f, wb = fb != 0.f ? fb * (b.w + b.s * db) : 0.f;
  a.s = (a.m == -INFINITY ? 0.f : a.s * fa) + (b.m == -INFINITY ? 0.f : b.s * fb);
  a.w = (a.m == -INFINITY ? 0.f : wa) + (b.m == -INFINITY ? 0.f : wb);
  a.m = m;
}

// the order of the top tokens: larger value first (NaN above everything, -0 equal to 0), then the lower index
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = x != x ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)~index;
}

template <class T, class Id>
__global__ void __launch_bounds__(kBlock) k_logprobs(const T* __restrict__ logits, const Id* __restrict__ ids, int64_t cols, int64_t ld, float scale, int top_k, LogProbsOut out) {
  __shared__ RowSum part[kBlock];
  __shared__ uint64_t best[kBlock];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  RowSum a{-INFINITY, 0.f, 0.f};
  for (int64_t c = threadIdx.x; c < cols; c += kBlock) merge(a, RowSum{widen(x[c]) * scale, 1.f, 0.f});
  part[threadIdx.x] = a;
  __syncthreads();
  for (int o = kBlock / 2; o > 0; o /= 2) {
    if (threadIdx.x < o) merge(part[threadIdx.x], part[threadIdx.x + o]);
    __syncthreads();
  }
  a = part[0];
  const bool empty = a.m == -INFINITY;  // nothing but -inf: no token has any probability
  const float lse = empty ? -INFINITY : a.m + logf(a.s);
  if (threadIdx.x == 0) {
    const int64_t id = ids[row];
    out.lse[row] = lse;
    out.entropy[row] = empty ? 0.f : logf(a.s) - a.w / a.s;
    out.logprob[row] = id < 0 || id >= cols ? 0.f : empty ? -INFINITY : widen(x[id]) * scale - lse;
  }
  uint64_t below = ~0ull;
  for (int k = 0; k < top_k; ++k) {
    uint64_t b = 0;
    for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
      const uint64_t key = order_key(widen(x[c]), (uint32_t)c);
      if ((k == 0 || key < below) && key > b) b = key;
    }
    best[threadIdx.x] = b;
    __syncthreads();
    for (int o = kBlock / 2; o > 0; o /= 2) {
      if (threadIdx.x < o && best[threadIdx.x + o] > best[threadIdx.x]) best[threadIdx.x] = best[threadIdx.x + o];
      __syncthreads();
    }
    below = best[0];
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t index = ~(uint32_t)below;
      out.top_value[row * top_k + k] = empty ? -INFINITY : widen(x[index]) * scale - lse;
      out.top_token[row * top_k + k] = (int32_t)index;
    }
  }
}

// dx = scale * (p (dlse - dlogprob - dentropy (log p + H)) + dlogprob [the token]),  p = exp(scale x - lse)
//
// Bound by memory: the logits are read and their gradient written once.  A block takes kBlock / TPR rows, TPR threads
// each (as many as a row has vectors of eight, up to the block), and blockIdx.y a segment of long rows; what a row
// needs is five numbers, read once per thread.  Rows that do not start on 16 bytes are walked from their first aligned
// element, with the few in front and behind taken one by one; VEC is false where the logits and the result do not
// lie alike (a window of a wider array with another pitch).
constexpr int kGradVecs = 4;  // vectors of a thread in flight

__device__ __forceinline__ float exp2_fast(float x) {  // within two units of the last place; results below 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

struct GradRow {
  float c, lse, h, a, gh, hot;  // a = dlse - dlogprob; hot = what the token's own element gets on top
  int32_t id;                   // the token, -1: none
  __device__ __forceinline__ float at(float x) const {
    const float logp = fmaf(x, c, -lse);
    const float p = exp2_fast(logp * 1.44269504088896340736f);
    // a masked logit has p = 0 and log p = -inf, whose product is not wanted
    return p != 0.f ? p * fmaf(-gh, logp + h, a) * c : 0.f;
  }
  __device__ __forceinline__ float one(float x, int32_t col) const { return at(x) + (col == id ? hot : 0.f); }
};

template <class T, class Id, int TPR, bool VEC>
__global__ void __launch_bounds__(kBlock) k_logprobs_grad(const T* __restrict__ logits, const Id* __restrict__ ids, int64_t rows, int64_t cols, int64_t ld, float scale, LogProbsGradIn in,
                                                          T* __restrict__ out) {
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;
  const T* x = logits + row * ld;
  T* y = out + row * cols;
  GradRow r;
  r.c = scale;
  r.lse = __ldg(in.lse + row);
  r.h = __ldg(in.entropy + row);
  const int64_t id = (int64_t)__ldg(ids + row);
  r.id = id >= 0 && id < cols ? (int32_t)id : -1;
  const float g = in.dlogprob && r.id >= 0 ? __ldg(in.dlogprob + row) : 0.f;
  r.gh = in.dentropy ? __ldg(in.dentropy + row) : 0.f;
  r.a = (in.dlse ? __ldg(in.dlse + row) : 0.f) - g;
  r.hot = g * scale;
  if (r.lse == -INFINITY) {  // a row without any probability has no gradient: every p becomes 0
    r.lse = INFINITY;
    r.id = -1;
  }
  if (VEC) {
    // elements in front of the first one on a 16-byte boundary (the same for both arrays)
    int64_t head = (int64_t)((16 - (uintptr_t)y % 16) % 16 / sizeof(T));
    if (head > cols) head = cols;
    const int64_t vecs = (cols - head) >> 3, tail = head + (vecs << 3);
    if (blockIdx.y == 0) {
      for (int64_t c = lane; c < head; c += TPR) put(y + c, r.one(widen(x[c]), (int32_t)c));
      for (int64_t c = tail + lane; c < cols; c += TPR) put(y + c, r.one(widen(x[c]), (int32_t)c));
    }
    const int64_t step = (int64_t)gridDim.y * TPR * kGradVecs;
    for (int64_t v0 = (int64_t)blockIdx.y * TPR * kGradVecs + lane; v0 < vecs; v0 += step) {
      Raw8<T> raw[kGradVecs];
#pragma unroll
      for (int k = 0; k < kGradVecs; ++k)
        if (v0 + k * TPR < vecs) raw[k] = load8(x + head + ((v0 + k * TPR) << 3));
#pragma unroll
      for (int k = 0; k < kGradVecs; ++k) {
        if (v0 + k * TPR >= vecs) break;
        const int64_t c = head + ((v0 + k * TPR) << 3);
        float v[8];
        widen8(raw[k], v);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = r.at(v[q]);
        const uint32_t hit = (uint32_t)(r.id - (int32_t)c);
        if (hit < 8u) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] += hit == q ? r.hot : 0.f;
        }
        store8(y + c, v);
      }
    }
  } else {
    for (int64_t c = (int64_t)blockIdx.y * TPR + lane; c < cols; c += (int64_t)gridDim.y * TPR) put(y + c, r.one(widen(x[c]), (int32_t)c));
  }
}

template <class F>
void with_types(DT in, DT ids, F f) {
  auto by_id = [&](auto* i) {
    if (ids == DT::S64) f(i, (int64_t*)nullptr);
    else f(i, (int32_t*)nullptr);
  };
  if (in == DT::BF16) by_id((uint16_t*)nullptr);
  else by_id((float*)nullptr);
}

}  // namespace

int64_t logprobs_workspace(const CallDesc&, int) { return 0; }

cudaError_t launch_logprobs(const LaunchCtx& c, const CallDesc& d, const void* logits, const void* ids, const LogProbsOut& out, void*) {
  if (!d.rows) return cudaSuccess;
  with_types(d.in_dt, d.ids_dt, [&](auto* i, auto* id) {
    k_logprobs<<<(unsigned)d.rows, kBlock, 0, c.stream>>>((decltype(i))logits, (decltype(id))ids, d.cols, d.ld, (float)d.scale, d.top_k, out);
  });
  ++*c.launches;
  return cudaGetLastError();
}

cudaError_t launch_logprobs_grad(const LaunchCtx& c, const CallDesc& d, const void* logits, const void* ids, const LogProbsGradIn& in, void* out) {
  if (d.rows * d.cols == 0) return cudaSuccess;
  const int64_t es = (int64_t)dt_size(d.in_dt);
  // the two arrays lie alike when every row of both starts at the same place of a 16-byte line
  const bool vec = ((uintptr_t)logits - (uintptr_t)out) % 16 == 0 && (d.rows == 1 || (d.ld - d.cols) * es % 16 == 0);
  const int64_t vecs = (d.cols + 7) / 8;
  int tpr = 8;
  while (tpr < kBlock && tpr * kGradVecs < vecs) tpr *= 2;
  const int64_t blocks = (d.rows + kBlock / tpr - 1) / (kBlock / tpr);
  // long rows are cut into segments only as far as the rows alone do not give every SM several blocks
  int64_t segments = 1;
  if (tpr == kBlock) segments = std::max<int64_t>(1, std::min((vecs + kBlock * kGradVecs - 1) / (kBlock * kGradVecs), (int64_t)c.sm_count * 16 / blocks));
  with_types(d.in_dt, d.ids_dt, [&](auto* i, auto* id) {
    using T = std::remove_pointer_t<decltype(i)>;
    using Id = std::remove_pointer_t<decltype(id)>;
    auto go = [&](auto* f) { f<<<dim3((unsigned)blocks, (unsigned)segments), kBlock, 0, c.stream>>>((const T*)logits, (const Id*)ids, d.rows, d.cols, d.ld, (float)d.scale, in, (T*)out); };
    auto by_tpr = [&](auto t) {
      constexpr int kTpr = decltype(t)::value;
      if (vec) go(k_logprobs_grad<T, Id, kTpr, true>);
      else go(k_logprobs_grad<T, Id, kTpr, false>);
    };
    switch (tpr) {
      case 8: by_tpr(std::integral_constant<int, 8>()); break;
      case 16: by_tpr(std::integral_constant<int, 16>()); break;
      case 32: by_tpr(std::integral_constant<int, 32>()); break;
      case 64: by_tpr(std::integral_constant<int, 64>()); break;
      case 128: by_tpr(std::integral_constant<int, 128>()); break;
      default: by_tpr(std::integral_constant<int, kBlock>()); break;
    }
  });
  ++*c.launches;
  return cudaGetLastError();
}

}  // namespace rx
