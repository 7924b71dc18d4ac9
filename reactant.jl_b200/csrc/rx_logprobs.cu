// Log probabilities of given tokens, with the entropy and the most likely tokens of every row, and their gradient.
#include "rx_device.cuh"
#include "rx_token.h"

namespace rx {

namespace {

constexpr int kBlock = 256;

__device__ __forceinline__ float read_logit(const float* p) { return *p; }
__device__ __forceinline__ float read_logit(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ void put_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_logit(uint16_t* p, float v) { *p = bf16_bits(v); }

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
  for (int64_t c = threadIdx.x; c < cols; c += kBlock) merge(a, RowSum{read_logit(x + c) * scale, 1.f, 0.f});
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
    out.logprob[row] = id < 0 || id >= cols ? 0.f : empty ? -INFINITY : read_logit(x + id) * scale - lse;
  }
  uint64_t below = ~0ull;
  for (int k = 0; k < top_k; ++k) {
    uint64_t b = 0;
    for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
      const uint64_t key = order_key(read_logit(x + c), (uint32_t)c);
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
      out.top_value[row * top_k + k] = empty ? -INFINITY : read_logit(x + index) * scale - lse;
      out.top_token[row * top_k + k] = (int32_t)index;
    }
  }
}

// dx = scale * (p (dlse - dlogprob - dentropy (log p + H)) + dlogprob [the token])
template <class T, class Id>
__global__ void __launch_bounds__(kBlock) k_logprobs_grad(const T* __restrict__ logits, const Id* __restrict__ ids, int64_t cols, int64_t ld, float scale, LogProbsGradIn in, T* __restrict__ out) {
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const int64_t id = ids[row];
  const float lse = in.lse[row], h = in.entropy[row];
  const float g = in.dlogprob && id >= 0 && id < cols ? in.dlogprob[row] : 0.f, gh = in.dentropy ? in.dentropy[row] : 0.f, gl = in.dlse ? in.dlse[row] : 0.f;
  for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
    const float logp = read_logit(x + c) * scale - lse;
    const float p = lse == -INFINITY ? 0.f : expf(logp);
    float dz = p == 0.f ? 0.f : p * (gl - g - gh * (logp + h));
    if (c == id && lse != -INFINITY) dz += g;
    put_logit(out + row * cols + c, dz * scale);
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
  with_types(d.in_dt, d.ids_dt, [&](auto* i, auto* id) {
    k_logprobs_grad<<<(unsigned)d.rows, kBlock, 0, c.stream>>>((decltype(i))logits, (decltype(id))ids, d.cols, d.ld, (float)d.scale, in, (decltype(i))out);
  });
  ++*c.launches;
  return cudaGetLastError();
}

}  // namespace rx
