// Log probabilities of given tokens, with the entropy and the most likely tokens of every row, and their gradient.
#include "rx_token.cuh"
#include "rx_token.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

namespace rx {

namespace {

constexpr int kBlock = 256;
// Rows up to kWarpRow are one warp's where there are enough of them to keep the SMs busy: kWarpRows per SM, twice as many
// for rows longer than kWarpLong.  (In brackets with a block of 128 a row: 25000 x 4100 f32 66 [87] us, with twenty top
// tokens 126 [181]; 12000 x 16500 bf16 80 [84], with five 96 [135]; 6000 x 33000 bf16 88 [73], with five 101 [97].)
constexpr int kWarpRow = 20000, kWarpLong = 8192, kWarpRows = 16;
constexpr int kMaxRanksPerRow = 8;   // blocks of a cluster that share a row

__device__ __forceinline__ float exp2_fast(float x) {  // within two units of the last place; results below 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float nan_max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two floats in one 64-bit register, one instruction for both
using Pair = uint64_t;
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(Pair p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// ---- the sums of a row -------------------------------------------------------------------------------------------
// With c = log2(e) / temperature and a reference ref, one pass keeps
//     s = sum 2^a,   w = sum 2^a a,   a = c (x - ref),
// from which lse = ref / temperature + ln s and H = ln s - ln(2) w / s.  The reference need not be the maximum: it is
// the maximum of the first vector a thread meets, and moves only when a logit lies 2^kSlack above it, so the sums are
// almost never rescaled and cannot overflow.  How far below the maximum it may lie decides how much of H is lost when ln s
// and w / s, both up to kSlack then, are subtracted, and how much of s and w is rounded away next to a large term; a vector's
// eight terms are therefore added up before they join the sums.  On 2048 rows of 50016 logits with one token standing out, H is
// off by 3.7e-7 (rms; the definition in 32 bits 4.3e-7) and 1.3e-6 at most; with a slack of 16 and every term added
// singly 1.6e-6 and 12e-6, for 1 to 4 % less time (4096 x 131072 bf16 172 us, now 176; a slack of 6 takes 177).
// x - ref is exact where it matters, whatever the size of the logits.
// Arguments are cut at kFloor, where 2^a is 0 already: -inf, and a mask of the type's lowest value, add 0 and not
// 0 * inf.  NaN and +inf go through (cut and maxima propagate NaN; inf - inf is NaN).
constexpr float kSlack = 8.f, kFloor = -300.f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct RowSum {
  float ref, s, w;
};
__device__ __forceinline__ void rescale(RowSum& a, float ref, float c) {
  const float d = nan_max((a.ref - ref) * c, kFloor), f = exp2_fast(d);
  a.w = f * fmaf(a.s, d, a.w);
  a.s *= f;
  a.ref = ref;
}
struct Running {
  float ref, limit, slack;  // limit = ref + slack
  float c;
  Pair s, w;
  __device__ __forceinline__ explicit Running(float c_) : ref(-3.402823466e38f), limit(-3.402823466e38f), slack(kSlack / c_), c(c_), s(0), w(0) {}
  __device__ __forceinline__ void move(float top) {
    RowSum lo, hi;
    lo.ref = hi.ref = ref;
    split(s, lo.s, hi.s);
    split(w, lo.w, hi.w);
    rescale(lo, top, c);
    rescale(hi, top, c);
    s = pair(lo.s, hi.s);
    w = pair(lo.w, hi.w);
    ref = top;
    limit = top + slack;
  }
  __device__ __forceinline__ float push(const float (&v)[8]) {  // returns the largest
    const float top = nan_max3(nan_max3(v[0], v[1], v[2]), nan_max3(v[3], v[4], v[5]), nan_max(v[6], v[7]));
    if (!(top <= limit)) move(top);
    const Pair minus = pair(-ref, -ref), cc = pair(c, c);
    Pair vs, vw;  // of this vector
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float a0, a1;
      split(mul2(add2(pair(v[2 * q], v[2 * q + 1]), minus), cc), a0, a1);
      a0 = nan_max(a0, kFloor);
      a1 = nan_max(a1, kFloor);
      const Pair e = pair(exp2_fast(a0), exp2_fast(a1));
      vs = q == 0 ? e : add2(vs, e);
      vw = q == 0 ? mul2(e, pair(a0, a1)) : fma2(e, pair(a0, a1), vw);
    }
    s = add2(s, vs);  // a quarter of the roundings next to a large sum
    w = add2(w, vw);
    return top;
  }
  __device__ __forceinline__ void push1(float x) {
    if (!(x <= limit)) move(x);
    const float a = nan_max((x - ref) * c, kFloor), e = exp2_fast(a);
    s = add2(s, pair(e, 0.f));
    w = add2(w, pair(e * a, 0.f));
  }
  __device__ __forceinline__ RowSum sum() const {
    float s0, s1, w0, w1;
    split(s, s0, s1);
    split(w, w0, w1);
    return {ref, s0 + s1, w0 + w1};
  }
};

// The sums of W neighbouring lanes together, in all of them: one common reference, one rescaling per lane, and sums in
// the order of a butterfly (the same in every lane: a + b is b + a).
template <int W>
__device__ __forceinline__ RowSum lanes_sum(RowSum a, float c) {
  float ref = a.ref;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) ref = nan_max(ref, __shfl_xor_sync(~0u, ref, o));
  rescale(a, ref, c);
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(~0u, a.s, o);
    a.w += __shfl_xor_sync(~0u, a.w, o);
  }
  return a;
}

// ---- the top tokens -----------------------------------------------------------------------------------------------
// One whole number per logit, larger for larger values (NaN above everything, -0 equal to 0) and, among equal ones, for
// lower tokens: what is selected does not depend on the order in which candidates are met.
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0xFFFFFFFFu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) { return (uint64_t)value_key(x) << 32 | (uint32_t)~index; }
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}

// The k largest of keys[0 .. n), which are all different: put(place, key) for each, by one of the `lanes` threads that
// work on it, this one being the lane-th.  The caller synchronises before and after.
template <class Put>
__device__ __forceinline__ void select_top(const uint64_t* keys, int n, int k, int lane, int lanes, Put put) {
  for (int i = lane; i < n; i += lanes) {
    const uint64_t mine = keys[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > mine;
    if (above < k) put(above, mine);
  }
}
__device__ __forceinline__ void select_top(const uint64_t* keys, int n, int k, uint64_t* best, int lane, int lanes) {
  select_top(keys, n, k, lane, lanes, [&](int place, uint64_t key) { best[place] = key; });
}

struct RowOut {
  float ref, scale, log_s;
  bool empty;  // nothing but -inf: no token has any probability
  __device__ __forceinline__ explicit RowOut(const RowSum& a, float scale_) : ref(a.ref), scale(scale_), log_s(logf(a.s)), empty(a.s == 0.f) {}
  __device__ __forceinline__ float logprob(float x) const { return empty ? -INFINITY : fmaf(x - ref, scale, -log_s); }
  __device__ __forceinline__ float lse() const { return empty ? -INFINITY : fmaf(ref, scale, log_s); }
  __device__ __forceinline__ float entropy(const RowSum& a) const { return empty ? 0.f : fmaf(-kLn2, a.w / a.s, log_s); }
};

template <class T, class Id>
__device__ __forceinline__ void write_row(const RowSum& a, const RowOut& o, const T* x, const Id* ids, int64_t row, int64_t cols, const LogProbsOut& out) {
  const int64_t id = (int64_t)__ldg(ids + row);
  out.lse[row] = o.lse();
  out.entropy[row] = o.entropy(a);
  out.logprob[row] = id < 0 || id >= cols ? 0.f : o.logprob(widen(x[id]));
}

// A row as vectors of eight from its first element on a 16-byte boundary, and the few in front and behind.
template <class T>
struct Span {
  const T* x;
  int64_t head, vecs, cols;
  __device__ __forceinline__ Span(const T* row, int64_t n) : x(row), cols(n) {
    head = min((int64_t)((16 - (uintptr_t)row % 16) % 16 / sizeof(T)), n);
    vecs = (n - head) >> 3;
  }
  __device__ __forceinline__ int loose() const { return (int)(cols - (vecs << 3)); }                          // at most 14
  __device__ __forceinline__ int64_t loose_at(int k) const { return k < head ? k : k + (vecs << 3); }          // where the k-th of them lies
  __device__ __forceinline__ int64_t at(int64_t v) const { return head + (v << 3); }
};

constexpr int kMaxLoose = 14;

// ---- W = 8 or 32 lanes per row: rows of up to 512 (bf16) or 1024 (f32) -----------------------------------------------------------------
// A row's elements sit in its lanes' registers, NE each, read one by one (eight lanes: a warp's four rows lie next to
// each other).  TOP: the k-th largest value is bounded bit by bit, its upper 16 bits first -- among all elements, or, with
// 32 lanes and k <= 32, among the lanes' largest, which is one vote a bit.  Where that leaves too many (most of the row
// is equal), it is searched for to the last bit, and then the last index that is still wanted among the elements equal
// to it.  What is left, little more than k, is ordered by counting.  One top token is the row's largest, which is known
// already (100000 rows of 128 bf16, none, one, five: 15, 19, 54 us; one as a case of several 52).
constexpr int kNarrowRow = 256, kNarrowTopRow = 128;  // longest rows of eight lanes
template <class T>
struct GroupRow { static constexpr int n = sizeof(T) == 4 ? 1024 : 512; };  // 16-bit loads one by one: 200000 x 1000 bf16 takes 173 us here, 113 with a warp's vectors
template <int W>
struct GroupCap { static constexpr int n = W == 8 ? 2 * kMaxTopK + 8 : 4 * kMaxTopK; };

// A bound from below on the k-th largest of the 32 lanes' keys (0: fewer lanes have one): for a small k the k-th itself,
// largest by largest; otherwise its upper 16 bits, bit by bit with one vote each.
__device__ __forceinline__ uint32_t bound_of_lanes(uint32_t key, int k) {
  uint32_t bound = 0;
  if (k <= 10) {
    for (int left = k;;) {
      bound = __reduce_max_sync(~0u, key);
      left -= __popc(__ballot_sync(~0u, key == bound));
      if (left <= 0 || bound == 0) return bound;
      if (key == bound) key = 0;
    }
  }
  for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
    if (__popc(__ballot_sync(~0u, key >= (bound | bit))) >= k) bound |= bit;
  return bound;
}

template <int W>
__device__ __forceinline__ int lanes_count(int n) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) n += __shfl_xor_sync(~0u, n, o);
  return n;
}

template <class T, class Id, bool TOP, int W, int NE>
__global__ void __launch_bounds__(kBlock, NE == 32 ? (W == 8 ? 2 : 3) : 4) k_logprobs_group(const T* __restrict__ logits, const Id* __restrict__ ids, int64_t rows, int64_t cols_, int64_t ld, float scale, int top_k, LogProbsOut out) {
  constexpr int kRows = kBlock / W, kCap = GroupCap<W>::n;
  __shared__ uint64_t buf_[TOP ? kRows : 1][kCap];
  const int lane = threadIdx.x % W, group = threadIdx.x / W, cols = (int)cols_;
  const int64_t row = (int64_t)blockIdx.x * kRows + group;
  const bool live = row < rows;
  const T* x = logits + (live ? row : 0) * ld;
  const float c = scale * kLog2e;
  float v[NE];
#pragma unroll
  for (int j = 0; j < NE; ++j) v[j] = lane + j * W < cols ? widen(__ldcs(x + lane + j * W)) : -INFINITY;
  float top = v[0];
#pragma unroll
  for (int j = 1; j + 1 < NE; j += 2) top = nan_max3(top, v[j], v[j + 1]);
  top = nan_max(top, v[NE - 1]);
  const float lane_top = top;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) top = nan_max(top, __shfl_xor_sync(~0u, top, o));
  RowSum a{nan_max(top, -3.402823466e38f), 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    const float t = nan_max((v[j] - a.ref) * c, kFloor), e = exp2_fast(t);
    a.s += e;
    a.w = fmaf(e, t, a.w);
  }
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(~0u, a.s, o);
    a.w += __shfl_xor_sync(~0u, a.w, o);
  }
  const RowOut o(a, scale);
  if (live && lane == 0) write_row(a, o, x, ids, row, cols_, out);
  if (TOP && top_k == 1) {  // the row's largest is known; its lowest index is not
    int at = INT32_MAX;
    if (top == top) {
#pragma unroll
      for (int j = NE - 1; j >= 0; --j)
        if (v[j] == top) at = lane + j * W;
    } else {
#pragma unroll
      for (int j = NE - 1; j >= 0; --j)
        if (v[j] != v[j]) at = lane + j * W;
    }
    if (W == 32) {
      at = __reduce_min_sync(~0u, at);
    } else {
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(~0u, at, o));
    }
    if (live && lane == 0) {
      out.top_value[row] = o.logprob(top);
      out.top_token[row] = at;
    }
    return;
  }
  if (TOP) {
    uint64_t* buf = buf_[group];
    const uint32_t mates = (W == 32 ? ~0u : (1u << W % 32) - 1) << (threadIdx.x % 32 / W * W), before = mates & ((1u << (threadIdx.x % 32)) - 1);
    int n = 0;
    bool done = false;
    if (W == 32 && top_k <= 32) {
      const uint32_t reach = bound_of_lanes(lane < cols ? value_key(lane_top) : 0u, top_k);
      const float least = key_value((uint64_t)reach << 32);  // NaN, where there is no bound: nothing is below it
      done = true;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        const int at = lane + j * W;
        const bool take = at < cols && !(v[j] < least);
        const uint32_t who = __ballot_sync(~0u, take);
        if (!who) continue;
        if (n + __popc(who) > kCap) {
          done = false;
          break;
        }
        if (take) buf[n + __popc(who & before)] = order_key(v[j], (uint32_t)at);
        n += __popc(who);
      }
    }
    if (!done) {
      __syncwarp();
      uint32_t reach = 0;
      int reached = cols, last = cols;  // of the elements equal to `reach`, those with an index up to `last` count
      uint32_t key[NE];
#pragma unroll
      for (int j = 0; j < NE; ++j) key[j] = lane + j * W < cols ? value_key(v[j]) : 0u;
      auto search = [&](uint32_t from, uint32_t to) {
        for (uint32_t bit = from; bit >= to && bit; bit >>= 1) {
          int m = 0;
#pragma unroll
          for (int j = 0; j < NE; ++j) m += key[j] >= (reach | bit);
          m = lanes_count<W>(m);
          if (m >= top_k) {
            reach |= bit;
            reached = m;
          }
        }
      };
      search(1u << 31, 1u << 16);
      if (__any_sync(~0u, reached > 2 * top_k + 8)) {
        search(1u << 15, 1u);
        int above = 0;
#pragma unroll
        for (int j = 0; j < NE; ++j) above += key[j] > reach;
        const int wanted = top_k - lanes_count<W>(above);
        last = 0;
        for (int bit = W * NE / 2; bit > 0; bit >>= 1) {  // the largest index with fewer than `wanted` equal ones below it
          int m = 0;
#pragma unroll
          for (int j = 0; j < NE; ++j) m += key[j] == reach && lane + j * W < (last | bit);
          if (lanes_count<W>(m) < wanted) last |= bit;
        }
      }
      n = 0;
#pragma unroll
      for (int j = 0; j < NE; ++j) {
        const int at = lane + j * W;
        const uint32_t k = key[j];
        const bool take = k != 0u && (k > reach || (k == reach && at <= last));
        const uint32_t who = __ballot_sync(~0u, take);
        if (take) buf[n + __popc(who & before)] = (uint64_t)k << 32 | (uint32_t)~at;
        n += __popc(who & mates);
      }
    }
    __syncwarp();
    if (live)
      select_top(buf, n, top_k, lane, W, [&](int place, uint64_t k) {
        out.top_value[row * top_k + place] = o.logprob(key_value(k));
        out.top_token[row * top_k + place] = (int32_t)~(uint32_t)k;
      });
  }
}

// ---- one warp per row: middling rows, many of them --------------------------------------------------------------------
// TOP (top_k <= 32): while it streams, a lane notes the largest value of each of its stretches of vectors.  The k-th
// largest of the 32 lanes' maxima bounds the k-th of the row from below, bit by bit with one vote each; only the stretches
// that reach it are read again, their vectors spread over the lanes, and little more than k candidates are kept.
constexpr int kWarpTop = 32, kWarpSpells = 16;
constexpr int kWarpCap = 256 + kWarpTop + kMaxLoose;

template <class T, class Id, bool TOP>
__global__ void __launch_bounds__(kBlock, !TOP && sizeof(T) == 4 ? 4 : 0) k_logprobs_warp(const T* __restrict__ logits, const Id* __restrict__ ids, int64_t rows, int64_t cols, int64_t ld, float scale, int top_k, LogProbsOut out) {
  constexpr int kWarps = kBlock / 32, kFly = 4;
  __shared__ uint64_t buf_[TOP ? kWarps : 1][kWarpCap], best_[TOP ? kWarps : 1][kWarpTop];
  __shared__ float spell_[TOP ? kWarps : 1][TOP ? kWarpSpells * 32 : 1];
  __shared__ uint16_t item_[TOP ? kWarps : 1][TOP ? kWarpSpells * 32 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= rows) return;
  const Span<T> sp(logits + row * ld, cols);
  const float c = scale * kLog2e;
  Running run(c);
  float mine = -INFINITY;
  const int loose = sp.loose();
  float extra = -INFINITY;
  if (lane < loose) {
    extra = widen(sp.x[sp.loose_at(lane)]);
    run.push1(extra);
  }
  const int vecs = (int)sp.vecs, tiles = (vecs + 32 * kFly - 1) / (32 * kFly), per = TOP ? (tiles + kWarpSpells - 1) / kWarpSpells : tiles;
  const T* body = sp.x + sp.head;
  for (int g = 0, tile = 0; tile < tiles; ++g) {
    float spell = -INFINITY;
    for (const int stop = min(tiles, tile + per); tile < stop; ++tile) {
      const int v0 = tile * 32 * kFly + lane;
      Raw8<T> raw[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k)
        if (v0 + k * 32 < vecs) raw[k] = TOP ? load8_cached(body + (v0 + k * 32) * 8) : load8(body + (v0 + k * 32) * 8);
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        if (v0 + k * 32 >= vecs) break;
        float v[8];
        widen8(raw[k], v);
        const float top = run.push(v);
        if (TOP) spell = nan_max(spell, top);
      }
    }
    if (TOP) {
      spell_[warp][g * 32 + lane] = spell;
      mine = nan_max(mine, spell);
    }
  }
  const RowSum a = lanes_sum<32>(run.sum(), c);
  const RowOut o(a, scale);
  if (lane == 0) write_row(a, o, sp.x, ids, row, cols, out);
  if (TOP) {
    uint64_t *buf = buf_[warp], *best = best_[warp];
    const uint32_t before = (1u << lane) - 1, reach = bound_of_lanes(lane < vecs ? value_key(mine) : 0u, top_k);
    // the same bound as a float: what is not below it is a candidate (NaN included; everything, where there is no bound)
    float least_value = key_value((uint64_t)reach << 32);
    int items = 0;
    for (int g = 0; g * per < tiles; ++g) {
      const bool take = g * per * 32 * kFly + lane < vecs && !(spell_[warp][g * 32 + lane] < least_value);
      const uint32_t who = __ballot_sync(~0u, take);
      if (take) item_[warp][items + __popc(who & before)] = (uint16_t)(g * 32 + lane);
      items += __popc(who);
    }
    uint64_t least = 0;
    int n = 0;
    auto keep = [&](bool take, float v, int at) {  // all lanes together
      uint32_t who = __ballot_sync(~0u, take);
      if (!who) return;
      const uint64_t key = order_key(v, (uint32_t)at);
      take = take && key > least;
      who = __ballot_sync(~0u, take);
      if (take) buf[n + __popc(who & before)] = key;
      n += __popc(who);
    };
    auto shrink = [&]() {
      __syncwarp();
      select_top(buf, n, top_k, best, lane, 32);
      __syncwarp();
      if (n > top_k) n = top_k;
      for (int i = lane; i < n; i += 32) buf[i] = best[i];
      if (n == top_k) {
        least = best[top_k - 1];
        least_value = key_value(least);
      }
      __syncwarp();
    };
    keep(lane < loose && !(extra < least_value), extra, lane < loose ? (int)sp.loose_at(lane) : 0);
    __syncwarp();
    const int slots = items * per * kFly;
    for (int s0 = 0; s0 < slots; s0 += 32) {
      const int slot = s0 + lane, item = slot < slots ? item_[warp][slot / (per * kFly)] : 0, k = slot % (per * kFly);
      const int tile = item / 32 * per + k / kFly, v0 = tile * 32 * kFly + k % kFly * 32 + item % 32;
      const bool have = slot < slots && tile < tiles && v0 < vecs;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (have) widen8(load8_cached(body + v0 * 8), v);
      const int at = (int)sp.head + v0 * 8;
#pragma unroll
      for (int q = 0; q < 8; ++q) keep(have && !(v[q] < least_value), v[q], at + q);
      if (n > kWarpTop) shrink();
    }
    __syncwarp();
    select_top(buf, n, top_k, lane, 32, [&](int place, uint64_t key) {
      out.top_value[row * top_k + place] = o.logprob(key_value(key));
      out.top_token[row * top_k + place] = (int32_t)~(uint32_t)key;
    });
  }
}

// ---- one block, or a cluster of blocks, per row: long rows ---------------------------------------------------------------
// The blocks of a cluster take a row's vectors in equal runs and write their sums, and their top tokens in order, into
// the first one's shared memory, which joins them: nobody waits for a load from another block, and a token's place is
// found by bisection in every block's list.  (4 x 131072 bf16 without top tokens and with one, twenty and 64: 4.9, 7.7,
// 10.2 and 12.6 us; when the first block read from the others one after another, 5.9, 11.6, 13.8 and 19.7.)
//
// TOP: while it streams, a thread notes the largest value of each of up to kSpells stretches of its vectors.  The k-th
// largest of the block's per-thread maxima bounds the k-th value of the row from below, so only the stretches that
// reach it (about k of them, whatever the order of the values) are read a second time, a vector a thread at a time, and only
// their elements that reach it are kept.
constexpr int kSpells = 8;
constexpr int kBatchCap = 8 * kMaxTopK + kMaxTopK + 16;

template <class T>
struct Fly { static constexpr int n = sizeof(T) == 2 ? 4 : 2; };  // vectors in flight per thread: 64 bytes

template <int kLong>
struct TopShared {
  uint32_t spell[kSpells][kLong];  // largest value key of a thread's stretch
  uint32_t top[kLong];             // and of all of them
  uint64_t key[kLong];
  uint64_t buf[kBatchCap], best[kMaxTopK];
  uint64_t all[kMaxRanksPerRow * kMaxTopK];  // the first block's: every block's top tokens, in order, 0 where there are fewer
  uint16_t item[kSpells * kLong];
  uint64_t bound;
  uint32_t reach;
  int n, n_items;
};

// A bound from below on the k-th largest of the block's value keys, to sh.reach.  For a small k that of the lanes' largest,
// each out of kLong / 32 keys, is close enough (twenty of 512 keys: about thirty reach it); otherwise the k-th's upper 20
// bits, bit by bit.  One warp does it (about 200 instructions with four keys a lane; comparing every key with every other
// took 16000 and doubled the time of a row).
constexpr int kTopOfLanes = 24;
template <int kLong>
__device__ __forceinline__ void reach_of_block(TopShared<kLong>& sh, uint32_t key, int k) {
  sh.top[threadIdx.x] = key;
  __syncthreads();
  if (threadIdx.x < 32) {
    uint32_t mine[kLong / 32];
#pragma unroll
    for (int j = 0; j < kLong / 32; ++j) mine[j] = sh.top[j * 32 + threadIdx.x];
    uint32_t found = 0;
    if (k <= kTopOfLanes) {
      uint32_t top = mine[0];
#pragma unroll
      for (int j = 1; j < kLong / 32; ++j) top = max(top, mine[j]);
      found = bound_of_lanes(top, k);
    } else {
      for (uint32_t bit = 1u << 31; bit >= 1u << 12; bit >>= 1) {
        const uint32_t want = found | bit;
        int n = 0;
#pragma unroll
        for (int j = 0; j < kLong / 32; ++j) n += mine[j] >= want;
        if (__reduce_add_sync(~0u, n) >= k) found = want;
      }
    }
    if (threadIdx.x == 0) sh.reach = found;
  }
  __syncthreads();
}

// the k-th largest of the block's keys (ties by thread), to sh.bound; 0 is no key
template <int kLong>
__device__ __forceinline__ void kth_of_block(TopShared<kLong>& sh, uint64_t key, int k) {
  const int t = threadIdx.x;
  sh.key[t] = key;
  __syncthreads();
  int above = 0;
#pragma unroll 8
  for (int j = 0; j < kLong; ++j) {
    const uint64_t other = sh.key[j];
    above += other > key || (other == key && j < t);
  }
  if (above == k - 1) sh.bound = key;
  __syncthreads();
}

template <class T, class Id, bool TOP, int kLong>
__global__ void __launch_bounds__(kLong, kLong == 128 ? 6 : 1) k_logprobs_block(const T* __restrict__ logits, const Id* __restrict__ ids, int64_t cols, int64_t ld, float scale, int top_k, LogProbsOut out) {
  namespace cg = cooperative_groups;
  constexpr int kFly = Fly<T>::n, kTile = kLong * kFly;
  __shared__ RowSum part[kLong / 32], sums[kMaxRanksPerRow], total;
  __shared__ TopShared<kLong> sh[1];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  if (ranks > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");  // waited for before anything is written to the first block
  const int64_t row = blockIdx.x / ranks;
  const Span<T> sp(logits + row * ld, cols);
  const float c = scale * kLog2e;
  const int64_t share = ((sp.vecs + ranks - 1) / ranks + kTile - 1) / kTile * kTile;  // whole tiles
  const int64_t lo = min(sp.vecs, share * rank), hi = min(sp.vecs, lo + share);
  const int tid = threadIdx.x, loose = rank == 0 ? sp.loose() : 0;
  Running run(c);
  if (tid < loose) run.push1(widen(sp.x[sp.loose_at(tid)]));
  const int tiles = (int)((hi - lo + kTile - 1) / kTile), per = TOP ? max(1, (tiles + kSpells - 1) / kSpells) : max(1, tiles);
  uint32_t thread_top = 0;
  const int mine = (int)(hi - lo) - tid;  // vectors from this thread's first one to the end of the block's run
  const T* body = sp.x + sp.at(lo + tid);
  Raw8<T> next[kFly];
#pragma unroll
  for (int k = 0; k < kFly; ++k)
    if (k * kLong < mine) next[k] = load8(body + k * kLong * 8);
  for (int g = 0, tile = 0; tile < tiles; ++g) {
    float spell = -INFINITY;
    for (const int end = min(tiles, tile + per); tile < end; ++tile) {
      Raw8<T> raw[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k) raw[k] = next[k];
      const int at = (tile + 1) * kTile;
#pragma unroll
      for (int k = 0; k < kFly; ++k)
        if (at + k * kLong < mine) next[k] = load8(body + (int64_t)(at + k * kLong) * 8);
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        if (at - kTile + k * kLong >= mine) break;
        float v[8];
        widen8(raw[k], v);
        const float top = run.push(v);
        if (TOP) spell = nan_max(spell, top);
      }
    }
    if (TOP) {
      const bool any = lo + (int64_t)g * per * kTile + tid < hi;
      const uint32_t key = any ? value_key(spell) : 0u;
      sh[0].spell[g][tid] = key;
      thread_top = max(thread_top, key);
    }
  }
  RowSum a = lanes_sum<32>(run.sum(), c);
  if ((tid & 31) == 0) part[tid >> 5] = a;
  __syncthreads();
  if (tid < 32) {
    a = lanes_sum<kLong / 32>(part[tid % (kLong / 32)], c);
    if (tid == 0) total = a;
  }
  if (TOP) {
    TopShared<kLong>& t = sh[0];
    if (tid == 0) t.n = t.n_items = 0;
    reach_of_block(t, thread_top, top_k);
    const uint32_t reach = t.reach;
    for (int g = 0; g * per < tiles; ++g) {
      const uint32_t key = t.spell[g][tid];
      if (key >= reach && key != 0u) t.item[atomicAdd(&t.n_items, 1)] = (uint16_t)(g * kLong + tid);
    }
    if (tid < loose) {
      const int64_t at = sp.loose_at(tid);
      t.buf[atomicAdd(&t.n, 1)] = order_key(widen(sp.x[at]), (uint32_t)at);
    }
    __syncthreads();
    const int slots = t.n_items * per * kFly;
    uint64_t least = reach ? ((uint64_t)reach << 32) - 1 : 0;  // a key has to be above this to be among the k best
    for (int s0 = 0; s0 < slots; s0 += kLong) {
      uint64_t key[8], mine = 0;
      bool have = s0 + tid < slots;
      if (have) {
        const int slot = s0 + tid, item = t.item[slot / (per * kFly)], k = slot % (per * kFly);
        const int64_t v = lo + (int64_t)(item / kLong * per + k / kFly) * kTile + k % kFly * kLong + item % kLong;
        have = v < hi && item / kLong * per + k / kFly < tiles;
        if (have) {
          float x[8];
          widen8(load8_cached(sp.x + sp.at(v)), x);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            key[q] = order_key(x[q], (uint32_t)(sp.at(v) + q));
            if (key[q] > least) mine = max(mine, key[q]);
          }
        }
      }
      const int before = t.n;
      int wants = 0;
      if (have) {
#pragma unroll
        for (int q = 0; q < 8; ++q) wants += key[q] > least;
      }
      if (!__syncthreads_or(wants)) continue;
      // as a rule the bound leaves few keys and all of them fit; where most of a row is equal they may not, and then
      // only those that reach the k-th of the threads' best are taken: at most 8 k
      int at = wants ? atomicAdd(&t.n, wants) : 0;
      const bool fits = !__syncthreads_or(wants && at + wants > kBatchCap);
      uint64_t bound = 0;
      if (!fits) {
        if (tid == 0) t.n = before;
        kth_of_block(t, mine, top_k);
        bound = t.bound;
      }
      if (have) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (key[q] > least && key[q] >= bound) {
            if (!fits) at = atomicAdd(&t.n, 1);
            t.buf[at++] = key[q];
          }
      }
      __syncthreads();
      const int n = t.n;
      if (n > top_k && s0 + kLong < slots) {
        select_top(t.buf, n, top_k, t.best, tid, kLong);
        __syncthreads();
        if (tid < top_k) t.buf[tid] = t.best[tid];
        if (tid == 0) t.n = top_k;
        least = t.best[top_k - 1];
      }
      __syncthreads();
    }
    if (ranks == 1) select_top(t.buf, t.n, top_k, t.best, tid, kLong);
  }
  if (ranks > 1) {
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (tid == 0) *cluster.map_shared_rank(&sums[rank], 0) = total;
    if (TOP) {
      uint64_t* list = cluster.map_shared_rank(sh[0].all, 0) + rank * top_k;
      const int n = sh[0].n;
      if (tid >= n && tid < top_k) list[tid] = 0;
      select_top(sh[0].buf, n, top_k, tid, kLong, [&](int place, uint64_t key) { list[place] = key; });
    }
    cluster.sync();
    if (rank != 0) return;
    if (tid < 32) {
      const int r = tid % kMaxRanksPerRow;
      a = lanes_sum<kMaxRanksPerRow>(r < ranks ? sums[r] : RowSum{-3.402823466e38f, 0.f, 0.f}, c);
      if (tid == 0) total = a;
    }
    if (TOP) {
      for (int i = tid; i < ranks * top_k; i += kLong) {
        const uint64_t key = sh[0].all[i];
        if (!key) continue;
        int place = 0;
        for (int r = 0; r < ranks; ++r) {
          int lo = 0, hi = top_k;
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (sh[0].all[r * top_k + mid] > key) lo = mid + 1;
            else hi = mid;
          }
          place += lo;
        }
        if (place < top_k) sh[0].best[place] = key;
      }
    }
  }
  __syncthreads();
  a = total;
  const RowOut o(a, scale);
  if (tid == 0) write_row(a, o, sp.x, ids, row, cols, out);
  if (TOP && tid < top_k) {
    out.top_value[row * top_k + tid] = o.logprob(key_value(sh[0].best[tid]));
    out.top_token[row * top_k + tid] = (int32_t)~(uint32_t)sh[0].best[tid];
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
__global__ void __launch_bounds__(kBlock, 4) k_logprobs_grad(const T* __restrict__ logits, const Id* __restrict__ ids, int64_t rows, int64_t cols, int64_t ld, float scale, LogProbsGradIn in,
                                                          T* __restrict__ out) {
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;
  const T* x = logits + row * ld;
  T* y = out + row * cols;
  // elements in front of the first one on a 16-byte boundary (the same for both arrays)
  const int64_t head = VEC ? min((int64_t)((16 - (uintptr_t)y % 16) % 16 / sizeof(T)), cols) : 0, vecs = VEC ? (cols - head) >> 3 : 0, tail = head + (vecs << 3);
  const int64_t step = (int64_t)gridDim.y * TPR * kGradVecs;
  int64_t v0 = (int64_t)blockIdx.y * TPR * kGradVecs + lane;
  Raw8<T> raw[kGradVecs];
  auto fetch = [&]() {
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k)
      if (v0 + k * TPR < vecs) raw[k] = load8(x + head + ((v0 + k * TPR) << 3));
  };
  if (VEC) fetch();  // in flight while the row's own values come
  GradRow r;
  r.c = scale;
  r.lse = __ldg(in.lse + row);
  r.h = __ldg(in.entropy + row);
  const int64_t id = (int64_t)__ldg(ids + row);
  const float arrived = in.dlogprob ? __ldg(in.dlogprob + row) : 0.f;
  r.gh = in.dentropy ? __ldg(in.dentropy + row) : 0.f;
  const float dlse = in.dlse ? __ldg(in.dlse + row) : 0.f;
  r.id = id >= 0 && id < cols ? (int32_t)id : -1;
  const float g = r.id >= 0 ? arrived : 0.f;
  r.a = dlse - g;
  r.hot = g * scale;
  if (r.lse == -INFINITY) {  // a row without any probability has no gradient: every p becomes 0
    r.lse = INFINITY;
    r.id = -1;
  }
  if (VEC) {
    if (blockIdx.y == 0) {
      for (int64_t c = lane; c < head; c += TPR) put(y + c, r.one(widen(x[c]), (int32_t)c));
      for (int64_t c = tail + lane; c < cols; c += TPR) put(y + c, r.one(widen(x[c]), (int32_t)c));
    }
    while (v0 < vecs) {
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
      v0 += step;
      fetch();
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

cudaError_t launch_logprobs(const LaunchCtx& c, const CallDesc& d, const void* logits, const void* ids, const LogProbsOut& out) {
  if (!d.rows) return cudaSuccess;
  cudaError_t err = cudaSuccess;
  with_types(d.in_dt, d.ids_dt, [&](auto* i, auto* id) {
    using T = std::remove_pointer_t<decltype(i)>;
    using Id = std::remove_pointer_t<decltype(id)>;
    if (d.cols <= GroupRow<T>::n) {
      // with top tokens a warp a row pays earlier, its bound on the k-th costs so little (201615 x 203 f32, twelve: 214 us
      // with eight lanes, 142 with 32; 500000 x 128, twenty: 280 and 323)
      const bool wide = d.cols > (d.top_k && d.top_k <= 32 ? kNarrowTopRow : kNarrowRow);
      const int rows = kBlock / (wide ? 32 : 8);
      const unsigned blocks = (unsigned)((d.rows + rows - 1) / rows);
      auto go = [&](auto* f) { f<<<blocks, kBlock, 0, c.stream>>>((const T*)logits, (const Id*)ids, d.rows, d.cols, d.ld, (float)d.scale, d.top_k, out); };
      if (!wide) {
        if (d.cols <= 64) go(d.top_k ? k_logprobs_group<T, Id, true, 8, 8> : k_logprobs_group<T, Id, false, 8, 8>);
        else if (d.cols <= 128) go(d.top_k ? k_logprobs_group<T, Id, true, 8, 16> : k_logprobs_group<T, Id, false, 8, 16>);
        else go(d.top_k ? k_logprobs_group<T, Id, true, 8, 32> : k_logprobs_group<T, Id, false, 8, 32>);
      } else if (d.cols <= 256) {
        go(k_logprobs_group<T, Id, true, 32, 8>);
      } else if (d.cols <= 512 || sizeof(T) == 2) {
        go(d.top_k ? k_logprobs_group<T, Id, true, 32, 16> : k_logprobs_group<T, Id, false, 32, 16>);
      } else if constexpr (sizeof(T) == 4) {
        go(d.top_k ? k_logprobs_group<T, Id, true, 32, 32> : k_logprobs_group<T, Id, false, 32, 32>);
      }
      return;
    }
    if (d.cols <= kWarpRow && d.top_k <= kWarpTop && d.rows >= (int64_t)c.sm_count * kWarpRows * (d.cols > kWarpLong ? 2 : 1)) {
      const unsigned blocks = (unsigned)((d.rows + kBlock / 32 - 1) / (kBlock / 32));
      auto* f = d.top_k ? k_logprobs_warp<T, Id, true> : k_logprobs_warp<T, Id, false>;
      f<<<blocks, kBlock, 0, c.stream>>>((const T*)logits, (const Id*)ids, d.rows, d.cols, d.ld, (float)d.scale, d.top_k, out);
      return;
    }
    // Up to one row for every SM, blocks of 512, one to an SM, and as many to a row as the SMs allow (clusters of eight do
    // not pack on more than half of them); beyond that blocks of 128, about six to an SM.  A block has at least one tile
    // of its row, or two.  131072 bf16, twenty top tokens, us, with blocks of 512 by 1, 2, 4 and 8 a row [of 128]:
    //   16 rows   14.6 12.6 10.6 16.7  [27.0 18.8 14.7 16.7]
    //   64        15.1 12.7 20.8 34.7  [32.9 21.2 16.7 18.7]
    //   148       16.4 23.3 41.3 65.9  [34.3 23.6 22.6 30.9]
    //   200       27.4 33.1 53.1 86.0  [37.8 25.4 24.9 35.3]
    //   512       52.0 74.0  122  204  [46.4 41.1 51.8 71.5]
    //   1024      90.3  144  235  399  [68.3 72.2 88.4  128]
    auto go = [&](auto size) {
      constexpr int kLong = decltype(size)::value;
      const int64_t sms = c.sm_count;
      auto fits = [&](int ranks) {
        if (d.cols < (int64_t)ranks * (kLong == 128 ? 2 : 1) * kLong * Fly<T>::n * 8) return false;
        if (kLong != 128) return d.rows * ranks <= (ranks == 8 ? sms / 2 : sms);
        return d.rows * ranks <= sms * (ranks == 2 ? 7 : ranks == 4 ? 6 : 0);
      };
      int ranks = 1;
      while (ranks < kMaxRanksPerRow && fits(ranks * 2)) ranks *= 2;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(d.rows * ranks));
      cfg.blockDim = dim3(kLong);
      cfg.stream = c.stream;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)ranks;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      auto* f = d.top_k ? k_logprobs_block<T, Id, true, kLong> : k_logprobs_block<T, Id, false, kLong>;
      err = cudaLaunchKernelEx(&cfg, f, (const T*)logits, (const Id*)ids, d.cols, d.ld, (float)d.scale, d.top_k, out);
    };
    if (d.rows <= c.sm_count) go(std::integral_constant<int, 512>());
    else go(std::integral_constant<int, 128>());
  });
  ++*c.launches;
  return err != cudaSuccess ? err : cudaGetLastError();
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
