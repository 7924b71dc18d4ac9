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
// all of them before it stores.  Rows of the table start on 16 bytes, those of the result on eight elements, so a unit is a vector of one row.
// 65536 tokens of 2048 bf16 features out of 131072 rows: 71 us with two units a thread (one 88, four 73, eight 82; one
// element a thread and a 64-bit division each 361), where the bytes alone need 54.  What is left is the way through L2:
// with the whole table in there the same result takes 54.
constexpr int kUnits = 2;

template <class Id>
__device__ __forceinline__ int64_t row_of(const Id* ids, int64_t t, int64_t vocab) {
  const int64_t id = (int64_t)__ldg(ids + t);
  return id >= 0 && id < vocab ? id : -1;
}

template <class In, class Out, class Id>
__global__ void __launch_bounds__(kBlock) k_embedding(const In* __restrict__ table, const Id* __restrict__ ids, Out* __restrict__ out, int64_t n, int64_t cols, Divisor by_row, bool small, int64_t ld,
                                                      int64_t vocab, float scale) {
  const int64_t units = n >> 3, per_row = cols >> 3;
  const int64_t base = (int64_t)blockIdx.x * (kBlock * kUnits) + threadIdx.x;
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
    store8_whole(out + (base + k * kBlock) * 8, v);
  }
}

// Rows that do not start on 16 bytes (an odd length, a window of a wider table, a result off its vectors): a warp takes kRowVecs vectors of a row of
// the result, cut at the result's vectors, and reads the 16-byte lines that hold the elements; the few in front of the
// first vector and behind the last go one by one.  (65536 x 2047 bf16: 87 us, 2048 73; units across rows, each with its own
// shift, took 184.)
constexpr int kRowVecs = 128;

template <class In, class Out, class Id>
__global__ void __launch_bounds__(kBlock) k_embedding_rows(const In* __restrict__ table, const In* end, const Id* __restrict__ ids, Out* __restrict__ out, int64_t rows, int64_t cols, int parts,
                                                           Divisor by_part, int64_t ld, int64_t vocab, float scale) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * (kBlock / 32) + threadIdx.x / 32;
  const int64_t t = w < (int64_t)1 << 31 ? by_part.quotient((uint32_t)w) : w / parts;
  if (t >= rows) return;
  const int part = (int)(w - t * parts);
  const int64_t row = row_of(ids, t, vocab);
  const In* x = table + (row < 0 ? 0 : row) * ld;
  Out* y = out + t * cols;
  constexpr int kWhole = 8 * sizeof(Out);
  const int head = (int)min((int64_t)((kWhole - (uintptr_t)y % kWhole) % kWhole / sizeof(Out)), cols), vecs = (int)((cols - head) >> 3);
  const int64_t rest = head + 8 * (int64_t)vecs;  // with a lane's number on top it may pass 2^31
  if (part == 0 && lane < head) put(y + lane, row < 0 ? 0.f : scale * widen(__ldg(x + lane)));
  if (part == parts - 1 && rest + lane < cols) put(y + rest + lane, row < 0 ? 0.f : scale * widen(__ldg(x + rest + lane)));
  const int last = min(vecs, (part + 1) * kRowVecs);
  constexpr int kFly = kRowVecs / 32;
  const int v0 = part * kRowVecs + lane;
  Lines<In> lines[kFly];
  if (row >= 0) {
#pragma unroll
    for (int k = 0; k < kFly; ++k)
      if (v0 + k * 32 < last) lines[k].fetch(x + head + (v0 + k * 32) * 8, end);
  }
#pragma unroll
  for (int k = 0; k < kFly; ++k) {
    if (v0 + k * 32 >= last) break;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row >= 0) {
      lines[k].get(v);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] *= scale;
    }
    store8_whole(y + head + (v0 + k * 32) * 8, v);
  }
}

// ---- the gradient ----------------------------------------------------------------------------------------------------
// dtable[v] = scale * sum of dy[t] over the tokens with id v, added in the order of the tokens and so the same from run
// to run, in four parts:
//   sort            the tokens' places sorted by id (stably), and which rows have a token at all
//   k_sum_runs      chunks of the sorted places: a run of one id is summed and written to its row by the chunk it begins
//                   in, if it ends no later than the next one; chunks that a longer run touches leave their parts of
//                   its sum in the workspace
//   (same launch)   rows without a token are filled with zeros
//   k_join_runs     the parts of the long runs, added in the order of the chunks
// No atomic touches a sum.  The work is bound by memory: the gradients are read once, the table's written once; cutting
// at fixed places rather than by id keeps the blocks even when few ids hold most of the tokens.

// Sort of many tokens: least significant digits first, up to 9 bits a pass, two launches of up to kPlaceBlocks blocks a
// pass.  Each warp owns a run of consecutive tokens: it counts their digits in its own row of shared memory (equal digits
// among 32 tokens are found by votes, the lowest lane adds), the counts become places through sums over warps, blocks and
// digits, and a second walk writes key and place.  What bounds a pass is latency, and on few SMs the scattered stores, one
// sector a cycle each (65536 tokens on one cluster of eight blocks: 51 us, spread over 64 blocks 22).  Writing the zeros
// of the untouched rows from further blocks of these launches made the whole slower, 251 -> 280 us at 65536 tokens and
// 131072 x 2048: the sort's loads and stores then wait behind the fill's.
constexpr int kBins = 512, kSortBlock = kBins, kSortWarps = kSortBlock / 32;  // a thread a digit
constexpr int kHold = 8;  // groups of 32 tokens whose keys a warp asks for at once
constexpr int kPlaceBlocks = 64;

struct SortShared {
  uint32_t count[kSortWarps][kBins];
  uint32_t base[kBins];
  uint32_t warp_sum[kSortWarps];
  int32_t seen[kBins];
};

// the lanes that have this lane's digit, by one vote a bit (one bit more than the digit where some lanes have none)
__device__ __forceinline__ uint32_t lanes_with(uint32_t d, int bits) {
  uint32_t same = ~0u;
  for (int b = 0; b < bits; ++b) {
    const uint32_t set = __ballot_sync(~0u, d >> b & 1);
    same &= d >> b & 1 ? set : ~set;
  }
  return same;
}

template <class Id>
struct SortPass {
  const Id* ids;
  const int32_t* from;  // keys and, `rows` behind them, places; null: the first pass, which reads the ids
  int32_t* to;
  uint8_t* touched;     // rows with a token, marked by the first pass
  int64_t rows, vocab, lo, hi;  // this warp's run
  int shift, digit, lane, warp;

  __device__ __forceinline__ void own(int rank, int ranks) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    const int64_t per = ((rows + ranks * kSortWarps - 1) / (ranks * kSortWarps) + 31) / 32 * 32;
    lo = min(rows, per * (rank * kSortWarps + warp));
    hi = min(rows, lo + per);
  }
  __device__ __forceinline__ int32_t key_at(int64_t t) const {
    if (from) return __ldcg(from + t);
    const int64_t id = (int64_t)__ldg(ids + t);
    return id >= 0 && id < vocab ? (int32_t)id : (int32_t)vocab;  // a token outside the table comes last
  }
  __device__ __forceinline__ void fetch(int64_t t0, int32_t (&key)[kHold]) const {
#pragma unroll
    for (int k = 0; k < kHold; ++k)
      if (t0 + k * 32 + lane < hi) key[k] = key_at(t0 + k * 32 + lane);
  }
  __device__ __forceinline__ bool held() const { return hi - lo <= 32 * kHold; }
  __device__ __forceinline__ void fetch_places(int64_t t0, int32_t (&pos)[kHold]) const {
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      const int64_t t = t0 + k * 32 + lane;
      if (t < hi) pos[k] = from ? __ldcg(from + rows + t) : (int32_t)t;
    }
  }
  // First walk: counts of this block's digits, as sums over the warps in front; returns the total of digit threadIdx.x.
  __device__ __forceinline__ uint32_t count(SortShared& sh, int32_t (&key)[kHold], bool fetched = false) const {
    for (int k = lane; k < kBins; k += 32) sh.count[warp][k] = 0;
    __syncwarp();
    const uint32_t below = (1u << lane) - 1, mask = (1u << digit) - 1;
    for (int64_t t0 = lo; t0 < hi; t0 += 32 * kHold) {
      if (!fetched || !held()) fetch(t0, key);
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        if (t0 + k * 32 >= hi) break;
        const bool have = t0 + k * 32 + lane < hi;
        const uint32_t d = have ? (uint32_t)key[k] >> shift & mask : ~0u;
        const uint32_t same = lanes_with(d, digit + 1);
        if (have && !(same & below)) sh.count[warp][d] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t n = sh.count[w][threadIdx.x];
      sh.count[w][threadIdx.x] = sum;
      sum += n;
    }
    return sum;
  }
  // all: tokens of all blocks with digit threadIdx.x; before: those of the blocks in front
  __device__ __forceinline__ void bases(SortShared& sh, uint32_t all, uint32_t before) const {
    uint32_t scan = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t n = __shfl_up_sync(~0u, scan, o);
      if (lane >= o) scan += n;
    }
    if (lane == 31) sh.warp_sum[warp] = scan;
    __syncthreads();
    const uint32_t front = __reduce_add_sync(~0u, lane < warp ? sh.warp_sum[lane] : 0);
    sh.base[threadIdx.x] = front + scan - all + before;
    __syncthreads();
  }
  __device__ __forceinline__ void place(SortShared& sh, int32_t (&key)[kHold], int32_t (&pos)[kHold]) const {
    const uint32_t below = (1u << lane) - 1, mask = (1u << digit) - 1;
    for (int64_t t0 = lo; t0 < hi; t0 += 32 * kHold) {
      if (!held()) {
        fetch(t0, key);
        fetch_places(t0, pos);
      }
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        if (t0 + k * 32 >= hi) break;
        const bool have = t0 + k * 32 + lane < hi;
        const uint32_t d = have ? (uint32_t)key[k] >> shift & mask : ~0u;
        const uint32_t same = lanes_with(d, digit + 1);
        const uint32_t at = have ? sh.base[d] + sh.count[warp][d] + __popc(same & below) : 0;
        __syncwarp();
        if (have) {
          if (!(same & below)) sh.count[warp][d] += __popc(same);
          to[at] = key[k];
          to[rows + at] = pos[k];
          // thousands of stores to the one byte of a frequent id would queue up (26 us instead of 8): a block marks
          // an id again only when another one has taken its place among the last seen
          if (!from && key[k] < vocab && sh.seen[key[k] % kBins] != key[k]) {
            sh.seen[key[k] % kBins] = key[k];
            touched[key[k]] = 1;
          }
        }
        __syncwarp();
      }
    }
  }
};

__device__ __forceinline__ void clear_touched(uint8_t* touched, int64_t vocab, int32_t* crossing, int rank, int ranks) {
  const int64_t words = (vocab + 15) / 16;
  for (int64_t i = (int64_t)rank * kSortBlock + threadIdx.x; i < words; i += (int64_t)ranks * kSortBlock) ((uint4*)touched)[i] = make_uint4(0, 0, 0, 0);
  if (rank == 0 && threadIdx.x == 0) *crossing = 0;
}

// Up to kRankTokens: every token's place is the number of tokens that come before it, counted outright, which replaces
// four launches by one without any exchange between blocks.  A warp takes four tokens and compares them with four keys a
// lane at a time; `parts` warps share the keys, so that there is about a block to an SM, of 32 warps.  (8148 tokens: 15 us;
// with half as many warps and no sharing 19; two blocks to an SM read the ids twice and take 16.6.  The comparisons are most of it.)
constexpr int kRankTokens = 8192, kRankBlock = 1024, kRankWarps = kRankBlock / 32;

template <class Id>
__global__ void __launch_bounds__(kRankBlock) k_rank_tokens(const Id* __restrict__ ids, int rows, int64_t vocab, int parts, int32_t* __restrict__ key, int32_t* __restrict__ pos, uint8_t* touched,
                                                            int32_t* crossing) {
  __shared__ __align__(16) uint32_t sh[kRankTokens];
  __shared__ int count[4 * kRankWarps];
  pdl_release();
  if (blockIdx.x == 0 && threadIdx.x == 0) *crossing = 0;
  if (threadIdx.x < 4 * kRankWarps) count[threadIdx.x] = 0;
  const int vecs = (rows + 3) / 4, lane = threadIdx.x & 31;
#pragma unroll 8
  for (int t = threadIdx.x; t < vecs * 4; t += kRankBlock) {
    uint32_t k = ~0u;
    if (t < rows) {
      const int64_t id = (int64_t)__ldg(ids + t);
      k = id >= 0 && id < vocab ? (uint32_t)id : (uint32_t)vocab;  // a token outside the table comes last
    }
    sh[t] = k;
  }
  __syncthreads();
  const int groups = kRankWarps / parts, group = threadIdx.x / 32 / parts, part = threadIdx.x / 32 % parts;
  const int own = blockIdx.x * groups + group;
  if (own < vecs) {
    const uint4 m4 = ((const uint4*)sh)[own];
    const uint32_t mine[4] = {m4.x, m4.y, m4.z, m4.w};
    int before[4] = {0, 0, 0, 0};
#pragma unroll 2
    for (int v = part * 32 + lane; v < vecs; v += 32 * parts) {
      const uint4 k = ((const uint4*)sh)[v];
      const uint32_t front = v < own;  // equal ids in front count, those behind do not
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t limit = mine[i] + front;
        before[i] += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      before[i] = __reduce_add_sync(~0u, before[i]);
      if (lane == i) atomicAdd(&count[group * 4 + i], before[i]);
    }
  }
  __syncthreads();
  const int t = blockIdx.x * groups * 4 + threadIdx.x;
  if (threadIdx.x < groups * 4 && t < rows) {
    const uint32_t mine = sh[t];
    int at = count[threadIdx.x];
    for (int j = t & ~3; j < t; ++j) at += sh[j] == mine;  // those of its own four that come first
    key[at] = (int32_t)mine;
    pos[at] = t;
    if (touched && mine < (uint32_t)vocab) touched[mine] = 1;
  }
}

// one pass in two launches: totals[block][digit], then the places
template <class Id>
__global__ void __launch_bounds__(kSortBlock) k_count_tokens(SortPass<Id> s, uint32_t* totals, int32_t* crossing) {
  __shared__ SortShared sh;
  pdl_wait();
  pdl_release();
  if (!s.from) clear_touched(s.touched, s.vocab, crossing, blockIdx.x, gridDim.x);
  s.own(blockIdx.x, gridDim.x);
  int32_t key[kHold];
  totals[blockIdx.x * kBins + threadIdx.x] = s.count(sh, key);
}
template <class Id>
__global__ void __launch_bounds__(kSortBlock) k_place_tokens(SortPass<Id> s, const uint32_t* __restrict__ totals) {
  __shared__ SortShared sh;
  pdl_wait();
  pdl_release();
  s.own(blockIdx.x, gridDim.x);
  sh.seen[threadIdx.x] = -1;  // (barriers follow)
  int32_t key[kHold], pos[kHold];
  s.fetch(s.lo, key);  // asked for ahead of the totals
  s.fetch_places(s.lo, pos);
  uint32_t before = 0, all = 0;
  const int ranks = gridDim.x;
#pragma unroll
  for (int r = 0; r < kPlaceBlocks; ++r) {
    const uint32_t n = r < ranks ? __ldg(totals + r * kBins + threadIdx.x) : 0;
    if (r < (int)blockIdx.x) before += n;
    all += n;
  }
  s.count(sh, key, true);
  s.bases(sh, all, before);
  s.place(sh, key, pos);
}

struct GradArgs {
  const int32_t *key, *pos;  // sorted
  const uint8_t* touched;    // null: no row has a token, or `search`
  float* part;               // [chunks][2][pitch]: what a chunk adds to the long run that enters it, and to the one that leaves it
  int32_t *crossing, *list;  // chunks in which a long run begins, how many and which
  int64_t rows, cols, ld, vocab, pitch;
  float scale;
  int chunk, lanes, log_lanes;  // places in a chunk; threads that share one
  int64_t chunks, chunk_blocks, slices;
  Divisor by_row;
  bool small;
  bool search;   // few tokens: whether a row has one is looked up among the sorted tokens
  bool by_rows;  // rows without a token are filled by a warp each
  bool joined;   // k_join_runs follows
};

constexpr int kMaxChunk = 128, kMaxPlaces = 1024, kFillUnits = 8;

// Up to this many tokens a warp finds a row among them in two steps, and there are no marks to clear and to set: one
// launch less (700 tokens, 10007 x 1001 f32: 24.7 -> 21.7 us).  Whole vectors, which otherwise go by units, take a warp a
// row for it, and so only where a row is this many bytes (131072 x 512 f32: 55 -> 52.4 us, but x 256: 37.6 -> 46).
constexpr int kSearchTokens = 1024, kSearchRow = 2048;

__device__ __forceinline__ bool has_token(const GradArgs& g, int64_t row) {  // a warp together
  const int lane = threadIdx.x & 31, step = (int)(g.rows + 31) / 32;
  const int at = lane * step;
  const int seg = __popc(__ballot_sync(~0u, at < g.rows && __ldg(g.key + at) <= row)) - 1;
  if (seg < 0) return false;
  const int here = seg * step + lane;
  return __any_sync(~0u, lane < step && here < g.rows && __ldg(g.key + here) == row);
}

// Zeros for the rows that no token has.  Rows that are whole vectors go by units of eight consecutive elements of the
// result, kFillUnits a thread, whose rows are all looked up before the first is written; other long rows, and those of a
// few tokens, by warps, a row at a time from its first element on a whole vector's boundary; other short ones by elements.
constexpr int kFillRow = 256;  // elements from which a row is a warp's

template <class Out, bool VEC>
__device__ __forceinline__ void fill_rows(const GradArgs& g, Out* out, int64_t block) {
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (g.by_rows) {
    const int lane = threadIdx.x & 31;
    const int64_t at = block * (kBlock / 32) + threadIdx.x / 32;
    if (at >= g.vocab || (g.search ? has_token(g, at) : g.touched && __ldg(g.touched + at))) return;
    Out* row = out + at * g.cols;
    constexpr int kWhole = 8 * sizeof(Out);
    const int head = (int)((kWhole - (uintptr_t)row % kWhole) % kWhole / sizeof(Out)), vecs = (int)((g.cols - head) >> 3);
    const int64_t rest = head + 8 * (int64_t)vecs;
    if (lane < head) put(row + lane, 0.f);
    for (int v = lane; v < vecs; v += 32) store8_whole(row + head + 8 * v, zero);
    if (rest + lane < g.cols) put(row + rest + lane, 0.f);
    return;
  }
  constexpr int kUnit = VEC ? 8 : 1;
  const int64_t units = g.vocab * g.cols / kUnit, per_row = g.cols / kUnit;
  const int64_t base = block * (kBlock * kFillUnits) + threadIdx.x;
  bool free[kFillUnits];
#pragma unroll
  for (int k = 0; k < kFillUnits; ++k) {
    const int64_t u = base + k * kBlock;
    free[k] = u < units && !(g.touched && __ldg(g.touched + (g.small ? (int64_t)g.by_row.quotient((uint32_t)u) : u / per_row)));
  }
#pragma unroll
  for (int k = 0; k < kFillUnits; ++k) {
    if (!free[k]) continue;
    if (VEC) store8_whole(out + (base + k * kBlock) * 8, zero);
    else put(out + base + k * kBlock, 0.f);
  }
}

// A thread has eight columns, STEP apart.  1: rows of dy start on 16 bytes, those of the result on eight elements, and the columns are vectors.
// Otherwise STEP is a warp's width (or that of the threads that share a chunk, if fewer) and they are read and written one by
// one, side by side with the neighbours' (22288 tokens, 1339 x 521 f32: the call 44 us; read as the 16-byte lines that hold eight
// consecutive ones, and turned through shared memory to be written, 78).
template <class In, class Out, int STEP>
__global__ void __launch_bounds__(kBlock, STEP == 1 ? 1 : 4) k_sum_runs(const In* __restrict__ dy, Out* __restrict__ out, const __grid_constant__ GradArgs g) {
  constexpr bool VEC = STEP == 1;
  __shared__ int32_t skey[kMaxPlaces + 2 * kMaxChunk + 2], spos[kMaxPlaces + kMaxChunk];
  pdl_wait();
  if (g.joined) pdl_release();
  if (blockIdx.x >= g.chunk_blocks * g.slices) {
    fill_rows<Out, VEC>(g, out, blockIdx.x - g.chunk_blocks * g.slices);
    return;
  }
  const int64_t block = blockIdx.x / g.slices, slice = blockIdx.x - block * g.slices;
  const int groups = kBlock >> g.log_lanes, places = groups * g.chunk;
  const int64_t first = block * places;
  // keys from one chunk and one place in front to one chunk and one place behind
  for (int i = threadIdx.x; i < places + 2 * g.chunk + 2; i += kBlock) {
    const int64_t q = first - g.chunk - 1 + i;
    skey[i] = q < 0 ? -1 : q < g.rows ? __ldg(g.key + q) : INT32_MAX;
  }
  for (int i = threadIdx.x; i < places + g.chunk; i += kBlock) spos[i] = first + i < g.rows ? __ldg(g.pos + first + i) : 0;
  __syncthreads();
  const int lane = threadIdx.x & (g.lanes - 1), group = threadIdx.x >> g.log_lanes;
  const int64_t chunk = block * groups + group;
  const int32_t *key = skey + g.chunk + 1 + group * g.chunk, *pos = spos + group * g.chunk;
  const int64_t c0 = (slice * g.lanes + (VEC ? lane : lane / STEP * STEP)) * 8 + (VEC ? 0 : lane % STEP);
  if (chunk >= g.chunks || c0 >= g.cols) return;
  const int live = (int)min((g.cols - c0 + STEP - 1) / STEP, (int64_t)8);  // columns
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (key[0] >= g.vocab) return;  // nothing but tokens outside the table, or no chunk at all: a whole group
  // The run that enters belongs to the chunk in front if it begins there and ends here: it is passed over.  The run
  // that leaves is this chunk's, to its end, if it begins here and ends in the next one.
  int begin = 0, stop = g.chunk;
  bool enters = key[0] == key[-1];
  if (enters && key[g.chunk] != key[0] && key[-g.chunk - 1] != key[0]) {
    while (begin < g.chunk && key[begin] == key[0]) ++begin;
    enters = false;
  }
  const int32_t last = key[g.chunk - 1];
  bool leaves = key[g.chunk] == last;
  if (leaves && key[2 * g.chunk] != last && !(key[0] == last && key[0] == key[-1])) {
    while (key[stop] == last) ++stop;
    leaves = false;
  }
  if (begin == stop) return;
  int32_t now = key[begin];
  if (now >= g.vocab) return;
  auto flush = [&](bool to_part) {
    if (enters || to_part) {
      float* p = g.part + (chunk * 2 + (enters ? 0 : 1)) * g.pitch + c0;
      if (VEC) {
        *(float4*)p = make_float4(acc[0], acc[1], acc[2], acc[3]);
        *(float4*)(p + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < live) p[j * STEP] = acc[j];
      }
      return;
    }
    Out* p = out + (int64_t)now * g.cols + c0;
    if (VEC) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = g.scale * acc[j];
      store8_whole(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < live) put(p + j * STEP, g.scale * acc[j]);
    }
  };
  constexpr int kFly = 4;
  for (int i = begin; i < stop && key[i] < g.vocab; i += kFly) {
    Raw8<In> raw[VEC ? kFly : 1];
    In one[VEC ? 1 : kFly][8];
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (i + k >= stop || key[i + k] >= g.vocab) continue;
      const In* p = dy + (int64_t)pos[i + k] * g.ld + c0;
      if (VEC) {
        raw[VEC ? k : 0] = load8(p);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) one[VEC ? 0 : k][j] = j < live ? __ldcs(p + j * STEP) : In(0);
      }
    }
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (i + k >= stop || key[i + k] >= g.vocab) break;
      if (key[i + k] != now) {
        flush(false);
        enters = false;
        now = key[i + k];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      }
      float v[8];
      if (VEC) {
        widen8(raw[VEC ? k : 0], v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = widen(one[VEC ? 0 : k][j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += v[j];
    }
  }
  leaves = leaves && now == last;
  flush(leaves);
  if (leaves && !enters && lane == 0 && slice == 0) g.list[atomicAdd(g.crossing, 1)] = (int32_t)chunk;
}

// The long runs.  A block adds the parts of one run for 256 columns: its eight warps take equal
// stretches of the run's chunks, their sums are added in the order of the warps.
template <class Out>
__global__ void __launch_bounds__(kBlock) k_join_runs(Out* __restrict__ out, const __grid_constant__ GradArgs g) {
  __shared__ float sum[kBlock / 32][kBlock];
  pdl_wait();
  const int n = *g.crossing, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t slices = (g.cols + kBlock - 1) / kBlock, work = n * slices;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int64_t item = w / slices, c0 = (w - item * slices) * kBlock;
    const int64_t chunk = g.list[item];
    const int32_t key = __ldg(g.key + (chunk + 1) * g.chunk - 1);
    int64_t m = 0;  // chunks behind this one that begin inside the run
    for (;;) {
      const int64_t c = chunk + 1 + m + threadIdx.x;
      const int same = __syncthreads_count(c < g.chunks && __ldg(g.key + c * g.chunk) == key);
      m += same;
      if (same < kBlock) break;
    }
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int64_t lo = chunk + 1 + m * warp / (kBlock / 32), hi = chunk + 1 + m * (warp + 1) / (kBlock / 32);
#pragma unroll 4
    for (int64_t c = lo; c < hi; ++c) {
      const float* p = g.part + c * 2 * g.pitch + c0 + lane;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + lane + j * 32 < g.cols) acc[j] += __ldg(p + j * 32);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[warp][lane + j * 32] = acc[j];
    __syncthreads();
    const int64_t c = c0 + threadIdx.x;
    if (c < g.cols) {
      float total = __ldg(g.part + (chunk * 2 + 1) * g.pitch + c);
#pragma unroll
      for (int k = 0; k < kBlock / 32; ++k) total += sum[k][threadIdx.x];
      put(out + (int64_t)key * g.cols + c, g.scale * total);
    }
    __syncthreads();
  }
}

// How the gradient is cut, and where its parts lie in the workspace.
struct GradPlan {
  int passes, digit, ranks;  // of the sort of many tokens
  GradArgs g;
  int64_t keys_a, keys_b, touched, crossing, list, totals, part, bytes;  // byte offsets
  GradPlan(const CallDesc& d, int sm_count) : g{} {
    int bits = 1;
    while (bits < 31 && (d.vocab >> bits)) ++bits;
    passes = (bits + 8) / 9;
    digit = (bits + passes - 1) / passes;
    ranks = (int)std::min<int64_t>(kPlaceBlocks, (d.rows + 2 * kSortBlock - 1) / (2 * kSortBlock));
    g.rows = d.rows;
    g.cols = d.cols;
    g.ld = d.ld;
    g.vocab = d.vocab;
    g.scale = (float)d.scale;
    // As many threads as a row of up to 128 has columns by eight.  Longer rows are cut into slices of 256 to 2048 columns, the
    // longest of those that leave nearly the fewest threads without columns.
    auto width = [&](int lanes) { return (d.cols + 8 * lanes - 1) / (8 * lanes) * lanes; };
    g.lanes = 8;
    while (g.lanes < 32 && g.lanes * 8 < d.cols) g.lanes *= 2;
    if (g.lanes == 32)
      for (int lanes = 64; lanes <= kBlock; lanes *= 2)
        if (width(lanes) * 8 <= width(32) * 9) g.lanes = lanes;
    g.log_lanes = 3;
    while (1 << g.log_lanes < g.lanes) ++g.log_lanes;
    const int groups = kBlock / g.lanes;
    g.slices = std::max<int64_t>(1, (d.cols + 8 * g.lanes - 1) / (8 * g.lanes));
    // Chunks as long as they still give every SM six blocks (8148 tokens, 5000 x 4775 bf16: 72 us, with two blocks 86, with
    // eight 71; 65536 tokens, 131072 x 2048: 228, 232 and 234).
    const int64_t blocks = sm_count * 6, least = d.rows > 2048 ? 16 : d.rows > 1024 ? 8 : 4;
    g.chunk = std::min(kMaxChunk, kMaxPlaces / groups);
    while (g.chunk > least && (d.rows + (int64_t)g.chunk * groups - 1) / ((int64_t)g.chunk * groups) * g.slices < blocks) g.chunk /= 2;
    g.chunks = (d.rows + g.chunk - 1) / g.chunk;
    g.chunk_blocks = (g.chunks + groups - 1) / groups;
    auto take = [&](int64_t n) {
      const int64_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    bytes = 0;
    keys_a = take(2 * d.rows * 4);
    keys_b = take(2 * d.rows * 4);
    touched = take(d.vocab + 16);
    crossing = take(4);
    list = take(g.chunks * 4);
    totals = take((int64_t)kPlaceBlocks * kBins * 4);
    g.pitch = (d.cols + 7) / 8 * 8;
    part = take(g.chunks * 2 * g.pitch * 4);
  }
};

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
  const bool vec = d.cols % 8 == 0 && aligned16(table) && d.ld * in_bytes % 16 == 0 && whole_stores(out, dt_size(d.out_dt));
  with_types(d.in_dt, d.out_dt, d.ids_dt, [&](auto* i, auto* o, auto* id) {
    using In = std::remove_pointer_t<decltype(i)>;
    using Out = std::remove_pointer_t<decltype(o)>;
    using Id = std::remove_pointer_t<decltype(id)>;
    if (vec) {
      const unsigned blocks = (unsigned)((n / 8 + kBlock * kUnits - 1) / (kBlock * kUnits));
      k_embedding<In, Out, Id><<<blocks, kBlock, 0, c.stream>>>((const In*)table, (const Id*)ids, (Out*)out, n, d.cols, Divisor(d.cols / 8), n < (int64_t)1 << 31, d.ld, d.vocab, (float)d.scale);
    } else {
      const int64_t parts = (d.cols / 8 + kRowVecs) / kRowVecs, warps = d.rows * parts;
      const unsigned blocks = (unsigned)((warps + kBlock / 32 - 1) / (kBlock / 32));
      k_embedding_rows<In, Out, Id><<<blocks, kBlock, 0, c.stream>>>((const In*)table, (const In*)table + (d.vocab ? (d.vocab - 1) * d.ld + d.cols : 0), (const Id*)ids, (Out*)out, d.rows, d.cols,
                                                                    (int)parts, Divisor(parts), d.ld, d.vocab, (float)d.scale);
    }
  });
  ++*c.launches;
  return cudaGetLastError();
}

int64_t embedding_grad_workspace(const CallDesc& d, int sm_count) { return d.rows && d.vocab * d.cols ? GradPlan(d, sm_count).bytes : 0; }

cudaError_t launch_embedding_grad(const LaunchCtx& c, const CallDesc& d, const void* dy, const void* ids, void* out, void* workspace) {
  if (d.vocab * d.cols == 0) return cudaSuccess;
  GradPlan p(d, c.sm_count);
  GradArgs& g = p.g;
  char* w = (char*)workspace;
  const int64_t n = d.vocab * d.cols;
  const bool vec_out = d.cols % 8 == 0 && whole_stores(out, dt_size(d.out_dt));
  const bool vec = vec_out && aligned16(dy) && d.ld * (int64_t)dt_size(d.in_dt) % 16 == 0;
  g.by_row = Divisor(vec ? d.cols / 8 : d.cols);
  g.small = n < (int64_t)1 << 31;
  g.search = d.rows > 0 && d.rows <= kSearchTokens && (vec ? d.cols * (int64_t)dt_size(d.out_dt) >= kSearchRow : d.cols >= kFillRow);
  g.by_rows = (!vec || g.search) && d.cols >= kFillRow;
  g.joined = g.chunks > 2;  // a run of at most two chunks' length never is a long one
  const int64_t per = g.by_rows ? kBlock / 32 : kBlock * kFillUnits, fills = g.by_rows ? d.vocab : vec ? n / 8 : n;
  const int64_t fill_blocks = (fills + per - 1) / per;
  // Every kernel but the first may be set up while the one in front is still running: it waits for that one's results
  // before it looks at anything.  The last lets nobody in ahead of its end, so what follows this call finds it done.
  cudaError_t err = cudaSuccess;
  bool behind = false;
  auto launch = [&](auto* kernel, int64_t blocks, int threads, auto... args) {
    if (err != cudaSuccess) return;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = behind ? 1 : 0;
    err = cudaLaunchKernelEx(&cfg, kernel, args...);
    behind = true;
    ++*c.launches;
  };
  with_types(d.in_dt, d.out_dt, d.ids_dt, [&](auto* i, auto* o, auto* id) {
    using In = std::remove_pointer_t<decltype(i)>;
    using Out = std::remove_pointer_t<decltype(o)>;
    using Id = std::remove_pointer_t<decltype(id)>;
    if (d.rows) {
      int32_t *a = (int32_t*)(w + p.keys_a), *b = (int32_t*)(w + p.keys_b);
      g.key = p.passes % 2 ? a : b;
      g.pos = g.key + d.rows;
      g.touched = g.search ? nullptr : (const uint8_t*)(w + p.touched);
      g.crossing = (int32_t*)(w + p.crossing);
      g.list = (int32_t*)(w + p.list);
      g.part = (float*)(w + p.part);
      if (d.rows <= kRankTokens) {
        if (!g.search) err = cudaMemsetAsync(w + p.touched, 0, (size_t)d.vocab, c.stream);
        int parts = 1;
        while (parts < 8 && (d.rows + 4 * kRankWarps / (parts * 2) - 1) / (4 * kRankWarps / (parts * 2)) <= c.sm_count) parts *= 2;
        const int per = 4 * kRankWarps / parts;
        launch(k_rank_tokens<Id>, (d.rows + per - 1) / per, kRankBlock, (const Id*)ids, (int)d.rows, d.vocab, parts, (int32_t*)g.key, (int32_t*)g.pos, (uint8_t*)g.touched, g.crossing);
      } else {
        SortPass<Id> pass{};
        pass.ids = (const Id*)ids;
        pass.touched = (uint8_t*)(w + p.touched);
        pass.rows = d.rows;
        pass.vocab = d.vocab;
        pass.digit = p.digit;
        uint32_t* totals = (uint32_t*)(w + p.totals);
        for (int k = 0; k < p.passes; ++k) {
          pass.from = k == 0 ? nullptr : k % 2 ? a : b;
          pass.to = k % 2 ? b : a;
          pass.shift = k * p.digit;
          launch(k_count_tokens<Id>, p.ranks, kSortBlock, pass, totals, g.crossing);
          launch(k_place_tokens<Id>, p.ranks, kSortBlock, pass, (const uint32_t*)totals);
        }
      }
    } else {
      g.chunk_blocks = 0;
    }
    launch(vec ? k_sum_runs<In, Out, 1> : g.lanes == 8 ? k_sum_runs<In, Out, 8> : g.lanes == 16 ? k_sum_runs<In, Out, 16> : k_sum_runs<In, Out, 32>, g.chunk_blocks * g.slices + fill_blocks, kBlock, (const In*)dy, (Out*)out, g);
    if (g.joined) launch(k_join_runs<Out>, std::min<int64_t>(g.chunks * ((d.cols + kBlock - 1) / kBlock), (int64_t)c.sm_count * 8), kBlock, (Out*)out, g);
  });
  return err != cudaSuccess ? err : cudaGetLastError();
}

}  // namespace rx
