// Embedding lookup and its gradient.
#include "rx_token.cuh"
#include "rx_token.h"

#include <cooperative_groups.h>

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
      store8_whole(out + (base + k * kBlock) * 8, v);
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
      if (m == 8) store8_whole(out + u * 8, v);
      else
        for (int q = 0; q < m; ++q) put(out + u * 8 + q, v[q]);
    }
  }
}

// ---- the gradient ----------------------------------------------------------------------------------------------------
// dtable[v] = scale * sum of dy[t] over the tokens with id v, added in the order of the tokens and so the same from run
// to run, in four parts:
//   sort            the tokens' places sorted by id (stably), and which rows have a token at all
//   k_sum_runs      chunks of the sorted places: a run of one id inside a chunk is summed and written to its row; a run
//                   that crosses a border of chunks leaves its part of the sum in the workspace
//   (same launch)   rows without a token are filled with zeros
//   k_join_runs     the parts of every run that crosses borders, added in the order of the chunks
// No atomic touches a sum.  The work is bound by memory: the gradients are read once, the table's written once; cutting
// at fixed places rather than by id keeps the blocks even when few ids hold most of the tokens.

// Sort: least significant digits first, up to 9 bits a pass.  Each warp owns a run of consecutive tokens: it counts their
// digits in its own row of shared memory (equal digits among 32 tokens are found by votes, the lowest lane adds), the
// counts become places through sums over warps, blocks and digits, and a second walk writes key and place.
//
// Up to kClusterTokens one cluster of up to eight blocks does all passes in one launch, the blocks' counts meeting in
// distributed shared memory.  More tokens are spread over up to kPlaceBlocks blocks, two launches a pass: what bounds a
// pass is the scattered stores, one sector a cycle and SM (65536 tokens: 51 us on the cluster's eight SMs).  (Writing
// the zeros of the untouched rows from further blocks of these launches made the whole slower, 251 -> 280 us at 65536
// tokens and 131072 x 2048: the sort's loads and stores then wait behind the fill's.)
constexpr int kSortBlock = 1024, kSortWarps = kSortBlock / 32, kBins = 512, kSortRanks = 8;
constexpr int kHold = 8;  // groups of 32 tokens whose keys a warp asks for at once
constexpr int64_t kClusterTokens = kSortRanks * kSortBlock;
constexpr int kPlaceBlocks = 128;

struct SortShared {
  uint32_t count[kSortWarps][kBins];
  uint32_t total[kBins], base[kBins];
  uint32_t warp_sum[kSortWarps];
  uint32_t half_all[kBins], half_before[kBins];
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
  // First walk: counts of this block's digits, as sums over the warps in front, and their totals.  `key` keeps the keys
  // of a short run.
  __device__ __forceinline__ void count(SortShared& sh, int32_t (&key)[kHold]) const {
    for (int k = lane; k < kBins; k += 32) sh.count[warp][k] = 0;
    __syncwarp();
    const uint32_t below = (1u << lane) - 1, mask = (1u << digit) - 1;
    for (int64_t t0 = lo; t0 < hi; t0 += 32 * kHold) {
      fetch(t0, key);
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
    if (threadIdx.x < kBins) {
      uint32_t sum = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t n = sh.count[w][threadIdx.x];
        sh.count[w][threadIdx.x] = sum;
        sum += n;
      }
      sh.total[threadIdx.x] = sum;
    }
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
    if (threadIdx.x < kBins) {
      uint32_t front = lane < warp ? sh.warp_sum[lane] : 0;  // (at most 16 warps are in front of a digit's)
      front = __reduce_add_sync(~0u, front);
      sh.base[threadIdx.x] = front + scan - all + before;
    }
    __syncthreads();
  }
  __device__ __forceinline__ void place(SortShared& sh, int32_t (&key)[kHold]) const {
    const uint32_t below = (1u << lane) - 1, mask = (1u << digit) - 1;
    for (int64_t t0 = lo; t0 < hi; t0 += 32 * kHold) {
      if (hi - lo > 32 * kHold) fetch(t0, key);
      int32_t pos[kHold];
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        const int64_t t = t0 + k * 32 + lane;
        if (t < hi) pos[k] = from ? __ldcg(from + rows + t) : (int32_t)t;
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
          if (!from && key[k] < vocab) touched[key[k]] = 1;
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

template <class Id>
__global__ void __launch_bounds__(kSortBlock) k_sort_tokens(SortPass<Id> s, int passes, int32_t* a, int32_t* b, int32_t* crossing) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t raw[];
  SortShared& sh = *(SortShared*)raw;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  clear_touched(s.touched, s.vocab, crossing, rank, ranks);
  s.own(rank, ranks);
  for (int pass = 0; pass < passes; ++pass) {
    s.from = pass == 0 ? nullptr : pass % 2 ? a : b;
    s.to = pass % 2 ? b : a;
    s.shift = pass * s.digit;
    int32_t key[kHold];
    s.count(sh, key);
    cluster.sync();
    uint32_t before = 0, all = 0;
    if (threadIdx.x < kBins)
      for (int r = 0; r < ranks; ++r) {
        const uint32_t n = *cluster.map_shared_rank(&sh.total[threadIdx.x], r);
        if (r < rank) before += n;
        all += n;
      }
    s.bases(sh, all, before);
    s.place(sh, key);
    cluster.sync();  // what was written is visible, and nobody reads this block's totals any more
  }
}

// Up to 1024 tokens: one block, a token a thread, sorted as (id, place) by Batcher's bitonic network; exchanges within a
// warp are shuffles (700 tokens: 4 us against 11 for two passes over digits).
template <class Id>
__global__ void __launch_bounds__(kSortBlock) k_sort_few_tokens(const Id* __restrict__ ids, int rows, int64_t vocab, int32_t* key, int32_t* pos, uint8_t* touched, int32_t* crossing) {
  __shared__ uint64_t sh[kSortBlock];
  const int t = threadIdx.x;
  uint64_t mine = ~0ull;
  int32_t k = INT32_MAX;
  if (t < rows) {
    const int64_t id = (int64_t)__ldg(ids + t);
    k = id >= 0 && id < vocab ? (int32_t)id : (int32_t)vocab;
    mine = (uint64_t)(uint32_t)k << 32 | (uint32_t)t;
  }
  clear_touched(touched, vocab, crossing, 0, 1);
  for (int size = 2; size <= kSortBlock; size *= 2)
    for (int apart = size / 2; apart > 0; apart /= 2) {
      uint64_t other;
      if (apart >= 32) {
        __syncthreads();
        sh[t] = mine;
        __syncthreads();
        other = sh[t ^ apart];
      } else {
        other = __shfl_xor_sync(~0u, mine, apart);
      }
      const bool low = ((t & apart) == 0) == ((t & size) == 0);  // this thread keeps the smaller of the two
      mine = low == (other < mine) ? other : mine;
    }
  if (t < rows) {
    key[t] = (int32_t)(mine >> 32);
    pos[t] = (int32_t)(uint32_t)mine;
  }
  if (k < vocab) touched[k] = 1;  // (every store of zeros is behind one of the barriers above)
}

// one pass in two launches: totals[block][digit], then the places
template <class Id>
__global__ void __launch_bounds__(kSortBlock) k_count_tokens(SortPass<Id> s, uint32_t* totals, int32_t* crossing) {
  extern __shared__ __align__(16) uint8_t raw[];
  SortShared& sh = *(SortShared*)raw;
  if (!s.from) clear_touched(s.touched, s.vocab, crossing, blockIdx.x, gridDim.x);
  s.own(blockIdx.x, gridDim.x);
  int32_t key[kHold];
  s.count(sh, key);
  if (threadIdx.x < kBins) totals[blockIdx.x * kBins + threadIdx.x] = sh.total[threadIdx.x];
}
template <class Id>
__global__ void __launch_bounds__(kSortBlock) k_place_tokens(SortPass<Id> s, const uint32_t* __restrict__ totals) {
  extern __shared__ __align__(16) uint8_t raw[];
  SortShared& sh = *(SortShared*)raw;
  s.own(blockIdx.x, gridDim.x);
  // the totals of all blocks, two threads a digit: every second block each
  const int bin = threadIdx.x % kBins, half = threadIdx.x / kBins, ranks = gridDim.x;
  uint32_t before = 0, all = 0;
#pragma unroll 16
  for (int r = half; r < ranks; r += 2) {
    const uint32_t n = __ldg(totals + r * kBins + bin);
    if (r < (int)blockIdx.x) before += n;
    all += n;
  }
  if (half) {
    sh.half_all[bin] = all;
    sh.half_before[bin] = before;
  }
  int32_t key[kHold];
  s.count(sh, key);
  if (!half) {
    all += sh.half_all[bin];
    before += sh.half_before[bin];
  }
  s.bases(sh, half ? 0 : all, before);
  s.place(sh, key);
}

struct GradArgs {
  const int32_t *key, *pos;  // sorted
  const uint8_t* touched;    // null: no row has a token
  float* part;               // [chunks][2][cols]: what a chunk adds to the run that enters it, and to the one that leaves it
  int32_t *crossing, *list;  // chunks in which a run starts that leaves them
  int64_t rows, cols, ld, vocab;
  float scale;
  int chunk, lanes, log_lanes;  // places in a chunk; threads that share one
  int64_t chunks, chunk_blocks, slices;
  Divisor by_row;
  bool small;
};

constexpr int kMaxChunk = 128, kMaxPlaces = 1024, kFillUnits = 8;

// Zeros for the rows that no token has: units of eight consecutive elements of the result, kFillUnits a thread, whose
// rows are all looked up before the first is written.  
template <class Out, bool VEC>
__device__ __forceinline__ void fill_rows(const GradArgs& g, Out* out, int64_t block) {
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int64_t n = g.vocab * g.cols, units = (n + 7) >> 3, per_row = g.cols >> 3;
  const int64_t base = block * (kBlock * kFillUnits) + threadIdx.x;
  auto row = [&](int64_t i) -> int64_t {  // of element i
    if (VEC) return g.small ? g.by_row.quotient((uint32_t)(i >> 3)) : (i >> 3) / per_row;
    return g.small ? g.by_row.quotient((uint32_t)i) : i / g.cols;
  };
  bool free[kFillUnits];
#pragma unroll
  for (int k = 0; k < kFillUnits; ++k) {
    const int64_t u = base + k * kBlock;
    free[k] = u < units;
    if (!free[k] || !g.touched) continue;
    const int64_t t = row(u * 8);
    uint32_t any = __ldg(g.touched + t);
    if (!VEC) any |= __ldg(g.touched + row(min(u * 8 + 7, n - 1)));
    free[k] = !any;
  }
#pragma unroll
  for (int k = 0; k < kFillUnits; ++k) {
    const int64_t u = base + k * kBlock;
    if (VEC) {
      if (free[k]) store8_whole(out + u * 8, zero);
    } else if (u < units) {
      // a unit whose ends lie in rows without a token: so do its middle's, where a row is eight elements or longer
      if (free[k] && u * 8 + 8 <= n && g.cols >= 8) store8_whole(out + u * 8, zero);
      else
        for (int64_t i = u * 8; i < min(u * 8 + 8, n); ++i)
          if (!g.touched || !__ldg(g.touched + row(i))) put(out + i, 0.f);
    }
  }
}

// Columns of a thread: eight consecutive ones (VEC), or eight that lie `lanes` apart (rows that do not start on 16 bytes).
template <class In, class Out, bool VEC>
__global__ void __launch_bounds__(kBlock, VEC ? 1 : 3) k_sum_runs(const In* __restrict__ dy, Out* __restrict__ out, const __grid_constant__ GradArgs g) {
  __shared__ int32_t skey[kMaxPlaces + 2], spos[kMaxPlaces];
  if (blockIdx.x >= g.chunk_blocks * g.slices) {
    fill_rows<Out, VEC>(g, out, blockIdx.x - g.chunk_blocks * g.slices);
    return;
  }
  const int64_t block = blockIdx.x / g.slices, slice = blockIdx.x - block * g.slices;
  const int groups = kBlock >> g.log_lanes, places = groups * g.chunk;
  const int64_t first = block * places;
  for (int i = threadIdx.x; i < places; i += kBlock) {
    const int64_t q = first + i;
    skey[i + 1] = q < g.rows ? __ldg(g.key + q) : INT32_MAX;
    spos[i] = q < g.rows ? __ldg(g.pos + q) : 0;
  }
  if (threadIdx.x == 0) skey[0] = first > 0 ? __ldg(g.key + first - 1) : -1;
  if (threadIdx.x == 1) skey[places + 1] = first + places < g.rows ? __ldg(g.key + first + places) : INT32_MAX;
  __syncthreads();
  const int lane = threadIdx.x & (g.lanes - 1), group = threadIdx.x >> g.log_lanes;
  const int64_t chunk = block * groups + group;
  if (chunk >= g.chunks) return;
  const int32_t *key = skey + 1 + group * g.chunk, *pos = spos + group * g.chunk;
  const int64_t c0 = slice * (8 * g.lanes) + (VEC ? lane * 8 : lane);
  auto col = [&](int j) { return c0 + (VEC ? j : j * g.lanes); };
  if (c0 >= g.cols && !(lane == 0 && slice == 0)) return;
  const bool mine = c0 < g.cols;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int32_t now = key[0];
  bool enters = now == key[-1];
  auto flush = [&](bool leaves) {
    if (!mine) return;
    if (enters || leaves) {
      float* p = g.part + (chunk * 2 + (enters ? 0 : 1)) * g.cols;
      if (VEC) {
        *(float4*)(p + c0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        *(float4*)(p + c0 + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col(j) < g.cols) p[col(j)] = acc[j];
      }
    } else {
      Out* p = out + (int64_t)now * g.cols;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = g.scale * acc[j];
      if (VEC) store8_whole(p + c0, v);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col(j) < g.cols) put(p + col(j), v[j]);
    }
  };
  constexpr int kFly = 4;
  int i = 0;
  for (; i < g.chunk && key[i] < g.vocab; i += kFly) {
    float v[kFly][8];
    Raw8<In> raw[kFly];
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (i + k >= g.chunk || key[i + k] >= g.vocab || !mine) continue;
      const In* p = dy + (int64_t)pos[i + k] * g.ld;
      if (VEC) raw[k] = load8(p + c0);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = col(j) < g.cols ? widen(__ldcs(p + col(j))) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (i + k >= g.chunk || key[i + k] >= g.vocab) break;
      if (key[i + k] != now) {
        flush(false);
        enters = false;
        now = key[i + k];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      }
      if (VEC && mine) widen8(raw[k], v[k]);
      if (mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[k][j];
      }
    }
  }
  if (now >= g.vocab) return;  // nothing but tokens outside the table
  const bool leaves = key[g.chunk - 1] == now && key[g.chunk] == now;
  flush(leaves);
  if (leaves && !enters && lane == 0 && slice == 0) g.list[atomicAdd(g.crossing, 1)] = (int32_t)chunk;
}

// The runs that cross borders of chunks.  A block adds the parts of one run for 256 columns: its eight warps take equal
// stretches of the run's chunks, their sums are added in the order of the warps.
template <class Out>
__global__ void __launch_bounds__(kBlock) k_join_runs(Out* __restrict__ out, const __grid_constant__ GradArgs g) {
  __shared__ float sum[kBlock / 32][kBlock];
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
      const float* p = g.part + c * 2 * g.cols + c0 + lane;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + lane + j * 32 < g.cols) acc[j] += __ldg(p + j * 32);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[warp][lane + j * 32] = acc[j];
    __syncthreads();
    const int64_t c = c0 + threadIdx.x;
    if (c < g.cols) {
      float total = __ldg(g.part + (chunk * 2 + 1) * g.cols + c);
#pragma unroll
      for (int k = 0; k < kBlock / 32; ++k) total += sum[k][threadIdx.x];
      put(out + (int64_t)key * g.cols + c, g.scale * total);
    }
    __syncthreads();
  }
}

// How the gradient is cut, and where its parts lie in the workspace.
struct GradPlan {
  int passes, digit, ranks;
  bool spread;  // the sort in launches of its own passes, over many SMs
  GradArgs g;
  int64_t keys_a, keys_b, touched, crossing, list, totals, part, bytes;  // byte offsets
  GradPlan(const CallDesc& d, int sm_count) : g{} {
    int bits = 1;
    while (bits < 31 && (d.vocab >> bits)) ++bits;
    passes = (bits + 8) / 9;
    digit = (bits + passes - 1) / passes;
    ranks = 2;
    while (ranks < kSortRanks && (int64_t)ranks * kSortBlock < d.rows) ranks *= 2;
    spread = d.rows > kClusterTokens;
    if (spread) ranks = (int)std::min<int64_t>(kPlaceBlocks, (d.rows + kSortBlock - 1) / kSortBlock);
    g.rows = d.rows;
    g.cols = d.cols;
    g.ld = d.ld;
    g.vocab = d.vocab;
    g.scale = (float)d.scale;
    g.lanes = 8;
    g.log_lanes = 3;
    while (g.lanes < kBlock && g.lanes * 8 < d.cols) {
      g.lanes *= 2;
      ++g.log_lanes;
    }
    const int groups = kBlock / g.lanes;
    g.slices = std::max<int64_t>(1, (d.cols + 8 * g.lanes - 1) / (8 * g.lanes));
    // chunks as long as they still give every SM two blocks
    g.chunk = std::min(kMaxChunk, kMaxPlaces / groups);
    while (g.chunk > 8 && (d.rows + (int64_t)g.chunk * groups - 1) / ((int64_t)g.chunk * groups) * g.slices < sm_count * 2) g.chunk /= 2;
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
    part = take(g.chunks * 2 * d.cols * 4);
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

int64_t embedding_grad_workspace(const CallDesc& d, int sm_count) { return d.rows && d.vocab * d.cols ? GradPlan(d, sm_count).bytes : 0; }

cudaError_t launch_embedding_grad(const LaunchCtx& c, const CallDesc& d, const void* dy, const void* ids, void* out, void* workspace) {
  if (d.vocab * d.cols == 0) return cudaSuccess;
  GradPlan p(d, c.sm_count);
  GradArgs& g = p.g;
  char* w = (char*)workspace;
  const int64_t n = d.vocab * d.cols;
  const bool vec_out = d.cols % 8 == 0;
  const bool vec = vec_out && aligned16(dy) && d.ld * (int64_t)dt_size(d.in_dt) % 16 == 0;
  g.by_row = Divisor(vec ? d.cols / 8 : d.cols);
  g.small = n < (int64_t)1 << 31;
  const int64_t units = (n + 7) / 8;
  const int64_t fill_blocks = (units + kBlock * kFillUnits - 1) / (kBlock * kFillUnits);
  cudaError_t err = cudaSuccess;
  with_types(d.in_dt, d.out_dt, d.ids_dt, [&](auto* i, auto* o, auto* id) {
    using In = std::remove_pointer_t<decltype(i)>;
    using Out = std::remove_pointer_t<decltype(o)>;
    using Id = std::remove_pointer_t<decltype(id)>;
    if (d.rows) {
      int32_t *a = (int32_t*)(w + p.keys_a), *b = (int32_t*)(w + p.keys_b);
      g.key = p.passes % 2 ? a : b;
      g.pos = g.key + d.rows;
      g.touched = (const uint8_t*)(w + p.touched);
      g.crossing = (int32_t*)(w + p.crossing);
      g.list = (int32_t*)(w + p.list);
      g.part = (float*)(w + p.part);
      SortPass<Id> pass{};
      pass.ids = (const Id*)ids;
      pass.touched = (uint8_t*)(w + p.touched);
      pass.rows = d.rows;
      pass.vocab = d.vocab;
      pass.digit = p.digit;
      auto allow = [&](auto* f) { return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared)); };  // of the current device
      if (d.rows <= kSortBlock) {
        k_sort_few_tokens<Id><<<1, kSortBlock, 0, c.stream>>>((const Id*)ids, (int)d.rows, d.vocab, (int32_t*)g.key, (int32_t*)g.pos, pass.touched, g.crossing);
        ++*c.launches;
      } else if (!p.spread) {
        auto* sort = k_sort_tokens<Id>;
        err = allow(sort);
        if (err != cudaSuccess) return;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)p.ranks);
        cfg.blockDim = dim3(kSortBlock);
        cfg.dynamicSmemBytes = sizeof(SortShared);
        cfg.stream = c.stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)p.ranks;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        err = cudaLaunchKernelEx(&cfg, sort, pass, p.passes, a, b, g.crossing);
        if (err != cudaSuccess) return;
        ++*c.launches;
      } else {
        auto* count = k_count_tokens<Id>;
        auto* place = k_place_tokens<Id>;
        err = allow(count);
        if (err == cudaSuccess) err = allow(place);
        if (err != cudaSuccess) return;
        uint32_t* totals = (uint32_t*)(w + p.totals);
        for (int k = 0; k < p.passes; ++k) {
          pass.from = k == 0 ? nullptr : k % 2 ? a : b;
          pass.to = k % 2 ? b : a;
          pass.shift = k * p.digit;
          count<<<p.ranks, kSortBlock, sizeof(SortShared), c.stream>>>(pass, totals, g.crossing);
          place<<<p.ranks, kSortBlock, sizeof(SortShared), c.stream>>>(pass, totals);
          *c.launches += 2;
        }
      }
    } else {
      g.chunk_blocks = 0;
    }
    auto* sum = vec ? k_sum_runs<In, Out, true> : k_sum_runs<In, Out, false>;
    sum<<<(unsigned)(g.chunk_blocks * g.slices + fill_blocks), kBlock, 0, c.stream>>>((const In*)dy, (Out*)out, g);
    ++*c.launches;
    if (g.chunks > 1) {
      const int64_t most = g.chunks * ((d.cols + kBlock - 1) / kBlock);
      k_join_runs<Out><<<(unsigned)std::min<int64_t>(most, (int64_t)c.sm_count * 8), kBlock, 0, c.stream>>>((Out*)out, g);
      ++*c.launches;
    }
  });
  return err != cudaSuccess ? err : cudaGetLastError();
}

}  // namespace rx
