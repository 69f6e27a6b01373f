// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//   forward   y[r] = scale * W[ids[r]]          (ids outside [0, V): a row of zeros, nothing is read)
//   backward  dW[v] = scale * sum over the rows r with ids[r] == v of dy[r]
// The forward is bound by the stores of y.  The backward reads every dy row once, whatever the spread of the ids, and adds in an order
// that the ids alone decide (reproducible, no atomics on memory).  Three routes lead there:
//   few classes   every thread keeps its columns of ALL table rows in LDS and adds the dy rows as they come; no order is needed.
//   few tokens    one launch puts the tokens in the order of their ids: each block owns a range of ids, scans all tokens for its own,
//                 counts those of smaller ids on the way - which is where its own begin - and sorts what it found in LDS.
//   otherwise     a stable radix sort, 8 bits a pass.
// Behind either order, runs of equal ids are summed chunk by chunk, so that an id that half of all tokens carry is spread over the chip
// like any others; what the chunks hold of such a run is joined by a second kernel.
#include "typed.h"
#include <algorithm>

namespace {

constexpr int RADIX = 256;
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int TILE = 8192;                      // tokens a sorting block handles: 512 a wave
constexpr int PER_WAVE = TILE / SORT_WAVES;

// Sort key of a token: its id, and V for every id outside the table, so that those come last.  The loads of all types leave whole
// registers that nothing is computed from until key() is called: a loop can have many of them under way.
struct Id {
  uint32_t lo, hi;
  __device__ __forceinline__ uint32_t key(uint32_t V) const { return hi == 0 && lo < V ? lo : V; }     // (a negative id is above 2^31)
};
__device__ __forceinline__ Id load_id(const void* ids, int type, int64_t r) {
  switch (type) {
    case MBVAE_ID_I8: return {(uint32_t)(int32_t)reinterpret_cast<const int8_t*>(ids)[r], 0};
    case MBVAE_ID_U8: return {reinterpret_cast<const uint8_t*>(ids)[r], 0};
    case MBVAE_ID_I16: return {(uint32_t)(int32_t)reinterpret_cast<const int16_t*>(ids)[r], 0};
    case MBVAE_ID_I32: return {reinterpret_cast<const uint32_t*>(ids)[r], 0};
    default: return {reinterpret_cast<const uint32_t*>(ids)[2 * r], reinterpret_cast<const uint32_t*>(ids)[2 * r + 1]};
  }
}
__device__ __forceinline__ uint32_t load_key(const void* ids, int type, int64_t r, uint32_t V) { return load_id(ids, type, r).key(V); }

// ------------------------------------------------------------------------------------------------ forward
// 2^LOG lanes own 16 bytes each of FWD_ROWS rows; a block's rows are neighbours, blockIdx.y counts its columns and blockIdx.z what grid x
// cannot hold.  There is no loop: a
// load behind a store waits for the store (one counter, in order), and a loop over rows spent more on addresses than on moving 16 bytes.
// All ids are asked for before the first table row, and those before the first store.  The pairs of 256 graphs (1 M x 64 fp32):
// 47.5 us = 5.7 TB/s of stores; with the rows in a grid-stride loop 65 us, with 1, 2 or 8 rows a thread 66, 53 and 48 us.
constexpr int FWD_ROWS = 4;
template <typename T, int ID, bool WHOLE>
__device__ __forceinline__ void embedding_fwd_rows(const void* __restrict__ ids, const T* __restrict__ W, T* __restrict__ y, unsigned rows, uint32_t V,
                                                   unsigned D, float scale, int log_lanes) {
  constexpr unsigned N = MbvaeVec<T>::N, U = FWD_ROWS;
  const unsigned teams = 256u >> log_lanes, team = threadIdx.x >> log_lanes, lane = threadIdx.x & ((1u << log_lanes) - 1);
  const unsigned r0 = (blockIdx.z * gridDim.x + blockIdx.x) * (teams * U) + team, col = ((blockIdx.y << log_lanes) + lane) * N;
  if (r0 >= rows || col >= D) return;
  Id id[U];
  typename MbvaeVec<T>::Aligned t[U];
#pragma unroll
  for (unsigned u = 0; u < U; ++u) id[u] = load_id(ids, ID, min(r0 + u * teams, rows - 1));
#pragma unroll
  for (unsigned u = 0; u < U; ++u) {
    const uint32_t k = id[u].key(V);
    id[u].lo = k;
    if (k < V) t[u] = mbvae_load_raw<T>(W + (uint64_t)k * D + col, WHOLE ? N : D - col);
  }
#pragma unroll
  for (unsigned u = 0; u < U; ++u) {
    const unsigned r = r0 + u * teams;
    if (r >= rows) return;
    float v[N];
#pragma unroll
    for (unsigned e = 0; e < N; ++e) v[e] = id[u].lo < V ? (float)t[u][e] * scale : 0.f;      // (padding stays zero whatever the scale)
    mbvae_store_vec<T>(y + (uint64_t)r * D + col, WHOLE ? N : D - col, v);
  }
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* __restrict__ ids, int id_type, const T* __restrict__ W, T* __restrict__ y,
                                                            unsigned rows, uint32_t V, unsigned D, float scale, int log_lanes) {
  switch (id_type) {
    case MBVAE_ID_I8: return embedding_fwd_rows<T, MBVAE_ID_I8, WHOLE>(ids, W, y, rows, V, D, scale, log_lanes);
    case MBVAE_ID_U8: return embedding_fwd_rows<T, MBVAE_ID_U8, WHOLE>(ids, W, y, rows, V, D, scale, log_lanes);
    case MBVAE_ID_I16: return embedding_fwd_rows<T, MBVAE_ID_I16, WHOLE>(ids, W, y, rows, V, D, scale, log_lanes);
    case MBVAE_ID_I32: return embedding_fwd_rows<T, MBVAE_ID_I32, WHOLE>(ids, W, y, rows, V, D, scale, log_lanes);
    default: return embedding_fwd_rows<T, MBVAE_ID_I64, WHOLE>(ids, W, y, rows, V, D, scale, log_lanes);
  }
}

// ------------------------------------------------------------------------------------------------ few classes
// A thread owns N columns and their sums for every class in LDS, four in a cell: cell[class][column / 4][thread].  No two threads share a
// cell, and a wave's 16-byte accesses are consecutive.  Ids outside the table add nothing.  (LDS's own float additions took
// four times as long as reading, adding and writing.)  1 M rows of 64 fp32 values and 5 classes: 53 us = 5.1 TB/s alone, 76 us behind a
// forward whose stores are still on their way to memory; the sorted route 182 us.
template <typename T>
__global__ __launch_bounds__(256) void embedding_few_kernel(const void* __restrict__ ids, int id_type, const T* __restrict__ dy, int64_t ldy,
                                                            float* __restrict__ part, int64_t rows, uint32_t V, int64_t D, int lanes) {
  constexpr int N = MbvaeVec<T>::N, U = 4;
  extern __shared__ float4 cell[];
  const int teams = 256 / lanes, team = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const int64_t col = ((int64_t)blockIdx.y * lanes + lane) * N;
  const int left = (int)(D - col);
  for (uint32_t i = threadIdx.x; i < V * (N / 4) * 256; i += 256) cell[i] = make_float4(0.f, 0.f, 0.f, 0.f);      // (a thread clears its own)
  const int64_t stride = (int64_t)gridDim.x * teams;
  if (left > 0) {
    for (int64_t r0 = (int64_t)blockIdx.x * teams + team; r0 < rows; r0 += U * stride) {
      typename MbvaeVec<T>::Aligned t[U];
      Id id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = min(r0 + u * stride, rows - 1);
        id[u] = load_id(ids, id_type, r);
        t[u] = mbvae_load_raw<T>(dy + r * ldy + col, left);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t k = id[u].key(V);
        if (k >= V || r0 + u * stride >= rows) continue;
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
          float4* c = cell + (k * (N / 4) + q) * 256 + threadIdx.x;
          float4 s = *c;
          s.x += (float)t[u][4 * q]; s.y += (float)t[u][4 * q + 1]; s.z += (float)t[u][4 * q + 2]; s.w += (float)t[u][4 * q + 3];
          *c = s;
        }
      }
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < V * N * lanes; i += 256) {
    const uint32_t l = i % lanes, e = i / lanes % N, v = i / (lanes * N);
    const int64_t c = ((int64_t)blockIdx.y * lanes + l) * N + e;
    float s = 0.f;
    for (int k = 0; k < teams; ++k) s += reinterpret_cast<const float*>(&cell[(v * (N / 4) + e / 4) * 256 + k * lanes + l])[e % 4];
    if (c < D) part[((int64_t)blockIdx.x * V + v) * D + c] = s;
  }
}

// dW = scale * sum of the blocks' tables: 8 values x 32 groups of blocks, joined in order.
template <typename T>
__global__ __launch_bounds__(256) void embedding_few_join_kernel(const float* __restrict__ part, T* __restrict__ dW, int blocks, int64_t values, float scale) {
  __shared__ float red[32][9];
  const int cx = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int64_t c = (int64_t)blockIdx.x * 8 + cx;
  float a[8] = {};
  if (c < values) {
    int b = g;
    for (; b + 7 * 32 < blocks; b += 8 * 32) {
#pragma unroll
      for (int q = 0; q < 8; ++q) a[q] += part[(b + 32 * q) * values + c];
    }
    for (; b < blocks; b += 32) a[0] += part[b * values + c];
  }
  red[g][cx] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  __syncthreads();
  if (g == 0 && c < values) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][cx];
    dW[c] = (T)(t * scale);
  }
}

// ------------------------------------------------------------------------------------------------ places by digit
// Lanes of the wave with this lane's digit (of the lanes in `active`).
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint64_t active) {
  uint64_t m = active;
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1);
    m &= (digit >> b) & 1 ? set : ~set;
  }
  return m;
}

// What one lane of the wave wrote to LDS before is seen by the others behind.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Exclusive sum over the block's first 256 threads of one value each; `scan`: 4 words.  Called by every thread.
__device__ __forceinline__ uint32_t scan_bins(uint32_t mine, uint32_t* scan) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t sum = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t below = __shfl_up(sum, o, 64);
    if (lane >= o) sum += below;
  }
  if (wave < RADIX / 64 && lane == 63) scan[wave] = sum;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < RADIX / 64 - 1; ++w) before += w < wave ? scan[w] : 0;
  return before + sum - mine;
}

// Fills `values` elements of the table's gradient with zeros: blocks from `first` on of a launch.
template <typename T>
__device__ __forceinline__ void fill_zero(T* p, int64_t values, int64_t block, int64_t blocks) {
  constexpr int N = MbvaeVec<T>::N;
  const float zero[N] = {};
  for (int64_t i = (block * blockDim.x + threadIdx.x) * N; i < values; i += blocks * blockDim.x * N)
    mbvae_store_vec<T>(p + i, (int)min(values - i, (int64_t)N), zero);         // (what is left of a table may not fit 32 bits)
}
__device__ __forceinline__ void fill_zero_any(void* p, int dtype, int64_t values, int64_t block, int64_t blocks) {
  if (dtype == MBVAE_F32) fill_zero(reinterpret_cast<float*>(p), values, block, blocks);
  else fill_zero(reinterpret_cast<mbvae_bf16*>(p), values, block, blocks);       // (zero has the same bits in both 16-bit types)
}

// ------------------------------------------------------------------------------------------------ few tokens: order in one launch
// Block b puts the tokens with keys in [b * range, (b + 1) * range) in order (range <= 256) and clears the gradient rows of its keys
// that no token has.  Every wave scans a 16th of all tokens; its finds (place | local key << 16) go to its own part of the list.
// 21 248 tokens of 4170 ids: 15.7 us, 16 384 of 32 000: 19.9 us with the clearing of 48 MB; the radix sort 54 and 62 us.
constexpr int ORDER_TOKENS = 32768;             // list entries: 128 KB of LDS, places fit 16 bits
constexpr int ORDER_BLOCKS = 256;               // of a table of up to 65 536 rows; larger ones take blocks of 256 rows each
constexpr int64_t ORDER_VOCAB = (int64_t)1 << 18;
constexpr int ORDER_COUNTERS = SORT_WAVES * RADIX + 2 * RADIX + SORT_WAVES;
static_assert(4 * (ORDER_TOKENS + ORDER_COUNTERS) <= MBVAE_LDS_LIMIT, "LDS of one block");

template <typename T>
__global__ __launch_bounds__(SORT_THREADS) void embedding_order_kernel(const void* __restrict__ ids, int id_type, uint32_t V, int rows, uint32_t range,
                                                                       int span, uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out,
                                                                       T* __restrict__ dW, int64_t D) {
  extern __shared__ uint32_t list[];              // [SORT_WAVES][span], then the counters
  uint32_t* count = list + SORT_WAVES * span;     // [SORT_WAVES][RADIX]
  uint32_t* scan = count + SORT_WAVES * RADIX;
  uint32_t* total = scan + RADIX;
  uint32_t* less = total + RADIX;                 // [SORT_WAVES]
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t lo = blockIdx.x * range, hi = min(V + 1, lo + range);
  uint32_t* mine = list + wave * span;
  for (int i = threadIdx.x; i < SORT_WAVES * RADIX; i += SORT_THREADS) count[i] = 0;
  const int begin = min(rows, wave * span), end = min(rows, begin + span);
  int found = 0;
  uint32_t smaller = 0;
  constexpr int AHEAD = 16;
  for (int i0 = begin; i0 < end; i0 += 64 * AHEAD) {
    Id id[AHEAD];
    uint32_t k[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) id[a] = load_id(ids, id_type, min(i0 + a * 64 + lane, end - 1));
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) k[a] = i0 + a * 64 + lane < end ? id[a].key(V) : 0xffffffffu;
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const bool own = k[a] >= lo && k[a] < hi;
      const uint64_t owned = __ballot(own);
      smaller += (uint32_t)__popcll(__ballot(k[a] < lo));
      if (own) mine[found + __popcll(owned & ((1ull << lane) - 1))] = (uint32_t)(i0 + a * 64 + lane) | (k[a] - lo) << 16;
      found += __popcll(owned);
    }
  }
  if (lane == 0) less[wave] = smaller;
  __syncthreads();
  for (int i0 = 0; i0 < found; i0 += 64) {
    const bool in = i0 + lane < found;
    const uint32_t d = in ? mine[i0 + lane] >> 16 : 0;
    const uint64_t same = same_digit(d, __ballot(in));
    if (in && (same & ((1ull << lane) - 1)) == 0) count[wave * RADIX + d] += (uint32_t)__popcll(same);
    wave_order();
  }
  __syncthreads();
  uint32_t sum = 0;
  if (threadIdx.x < RADIX) {
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) sum += count[w * RADIX + threadIdx.x];
    total[threadIdx.x] = sum;
  }
  uint32_t at = scan_bins(sum, scan);
  if (threadIdx.x < RADIX) {
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) at += less[w];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const uint32_t c = count[w * RADIX + threadIdx.x];
      count[w * RADIX + threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i0 = 0; i0 < found; i0 += 64) {
    const bool in = i0 + lane < found;
    const uint32_t entry = in ? mine[i0 + lane] : 0, d = entry >> 16;
    const uint64_t same = same_digit(d, __ballot(in));
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (in) {
      const uint32_t to = count[wave * RADIX + d] + rank;
      keys_out[to] = lo + d;
      pos_out[to] = entry & 0xffff;
      if (rank == 0) count[wave * RADIX + d] += (uint32_t)__popcll(same);
    }
    wave_order();
  }
  // rows without a token: a wave each
  const float zero[MbvaeVec<T>::N] = {};
  for (uint32_t k = lo + wave; k < min(hi, V); k += SORT_WAVES)
    if (total[k - lo] == 0)
      for (int64_t c = (int64_t)lane * MbvaeVec<T>::N; c < D; c += 64 * MbvaeVec<T>::N) mbvae_store_vec<T>(dW + (int64_t)k * D + c, (int)(D - c), zero);
}

// ------------------------------------------------------------------------------------------------ many tokens: radix sort
// One pass over more tokens, first half: digits of every tile.  hist[digit][tile].  keys == null: the keys come from the ids (first pass),
// and the blocks behind the tiles clear the gradient.
__global__ __launch_bounds__(SORT_THREADS) void embedding_hist_kernel(const void* __restrict__ ids, int id_type, uint32_t V, const uint32_t* __restrict__ keys,
                                                                      int64_t rows, int shift, int tiles, uint32_t* __restrict__ hist,
                                                                      void* __restrict__ dW, int dtype, int64_t values) {
  if ((int)blockIdx.x >= tiles) {
    fill_zero_any(dW, dtype, values, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  __shared__ uint32_t count[RADIX];
  if (threadIdx.x < RADIX) count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * TILE;
#pragma unroll
  for (int j = 0; j < TILE / SORT_THREADS; ++j) {
    const int64_t i = base + j * SORT_THREADS + threadIdx.x;
    const bool in = i < rows;
    const uint32_t d = in ? ((keys ? keys[i] : load_key(ids, id_type, i, V)) >> shift) & 255 : 0;
    const uint64_t same = same_digit(d, __ballot(in));               // one addition per digit and wave: a common id would queue otherwise
    if (in && (same & ((1ull << (threadIdx.x & 63)) - 1)) == 0) atomicAdd(&count[d], (uint32_t)__popcll(same));
  }
  __syncthreads();
  if (threadIdx.x < RADIX) hist[(int64_t)threadIdx.x * tiles + blockIdx.x] = count[threadIdx.x];
}

// Second: hist[digit][tile] becomes the number of tokens of that digit in the tiles before, total[digit] their number in all.
__global__ __launch_bounds__(256) void embedding_scan_kernel(uint32_t* __restrict__ hist, uint32_t* __restrict__ total, int tiles) {
  __shared__ uint32_t part[256];
  uint32_t* h = hist + (int64_t)blockIdx.x * tiles;
  uint32_t carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + threadIdx.x;
    const uint32_t mine = t < tiles ? h[t] : 0;
    part[threadIdx.x] = mine;
    __syncthreads();
    for (int o = 1; o < 256; o <<= 1) {
      const uint32_t below = (int)threadIdx.x >= o ? part[threadIdx.x - o] : 0;
      __syncthreads();
      part[threadIdx.x] += below;
      __syncthreads();
    }
    if (t < tiles) h[t] = carry + part[threadIdx.x] - mine;
    carry += part[255];
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// Third: every tile's tokens to their places.  Stable: waves own consecutive tokens and walk over them in order.
__global__ __launch_bounds__(SORT_THREADS) void embedding_scatter_kernel(const void* __restrict__ ids, int id_type, uint32_t V,
                                                                         const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, int64_t rows,
                                                                         int shift, int tiles, const uint32_t* __restrict__ hist,
                                                                         const uint32_t* __restrict__ total, uint32_t* __restrict__ keys_out,
                                                                         uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t count[SORT_WAVES * RADIX];
  __shared__ uint32_t scan[RADIX];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t base = (int64_t)blockIdx.x * TILE + wave * PER_WAVE;
  for (int i = threadIdx.x; i < SORT_WAVES * RADIX; i += SORT_THREADS) count[i] = 0;
  __syncthreads();
  uint32_t k[PER_WAVE / 64];
#pragma unroll
  for (int j = 0; j < PER_WAVE / 64; ++j) {
    const int64_t i = base + j * 64 + lane;
    const bool in = i < rows;
    k[j] = in ? (keys ? keys[i] : load_key(ids, id_type, i, V)) : 0;
    const uint32_t d = (k[j] >> shift) & 255;
    const uint64_t same = same_digit(d, __ballot(in));
    if (in && (same & ((1ull << lane) - 1)) == 0) atomicAdd(&count[wave * RADIX + d], (uint32_t)__popcll(same));
  }
  __syncthreads();
  const uint32_t first = scan_bins(threadIdx.x < RADIX ? total[threadIdx.x] : 0, scan);
  if (threadIdx.x < RADIX) {
    uint32_t at = first + hist[(int64_t)threadIdx.x * tiles + blockIdx.x];
    for (int w = 0; w < SORT_WAVES; ++w) {
      const uint32_t c = count[w * RADIX + threadIdx.x];
      count[w * RADIX + threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER_WAVE / 64; ++j) {
    const int64_t i = base + j * 64 + lane;
    const bool in = i < rows;
    const uint32_t d = (k[j] >> shift) & 255;
    const uint64_t same = same_digit(d, __ballot(in));
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (in) {
      const uint32_t at = count[wave * RADIX + d] + rank;
      keys_out[at] = k[j];
      pos_out[at] = pos ? pos[i] : (uint32_t)i;
      if (rank == 0) count[wave * RADIX + d] += (uint32_t)__popcll(same);
    }
    wave_order();
  }
}

// ------------------------------------------------------------------------------------------------ sums over runs of equal ids
// Sorted tokens are cut into chunks; a team of `lanes` lanes (<= 64, a power of two) sums one chunk over lanes * N columns (blockIdx.y:
// which).  A run belongs to the chunk that it begins in, and the team follows it behind the chunk's end.  Only a run that covers a whole
// chunk other than its first - it is longer than a chunk then - is left in pieces: each chunk's piece goes to part[chunk][0], its
// first to part[chunk][1], and the join adds them up.  A team so has at most two chunks of rows to add.  Bound by the latency of
// key -> place -> row: the keys at both ends and the first tokens are asked for at once, the next tokens before the rows are added up
// (21 248 rows of 512 bf16 values 14.4 us, 16 384 of 1024: 18.6 us = 1.8 TB/s; the join 5 us, most blocks of which end at once).
template <typename T>
__global__ __launch_bounds__(256) void embedding_runs_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, const T* __restrict__ dy,
                                                             int64_t ldy, T* __restrict__ dW, float* __restrict__ part, int64_t rows, uint32_t V, int64_t D,
                                                             float scale, int chunk, int64_t chunks, int lanes) {
  constexpr int N = MbvaeVec<T>::N, AHEAD = 8;
  constexpr uint32_t NONE = 0xffffffffu;
  const int teams = 256 / lanes, team = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const int64_t c = (int64_t)blockIdx.x * teams + team;
  const int64_t col = ((int64_t)blockIdx.y * lanes + lane) * N;
  if (c >= chunks || col >= D) return;
  const int64_t begin = c * chunk, end = min(rows, begin + chunk), far = min(rows, end + chunk);
  const int left = (int)(D - col);
  // the first tokens, and the keys at both ends of this chunk and its neighbours: all on their way before any is looked at
  uint32_t k[AHEAD], p[AHEAD];
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) {
    k[a] = keys[min(begin + a, rows - 1)];
    p[a] = pos[min(begin + a, rows - 1)];
  }
  const uint32_t earlier = keys[max(begin - chunk - 1, (int64_t)0)], before = keys[max(begin - 1, (int64_t)0)], first = k[0], last = keys[end - 1],
                 next = keys[min(end, rows - 1)], at_far = keys[far - 1];
  const bool continued = begin > 0 && before == first;
  // The run that the chunk begins in the middle of is left in pieces if it covers this chunk, or began before the one before and so
  // covers that; otherwise the chunk before sums it.
  const bool piece_first = continued && (last == first || (begin > chunk && earlier == first));
  const uint32_t skip = continued && !piece_first ? first : NONE;
  // The run that goes on behind the chunk: followed to its end unless it is left in pieces.
  const bool goes_on = end < rows && last < V && next == last && !(continued && last == first);
  const bool piece_last = goes_on && at_far == last;
  const int64_t stop = goes_on && !piece_last ? far : end;

  float acc[N] = {};
  uint32_t cur = NONE;
  const auto flush = [&]() {
    const bool to_first = piece_first && cur == first, to_last = piece_last && cur == last;
    if (to_first || to_last) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < left) part[(c * 2 + (to_first ? 0 : 1)) * D + col + e] = acc[e];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] *= scale;
      mbvae_store_vec<T>(dW + (int64_t)cur * D + col, left, acc);
    }
  };
  for (int64_t i = begin; i < stop; i += AHEAD) {
    typename MbvaeVec<T>::Aligned t[AHEAD];
    bool on[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      // (behind the chunk only its last run goes on)
      on[a] = i + a < stop && k[a] < V && k[a] != skip && (i + a < end || k[a] == last);
      t[a] = mbvae_load_raw<T>(dy + (int64_t)p[a] * ldy + col, on[a] ? left : 0);
    }
    uint32_t kn[AHEAD], pn[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      kn[a] = keys[min(i + AHEAD + a, rows - 1)];
      pn[a] = pos[min(i + AHEAD + a, rows - 1)];
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (!on[a]) continue;
      if (k[a] != cur) {
        if (cur != NONE) flush();
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.f;
        cur = k[a];
      }
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += (float)t[a][e];
    }
    if (k[AHEAD - 1] >= V) break;                                       // (only padding is left)
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) { k[a] = kn[a]; p[a] = pn[a]; }
  }
  if (cur != NONE) flush();
}

// Runs in pieces: the block of the chunk in which such a run begins adds its pieces up, 64 lanes of four columns each for every
// JOIN_GROUPS-th chunk, joined in LDS in a fixed order.  All other blocks see after a few keys that they have nothing to do.
constexpr int JOIN_GROUPS = 8, JOIN_COLUMNS = 256;
template <typename T>
__global__ __launch_bounds__(64 * JOIN_GROUPS) void embedding_join_kernel(const uint32_t* __restrict__ keys, const float* __restrict__ part,
                                                                          T* __restrict__ dW, int64_t rows, uint32_t V, int64_t D, float scale, int chunk) {
  const int64_t c = blockIdx.x, begin = c * chunk, end = min(rows, begin + chunk);
  const uint32_t key = keys[end - 1], next = keys[min(end, rows - 1)], at_far = keys[min(rows, end + chunk) - 1], first = keys[begin],
                 before = keys[max(begin - 1, (int64_t)0)];
  if (key >= V || end >= rows || next != key || at_far != key) return;                  // no run in pieces leaves the chunk
  if (begin > 0 && first == key && before == key) return;                               // ... or it began before
  constexpr int U = 4;
  __shared__ float4 red[JOIN_GROUPS][64];
  const int lane = threadIdx.x & 63, group = threadIdx.x >> 6;
  for (int64_t col0 = JOIN_COLUMNS * (int64_t)blockIdx.y; col0 < D; col0 += JOIN_COLUMNS * (int64_t)gridDim.y) {
    const int64_t col = col0 + 4 * lane;
    const int left = (int)(D - col);
    float s[U][4] = {};
    if (left > 0) {
      if (group == 0) mbvae_load_vec<float>(part + (c * 2 + 1) * D + col, left, s[0]);
      for (int64_t k = c + 1 + group;; k += U * JOIN_GROUPS) {
        uint32_t head[U];
        float v[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t q = min(k + u * JOIN_GROUPS, (rows - 1) / chunk);
          head[u] = k + u * JOIN_GROUPS == q ? keys[q * chunk] : V;
          mbvae_load_vec<float>(part + q * 2 * D + col, left, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][e] += head[u] == key ? v[u][e] : 0.f;        // (behind the run the piece is another's, or nobody's)
        if (head[U - 1] != key) break;
      }
    }
    __syncthreads();
    red[group][lane] = make_float4((s[0][0] + s[1][0]) + (s[2][0] + s[3][0]), (s[0][1] + s[1][1]) + (s[2][1] + s[3][1]),
                                   (s[0][2] + s[1][2]) + (s[2][2] + s[3][2]), (s[0][3] + s[1][3]) + (s[2][3] + s[3][3]));
    __syncthreads();
    const int64_t mine = col0 + threadIdx.x;
    if (threadIdx.x < JOIN_COLUMNS && mine < D) {
      float t = 0.f;
#pragma unroll
      for (int g = 0; g < JOIN_GROUPS; ++g) t += reinterpret_cast<const float*>(&red[g][0])[threadIdx.x];
      dW[(int64_t)key * D + mine] = (T)(t * scale);
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
int lanes_for(int64_t pieces, int most) {
  int l = 1;
  while (l < most && l < pieces) l <<= 1;
  return l;
}

// Blocks of 256 threads over grid x and z: a grid has at most 2^32 - 1 threads along each of its sides.
dim3 grid_of(int64_t blocks) {
  const int64_t sheets = (blocks + (1 << 23) - 1) >> 23;
  return dim3((unsigned)((blocks + sheets - 1) / sheets), 1, (unsigned)sheets);
}

// Tokens a chunk holds.  A chunk is one team's work: enough chunks to fill the chip, and at least 16 tokens so that the two rows of
// partials a chunk may leave stay small next to what it reads.
int chunk_for(int64_t rows, int64_t D) {
  const int64_t slabs = (D + 255) / 256;
  int64_t c = rows * slabs / 8192;
  c = std::max<int64_t>(16, std::min<int64_t>(1024, c));
  return (int)c;
}

// Blocks that clear `values` elements.
int64_t clear_blocks(int64_t values) { return std::min<int64_t>(std::max<int64_t>(1, values / (4 * SORT_THREADS * 4)), 512); }

// The route (see the top): few tokens while the list of one block fits LDS; few classes while their cells do and the blocks' tables stay small
// next to what an ordering costs.  Near FEW_CELLS a block adds up no more rows than its table has, so that many blocks of wide tables would
// write, and read again, as much as dy holds.  Few classes / ordered, us, fp32: 16 384 rows of 5 x 512 16.5 / 30.4, 5 x 1024 25 / 37,
// 8 x 1024 34 / 34, 12 x 512 29 / 25, 32 x 128 17 / 20, 32 x 512 85 / 24; 4096 rows of 5 x 4096 25 / 31, 8 x 4096 34 / 33, 32 x 256 22 / 18;
// 131 072 of 5 x 1024 156 / 174, 16 x 512 110 / 97; bf16: 16 384 rows of 16 x 256 17 / 23, 8 x 512 22 / 27, 12 x 512 38 / 26, 131 072 of
// 8 x 512 58 / 77, 12 x 512 108 / 74.  One or two classes are never worth an order: 16 384 rows of 2 x 4096 67 / 91 and 46 / 72.
enum Route { FEW_CLASSES, FEW_TOKENS, RADIX_SORT };
constexpr int64_t FEW_CELLS = 128;              // columns a thread x classes: 128 KB of LDS
constexpr int64_t FEW_BLOCKS = 1024;
constexpr int64_t FEW_PARTIALS = 5120 * 512;    // values in the tables of the first 512 blocks (more blocks have rows enough each)
template <typename T>
constexpr int vec() { return MbvaeVec<T>::N; }
int vec_of(int dtype) { return dtype == MBVAE_F32 ? vec<float>() : vec<mbvae_bf16>(); }

struct Plan {
  Route route;
  int64_t blocks, tiles, chunks;
  int chunk, passes, lanes;
  int64_t keys[2], pos[2], hist, total, part, bytes;       // offsets
};
Plan plan_for(int64_t rows, int64_t V, int64_t D, int dtype) {
  Plan p = {};
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  p.lanes = lanes_for((D + vec_of(dtype) - 1) / vec_of(dtype), 64);
  const int64_t teams = 256 / p.lanes, few_blocks = std::max<int64_t>(1, std::min<int64_t>(FEW_BLOCKS, (rows + 8 * teams - 1) / (8 * teams)));
  if (V * vec_of(dtype) <= FEW_CELLS && (V <= 2 || V * D * std::min<int64_t>(few_blocks, 512) <= FEW_PARTIALS)) p.route = FEW_CLASSES;
  else p.route = rows <= ORDER_TOKENS && V < ORDER_VOCAB ? FEW_TOKENS : RADIX_SORT;
  if (p.route == FEW_CLASSES) {
    p.blocks = few_blocks;
    p.part = take(4 * p.blocks * V * D);
  } else {
    p.chunk = chunk_for(rows, D);
    p.chunks = (rows + p.chunk - 1) / p.chunk;
    p.part = take(4 * 2 * p.chunks * D);
    for (int i = 0; i < (p.route == FEW_TOKENS ? 1 : 2); ++i) {
      p.keys[i] = take(4 * rows);
      p.pos[i] = take(4 * rows);
    }
  }
  if (p.route == RADIX_SORT) {
    p.tiles = (rows + TILE - 1) / TILE;
    p.passes = 1;
    while (((uint64_t)V >> (8 * p.passes)) != 0) ++p.passes;
    p.hist = take(4 * p.tiles * RADIX);
    p.total = take(4 * RADIX);
  }
  p.bytes = at;
  return p;
}

bool id_type_ok(int t) { return t == MBVAE_ID_I8 || t == MBVAE_ID_U8 || t == MBVAE_ID_I16 || t == MBVAE_ID_I32 || t == MBVAE_ID_I64; }

constexpr int64_t MAX_ROWS = (int64_t)1 << 31, MAX_VOCAB = (int64_t)1 << 31, MAX_WIDTH = (int64_t)1 << 23;

template <typename T>
void launch_fwd(const void* ids, int id_type, const void* W, void* y, int64_t rows, int64_t V, int64_t D, float scale, hipStream_t stream) {
  const int lanes = lanes_for((D + vec<T>() - 1) / vec<T>(), 256), log_lanes = __builtin_ctz(lanes);
  const int64_t block_rows = FWD_ROWS * (256 / lanes), width = (int64_t)lanes * vec<T>();
  dim3 grid = grid_of((rows + block_rows - 1) / block_rows);
  grid.y = (unsigned)((D + width - 1) / width);
  if (D % vec<T>() == 0)
    hipLaunchKernelGGL((embedding_fwd_kernel<T, true>), grid, dim3(256), 0, stream, ids, id_type, reinterpret_cast<const T*>(W), reinterpret_cast<T*>(y),
                       (unsigned)rows, (uint32_t)V, (unsigned)D, scale, log_lanes);
  else
    hipLaunchKernelGGL((embedding_fwd_kernel<T, false>), grid, dim3(256), 0, stream, ids, id_type, reinterpret_cast<const T*>(W), reinterpret_cast<T*>(y),
                       (unsigned)rows, (uint32_t)V, (unsigned)D, scale, log_lanes);
}

// Everything behind the order of the tokens.
template <typename T>
void launch_runs(const Plan& p, const uint32_t* keys, const uint32_t* pos, const T* dy, int64_t ldy, T* dW, float* part, int64_t rows, int64_t V,
                 int64_t D, float scale, hipStream_t stream) {
  const int64_t teams = 256 / p.lanes, width = (int64_t)p.lanes * vec<T>();
  hipLaunchKernelGGL((embedding_runs_kernel<T>), dim3((unsigned)((p.chunks + teams - 1) / teams), (unsigned)((D + width - 1) / width)), dim3(256), 0,
                     stream, keys, pos, dy, ldy, dW, part, rows, (uint32_t)V, D, scale, p.chunk, p.chunks, p.lanes);
  if (p.chunks > 1)
    hipLaunchKernelGGL((embedding_join_kernel<T>), dim3((unsigned)p.chunks, (unsigned)std::min<int64_t>((D + JOIN_COLUMNS - 1) / JOIN_COLUMNS, 16)), dim3(64 * JOIN_GROUPS),
                       0, stream, keys, part, dW, rows, (uint32_t)V, D, scale, p.chunk);
}

template <typename T>
int launch_bwd(const Plan& p, const void* ids, int id_type, const T* dy, int64_t ldy, T* dW, int dtype, int64_t rows, int64_t V, int64_t D, float scale,
               char* w, hipStream_t stream) {
  float* part = reinterpret_cast<float*>(w + p.part);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(w + p.keys[0]), reinterpret_cast<uint32_t*>(w + p.keys[1])};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(w + p.pos[0]), reinterpret_cast<uint32_t*>(w + p.pos[1])};
  if (p.route == FEW_CLASSES) {
    const int64_t width = (int64_t)p.lanes * vec<T>(), values = V * D;
    if (!MBVAE_ALLOW_BIG_LDS(embedding_few_kernel<T>)) return MBVAE_ELAUNCH;
    hipLaunchKernelGGL((embedding_few_kernel<T>), dim3((unsigned)p.blocks, (unsigned)((D + width - 1) / width)), dim3(256), V * vec<T>() * 1024, stream,
                       ids, id_type, dy, ldy, part, rows, (uint32_t)V, D, p.lanes);
    hipLaunchKernelGGL((embedding_few_join_kernel<T>), dim3((unsigned)((values + 7) / 8)), dim3(256), 0, stream, part, dW, (int)p.blocks, values, scale);
    return mbvae_launch_status();
  }
  if (p.route == FEW_TOKENS) {
    const int64_t range = std::min<int64_t>((V + ORDER_BLOCKS) / ORDER_BLOCKS, RADIX);          // keys 0..V shared out over the blocks
    const int span = (int)((rows + 64 * SORT_WAVES - 1) / (64 * SORT_WAVES)) * 64;
    if (!MBVAE_ALLOW_BIG_LDS(embedding_order_kernel<T>)) return MBVAE_ELAUNCH;
    hipLaunchKernelGGL((embedding_order_kernel<T>), dim3((unsigned)((V + range) / range)), dim3(SORT_THREADS),
                       4 * (SORT_WAVES * span + ORDER_COUNTERS), stream, ids, id_type,
                       (uint32_t)V, (int)rows, (uint32_t)range, span, keys[0], pos[0], dW, D);
    launch_runs<T>(p, keys[0], pos[0], dy, ldy, dW, part, rows, V, D, scale, stream);
    return mbvae_launch_status();
  }
  uint32_t* hist = reinterpret_cast<uint32_t*>(w + p.hist);
  uint32_t* total = reinterpret_cast<uint32_t*>(w + p.total);
  const int64_t fill = clear_blocks(V * D);
  int at = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    const uint32_t* kin = pass ? keys[at] : nullptr;
    const uint32_t* pin = pass ? pos[at] : nullptr;
    const int to = pass ? 1 - at : 0;
    hipLaunchKernelGGL(embedding_hist_kernel, dim3((unsigned)(p.tiles + (pass ? 0 : fill))), dim3(SORT_THREADS), 0, stream, ids, id_type, (uint32_t)V, kin,
                       rows, 8 * pass, (int)p.tiles, hist, dW, dtype, V * D);
    hipLaunchKernelGGL(embedding_scan_kernel, dim3(RADIX), dim3(256), 0, stream, hist, total, (int)p.tiles);
    hipLaunchKernelGGL(embedding_scatter_kernel, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, stream, ids, id_type, (uint32_t)V, kin, pin, rows,
                       8 * pass, (int)p.tiles, hist, total, keys[to], pos[to]);
    at = to;
  }
  launch_runs<T>(p, keys[at], pos[at], dy, ldy, dW, part, rows, V, D, scale, stream);
  return mbvae_launch_status();
}

}  // namespace

extern "C" {

int mbvae_embedding_fwd(const void* ids, int id_type, const void* weight, void* y, int64_t rows, int64_t vocab, int64_t D, float scale, int dtype,
                        hipStream_t stream) {
  (void)hipGetLastError();  // drop stale (non-sticky) errors left by other runtime users
  if (rows < 0 || vocab < 0 || D < 0 || !id_type_ok(id_type) || mbvae_dtype_size(dtype) == 0) return MBVAE_EINVAL;
  if (rows == 0 || D == 0) return MBVAE_OK;
  if (!ids || !y || (vocab && !weight)) return MBVAE_EINVAL;
  if (rows >= MAX_ROWS || vocab >= MAX_VOCAB || D > MAX_WIDTH) return MBVAE_EUNSUPPORTED;
  if (dtype == MBVAE_F32) launch_fwd<float>(ids, id_type, weight, y, rows, vocab, D, scale, stream);
  else if (dtype == MBVAE_BF16) launch_fwd<mbvae_bf16>(ids, id_type, weight, y, rows, vocab, D, scale, stream);
  else launch_fwd<mbvae_f16>(ids, id_type, weight, y, rows, vocab, D, scale, stream);
  return mbvae_launch_status();
}

int64_t mbvae_embedding_bwd_workspace(int64_t rows, int64_t vocab, int64_t D, int dtype) {
  if (rows <= 0 || vocab <= 0 || D <= 0 || rows >= MAX_ROWS || vocab >= MAX_VOCAB || D > MAX_WIDTH || mbvae_dtype_size(dtype) == 0) return 0;
  return plan_for(rows, vocab, D, dtype).bytes;
}

int mbvae_embedding_bwd(const void* ids, int id_type, const void* dy, int64_t ldy, void* dweight, int64_t rows, int64_t vocab, int64_t D, float scale,
                        int dtype, void* ws, int64_t ws_bytes, hipStream_t stream) {
  (void)hipGetLastError();  // drop stale (non-sticky) errors left by other runtime users
  if (rows < 0 || vocab < 0 || D < 0 || ldy < 0 || !id_type_ok(id_type) || mbvae_dtype_size(dtype) == 0) return MBVAE_EINVAL;
  if (vocab == 0 || D == 0) return MBVAE_OK;
  if (!dweight || (rows && (!ids || !dy || !ws || ((uintptr_t)ws & 15)))) return MBVAE_EINVAL;
  if (rows >= MAX_ROWS || vocab >= MAX_VOCAB || D > MAX_WIDTH) return MBVAE_EUNSUPPORTED;
  if (rows && ws_bytes < mbvae_embedding_bwd_workspace(rows, vocab, D, dtype)) return MBVAE_EINVAL;
  if (rows == 0) {                                          // (a launch without tiles: every block clears)
    hipLaunchKernelGGL(embedding_hist_kernel, dim3((unsigned)clear_blocks(vocab * D)), dim3(SORT_THREADS), 0, stream, ids, id_type, (uint32_t)vocab,
                       nullptr, 0, 0, 0, nullptr, dweight, dtype, vocab * D);
    return mbvae_launch_status();
  }
  const Plan p = plan_for(rows, vocab, D, dtype);
  char* w = reinterpret_cast<char*>(ws);
  if (dtype == MBVAE_F32)
    return launch_bwd(p, ids, id_type, reinterpret_cast<const float*>(dy), ldy, reinterpret_cast<float*>(dweight), dtype, rows, vocab, D, scale, w, stream);
  if (dtype == MBVAE_BF16)
    return launch_bwd(p, ids, id_type, reinterpret_cast<const mbvae_bf16*>(dy), ldy, reinterpret_cast<mbvae_bf16*>(dweight), dtype, rows, vocab, D, scale, w,
                      stream);
  return launch_bwd(p, ids, id_type, reinterpret_cast<const mbvae_f16*>(dy), ldy, reinterpret_cast<mbvae_f16*>(dweight), dtype, rows, vocab, D, scale, w,
                    stream);
}

}  // extern "C"
