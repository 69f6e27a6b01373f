// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//   forward   y[r] = scale * W[ids[r]]          (ids outside [0, V): a row of zeros, nothing is read)
//   backward  dW[v] = scale * sum over the rows r with ids[r] == v of dy[r]
// The forward is bound by the stores of y.  The backward reads every dy row once: the tokens are put in the order of their ids by a
// stable radix sort (8 bits a pass) and runs of equal ids are summed in fp32 in that order, so the result does not depend on
// scheduling and the work does not depend on how the ids are spread: a row of the table that half of all tokens point at is cut into
// the same chunks as any others, and what a chunk holds of a run that it shares with its neighbours is joined by a second kernel.
#include "typed.h"
#include <algorithm>

namespace {

constexpr int RADIX = 256;
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int TILE = 8192;                      // tokens a sorting block handles: 512 a wave
constexpr int PER_WAVE = TILE / SORT_WAVES;

__device__ __forceinline__ int64_t load_id(const void* ids, int type, int64_t r) {
  switch (type) {
    case MBVAE_ID_I8: return reinterpret_cast<const int8_t*>(ids)[r];
    case MBVAE_ID_U8: return reinterpret_cast<const uint8_t*>(ids)[r];
    case MBVAE_ID_I16: return reinterpret_cast<const int16_t*>(ids)[r];
    case MBVAE_ID_I32: return reinterpret_cast<const int32_t*>(ids)[r];
    default: return reinterpret_cast<const int64_t*>(ids)[r];
  }
}
// Sort key of a token: its id, and V for every id outside the table, so that those come last.
__device__ __forceinline__ uint32_t load_key(const void* ids, int type, int64_t r, uint32_t V) {
  const int64_t id = load_id(ids, type, r);
  return id >= 0 && id < (int64_t)V ? (uint32_t)id : V;
}

// ------------------------------------------------------------------------------------------------ forward
// A team of `lanes` lanes (a power of two) owns a row and walks over it in 16-byte pieces.
template <typename T>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* __restrict__ ids, int id_type, const T* __restrict__ W, T* __restrict__ y,
                                                            int64_t rows, int64_t V, int64_t D, float scale, int lanes) {
  constexpr int N = MbvaeVec<T>::N;
  const int teams = 256 / lanes, team = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  for (int64_t r = (int64_t)blockIdx.x * teams + team; r < rows; r += (int64_t)gridDim.x * teams) {
    const int64_t id = load_id(ids, id_type, r);
    const bool valid = id >= 0 && id < V;
    const T* w = W + (valid ? id : 0) * D;
    for (int64_t c = (int64_t)lane * N; c < D; c += (int64_t)lanes * N) {
      float v[N];
      mbvae_load_vec<T>(w + c, valid ? D - c : 0, v);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] *= scale;
      if (!valid) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = 0.f;           // (a scale that is not finite makes no difference to padding)
      }
      mbvae_store_vec<T>(y + r * D + c, D - c, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort
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

// Exclusive sum over the block's first 256 threads of one value each, through `scan` (RADIX words).  Called by every thread.
__device__ __forceinline__ uint32_t scan_bins(uint32_t mine, uint32_t* scan) {
  const int t = threadIdx.x;
  if (t < RADIX) scan[t] = mine;
  __syncthreads();
  for (int o = 1; o < RADIX; o <<= 1) {
    const uint32_t below = t < RADIX && t >= o ? scan[t - o] : 0;
    __syncthreads();
    if (t < RADIX) scan[t] += below;
    __syncthreads();
  }
  return t < RADIX ? scan[t] - mine : 0;
}

// Fills `values` elements of the table's gradient with zeros: blocks from `first` on of a launch.
template <typename T>
__device__ __forceinline__ void fill_zero(T* p, int64_t values, int64_t block, int64_t blocks) {
  constexpr int N = MbvaeVec<T>::N;
  const float zero[N] = {};
  for (int64_t i = (block * blockDim.x + threadIdx.x) * N; i < values; i += blocks * blockDim.x * N) mbvae_store_vec<T>(p + i, values - i, zero);
}
__device__ __forceinline__ void fill_zero_any(void* p, int dtype, int64_t values, int64_t block, int64_t blocks) {
  if (dtype == MBVAE_F32) fill_zero(reinterpret_cast<float*>(p), values, block, blocks);
  else fill_zero(reinterpret_cast<mbvae_bf16*>(p), values, block, blocks);       // (zero has the same bits in both 16-bit types)
}

// The whole sort of at most TILE tokens in one block, in LDS; every other block of the launch clears the gradient.
// Per pass: the waves count their digits, the counts are turned into each wave's first place per digit, then every wave walks over
// its tokens in order, 64 at a time, and the lanes of one digit take consecutive places.
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_one_kernel(const void* __restrict__ ids, int id_type, uint32_t V, int rows, int passes,
                                                                          uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out,
                                                                          void* __restrict__ dW, int dtype, int64_t values) {
  if (blockIdx.x != 0) {
    fill_zero_any(dW, dtype, values, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  extern __shared__ uint32_t lds[];
  uint32_t* key = lds;                                                  // two buffers of TILE each
  uint16_t* pos = reinterpret_cast<uint16_t*>(lds + 2 * TILE);
  uint32_t* count = lds + 3 * TILE;                 // [SORT_WAVES][RADIX]
  uint32_t* scan = count + SORT_WAVES * RADIX;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < rows; i += SORT_THREADS) {
    key[i] = load_key(ids, id_type, i, V);
    pos[i] = (uint16_t)i;
  }
  const int span = (rows + SORT_WAVES - 1) / SORT_WAVES;
  const int begin = min(rows, wave * span), end = min(rows, begin + span);
  for (int p = 0; p < passes; ++p) {
    const uint32_t* kin = key + (p & 1) * TILE;
    const uint16_t* pin = pos + (p & 1) * TILE;
    uint32_t* kout = key + (~p & 1) * TILE;
    uint16_t* pout = pos + (~p & 1) * TILE;
    const int shift = 8 * p;
    for (int i = threadIdx.x; i < SORT_WAVES * RADIX; i += SORT_THREADS) count[i] = 0;
    __syncthreads();
    for (int i = begin + lane; i < end; i += 64) atomicAdd(&count[wave * RADIX + ((kin[i] >> shift) & 255)], 1u);
    __syncthreads();
    uint32_t total = 0;
    if (threadIdx.x < RADIX)
      for (int w = 0; w < SORT_WAVES; ++w) {
        const uint32_t c = count[w * RADIX + threadIdx.x];
        count[w * RADIX + threadIdx.x] = total;
        total += c;
      }
    const uint32_t first = scan_bins(total, scan);
    if (threadIdx.x < RADIX)
      for (int w = 0; w < SORT_WAVES; ++w) count[w * RADIX + threadIdx.x] += first;
    __syncthreads();
    for (int i0 = begin; i0 < end; i0 += 64) {
      const int i = i0 + lane;
      const bool in = i < end;
      const uint32_t k = in ? kin[i] : 0, d = (k >> shift) & 255;
      const uint64_t same = same_digit(d, __ballot(in));
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const uint32_t at = in ? count[wave * RADIX + d] + rank : 0;
      if (in) {
        kout[at] = k;
        pout[at] = pin[i];
        if (rank == 0) count[wave * RADIX + d] += (uint32_t)__popcll(same);
      }
      wave_order();
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < rows; i += SORT_THREADS) {
    keys_out[i] = key[(passes & 1) * TILE + i];
    pos_out[i] = pos[(passes & 1) * TILE + i];
  }
}

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
// A team of `lanes` lanes (<= 64, a power of two) sums one chunk of sorted tokens over lanes * N columns (blockIdx.y: which).
// A run that begins and ends in the chunk goes to the gradient.  What the chunk holds of a run that began in an earlier chunk goes to
// part[chunk][0], of one that begins here and goes on in the next to part[chunk][1].
template <typename T>
__global__ __launch_bounds__(256) void embedding_runs_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos, const T* __restrict__ dy,
                                                             int64_t ldy, T* __restrict__ dW, float* __restrict__ part, int64_t rows, uint32_t V, int64_t D,
                                                             float scale, int chunk, int64_t chunks, int lanes) {
  constexpr int N = MbvaeVec<T>::N, AHEAD = 4;
  const int teams = 256 / lanes, team = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const int64_t c = (int64_t)blockIdx.x * teams + team;
  const int64_t col = ((int64_t)blockIdx.y * lanes + lane) * N;
  if (c >= chunks || col >= D) return;
  const int64_t begin = c * chunk, end = min(rows, begin + chunk), left = D - col;
  uint32_t cur = keys[begin];
  bool continued = begin > 0 && keys[begin - 1] == cur;
  float acc[N] = {};
  for (int64_t i = begin; i < end && cur < V; i += AHEAD) {
    uint32_t k[AHEAD];
    float v[AHEAD][N];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int64_t j = min(i + a, end - 1);
      k[a] = i + a < end ? keys[j] : V;
      mbvae_load_vec<T>(dy + (int64_t)pos[j] * ldy + col, k[a] < V ? left : 0, v[a]);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i + a >= end || cur >= V) break;
      if (k[a] != cur) {                                    // the run ended inside the chunk
        if (continued) {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (e < left) part[(c * 2) * D + col + e] = acc[e];
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) acc[e] *= scale;
          mbvae_store_vec<T>(dW + (int64_t)cur * D + col, left, acc);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.f;
        continued = false;
        cur = k[a];
        if (cur >= V) break;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += v[a][e];
    }
  }
  if (cur >= V) return;
  const bool goes_on = end < rows && keys[end] == cur;
  if (continued || goes_on) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left) part[(c * 2 + (continued ? 0 : 1)) * D + col + e] = acc[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= scale;
    mbvae_store_vec<T>(dW + (int64_t)cur * D + col, left, acc);
  }
}

// Runs that cross chunks: the block of the chunk in which such a run begins adds up what the chunks hold of it, JOIN_GROUPS waves of
// 64 columns taking every JOIN_GROUPS-th chunk, joined in LDS in a fixed order.
constexpr int JOIN_GROUPS = 16;
template <typename T>
__global__ __launch_bounds__(64 * JOIN_GROUPS) void embedding_join_kernel(const uint32_t* __restrict__ keys, const float* __restrict__ part,
                                                                          T* __restrict__ dW, int64_t rows, uint32_t V, int64_t D, float scale, int chunk) {
  const int64_t c = blockIdx.x;
  const int64_t end = min(rows, (c + 1) * chunk);
  const uint32_t key = keys[end - 1];
  if (key >= V || end >= rows || keys[end] != key) return;                       // the chunk's last run ends in it
  if (keys[c * chunk] == key && c > 0 && keys[c * chunk - 1] == key) return;     // ... or began before it
  int64_t lo = end, hi = rows;                                                   // the first token behind the run
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] > key) hi = mid; else lo = mid + 1;
  }
  const int64_t last = (lo - 1) / chunk;                                         // the chunk that the run ends in
  constexpr int U = 8;
  __shared__ float red[JOIN_GROUPS][64];
  const int lane = threadIdx.x & 63, group = threadIdx.x >> 6;
  for (int64_t col0 = 64 * (int64_t)blockIdx.y; col0 < D; col0 += 64 * (int64_t)gridDim.y) {
    const int64_t col = col0 + lane;
    float s[U] = {};
    if (col < D) {
      if (group == 0) s[0] = part[(c * 2 + 1) * D + col];
      int64_t k = c + 1 + group;
      for (; k + (U - 1) * JOIN_GROUPS <= last; k += U * JOIN_GROUPS) {
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] += part[(k + u * JOIN_GROUPS) * 2 * D + col];
      }
      for (; k <= last; k += JOIN_GROUPS) s[0] += part[k * 2 * D + col];
    }
    __syncthreads();
    red[group][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (group == 0 && col < D) {
      float t = 0.f;
#pragma unroll
      for (int g = 0; g < JOIN_GROUPS; ++g) t += red[g][lane];
      dW[(int64_t)key * D + col] = (T)(t * scale);
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
int lanes_for(int64_t pieces, int most) {
  int l = 1;
  while (l < most && l < pieces) l <<= 1;
  return l;
}

// Tokens a chunk holds.  A chunk is one team's work: enough chunks to fill the chip, and at least 16 tokens so that the two rows of
// partials a chunk may leave stay small next to what it reads.
int chunk_for(int64_t rows, int64_t D) {
  const int64_t slabs = (D + 255) / 256;
  int64_t c = rows * slabs / 8192;
  c = std::max<int64_t>(16, std::min<int64_t>(1024, c));
  return (int)c;
}

struct Plan {
  int64_t tiles, chunks;
  int chunk, passes;
  int64_t keys[2], pos[2], hist, total, part, bytes;       // offsets
};
Plan plan_for(int64_t rows, int64_t V, int64_t D) {
  Plan p;
  p.tiles = (rows + TILE - 1) / TILE;
  p.chunk = chunk_for(rows, D);
  p.chunks = (rows + p.chunk - 1) / p.chunk;
  p.passes = 1;
  while (((uint64_t)V >> (8 * p.passes)) != 0) ++p.passes;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  for (int i = 0; i < 2; ++i) {
    p.keys[i] = take(4 * rows);
    p.pos[i] = take(4 * rows);
  }
  p.hist = take(4 * p.tiles * RADIX);
  p.total = take(4 * RADIX);
  p.part = take(4 * 2 * p.chunks * D);
  p.bytes = at;
  return p;
}

bool id_type_ok(int t) { return t == MBVAE_ID_I8 || t == MBVAE_ID_U8 || t == MBVAE_ID_I16 || t == MBVAE_ID_I32 || t == MBVAE_ID_I64; }

constexpr int64_t MAX_ROWS = (int64_t)1 << 31, MAX_VOCAB = (int64_t)1 << 31, MAX_WIDTH = (int64_t)1 << 23;

template <typename T>
void launch_fwd(const void* ids, int id_type, const void* W, void* y, int64_t rows, int64_t V, int64_t D, float scale, hipStream_t stream) {
  const int lanes = lanes_for((D + MbvaeVec<T>::N - 1) / MbvaeVec<T>::N, 256);
  const int64_t blocks = std::min<int64_t>((rows + 256 / lanes - 1) / (256 / lanes), 16384);
  hipLaunchKernelGGL((embedding_fwd_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, stream, ids, id_type, reinterpret_cast<const T*>(W),
                     reinterpret_cast<T*>(y), rows, V, D, scale, lanes);
}

template <typename T>
void launch_runs(const Plan& p, const uint32_t* keys, const uint32_t* pos, const void* dy, int64_t ldy, void* dW, float* part, int64_t rows, int64_t V,
                 int64_t D, float scale, hipStream_t stream) {
  const int lanes = lanes_for((D + MbvaeVec<T>::N - 1) / MbvaeVec<T>::N, 64);
  const int64_t teams = 256 / lanes, width = (int64_t)lanes * MbvaeVec<T>::N;
  hipLaunchKernelGGL((embedding_runs_kernel<T>), dim3((unsigned)((p.chunks + teams - 1) / teams), (unsigned)((D + width - 1) / width)), dim3(256), 0,
                     stream, keys, pos, reinterpret_cast<const T*>(dy), ldy, reinterpret_cast<T*>(dW), part, rows, (uint32_t)V, D, scale, p.chunk, p.chunks,
                     lanes);
  if (p.chunks > 1)
    hipLaunchKernelGGL((embedding_join_kernel<T>), dim3((unsigned)p.chunks, (unsigned)std::min<int64_t>((D + 63) / 64, 16)), dim3(64 * JOIN_GROUPS), 0,
                       stream, keys, part, reinterpret_cast<T*>(dW), rows, (uint32_t)V, D, scale, p.chunk);
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

int64_t mbvae_embedding_bwd_workspace(int64_t rows, int64_t vocab, int64_t D) {
  if (rows <= 0 || vocab < 0 || D <= 0 || rows >= MAX_ROWS || vocab >= MAX_VOCAB || D > MAX_WIDTH) return 0;
  return plan_for(rows, vocab, D).bytes;
}

int mbvae_embedding_bwd(const void* ids, int id_type, const void* dy, int64_t ldy, void* dweight, int64_t rows, int64_t vocab, int64_t D, float scale,
                        int dtype, void* ws, int64_t ws_bytes, hipStream_t stream) {
  (void)hipGetLastError();  // drop stale (non-sticky) errors left by other runtime users
  if (rows < 0 || vocab < 0 || D < 0 || ldy < 0 || !id_type_ok(id_type) || mbvae_dtype_size(dtype) == 0) return MBVAE_EINVAL;
  if (vocab == 0 || D == 0) return MBVAE_OK;
  if (!dweight || (rows && (!ids || !dy || !ws || ((uintptr_t)ws & 15)))) return MBVAE_EINVAL;
  if (rows >= MAX_ROWS || vocab >= MAX_VOCAB || D > MAX_WIDTH) return MBVAE_EUNSUPPORTED;
  const int64_t values = vocab * D;
  const int64_t fill = std::min<int64_t>(std::max<int64_t>(1, values / (4 * SORT_THREADS * 4)), 512);
  if (rows && ws_bytes < mbvae_embedding_bwd_workspace(rows, vocab, D)) return MBVAE_EINVAL;
  if (rows == 0) {                                          // (a launch without tiles: every block clears)
    hipLaunchKernelGGL(embedding_hist_kernel, dim3((unsigned)fill), dim3(SORT_THREADS), 0, stream, ids, id_type, (uint32_t)vocab, nullptr, 0, 0, 0,
                       nullptr, dweight, dtype, values);
    return mbvae_launch_status();
  }
  const Plan p = plan_for(rows, vocab, D);
  char* w = reinterpret_cast<char*>(ws);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(w + p.keys[0]), reinterpret_cast<uint32_t*>(w + p.keys[1])};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(w + p.pos[0]), reinterpret_cast<uint32_t*>(w + p.pos[1])};
  uint32_t* hist = reinterpret_cast<uint32_t*>(w + p.hist);
  uint32_t* total = reinterpret_cast<uint32_t*>(w + p.total);
  int at = 0;
  if (rows <= TILE) {
    constexpr int LDS = 4 * (3 * TILE + SORT_WAVES * RADIX + RADIX);
    if (!MBVAE_ALLOW_BIG_LDS(embedding_sort_one_kernel)) return MBVAE_ELAUNCH;
    hipLaunchKernelGGL(embedding_sort_one_kernel, dim3((unsigned)(1 + fill)), dim3(SORT_THREADS), LDS, stream, ids, id_type, (uint32_t)vocab, (int)rows,
                       p.passes, keys[0], pos[0], dweight, dtype, values);
  } else {
    for (int pass = 0; pass < p.passes; ++pass) {
      const uint32_t* kin = pass ? keys[at] : nullptr;
      const uint32_t* pin = pass ? pos[at] : nullptr;
      const int to = pass ? 1 - at : 0;
      hipLaunchKernelGGL(embedding_hist_kernel, dim3((unsigned)(p.tiles + (pass ? 0 : fill))), dim3(SORT_THREADS), 0, stream, ids, id_type,
                         (uint32_t)vocab, kin, rows, 8 * pass, (int)p.tiles, hist, dweight, dtype, values);
      hipLaunchKernelGGL(embedding_scan_kernel, dim3(RADIX), dim3(256), 0, stream, hist, total, (int)p.tiles);
      hipLaunchKernelGGL(embedding_scatter_kernel, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, stream, ids, id_type, (uint32_t)vocab, kin, pin, rows,
                         8 * pass, (int)p.tiles, hist, total, keys[to], pos[to]);
      at = to;
    }
  }
  float* part = reinterpret_cast<float*>(w + p.part);
  if (dtype == MBVAE_F32) launch_runs<float>(p, keys[at], pos[at], dy, ldy, dweight, part, rows, vocab, D, scale, stream);
  else if (dtype == MBVAE_BF16) launch_runs<mbvae_bf16>(p, keys[at], pos[at], dy, ldy, dweight, part, rows, vocab, D, scale, stream);
  else launch_runs<mbvae_f16>(p, keys[at], pos[at], dy, ldy, dweight, part, rows, vocab, D, scale, stream);
  return mbvae_launch_status();
}

}  // extern "C"
