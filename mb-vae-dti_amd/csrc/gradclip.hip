// Global norm of a list of gradient tensors and their scaling to a largest norm.
//   norm = (sum |g|^p)^(1/p) over every value of every tensor (p = 1, 2 or infinity), out = g * min(1, max_norm / (norm + 1e-6)).
// The work is one streaming read for the norm and one read + write for the scaling; nothing is computed per tensor.  The tensors are laid
// end to end in units of CHUNK values and every block of a fixed grid takes an equal, contiguous share: it looks its first tensor up
// once and then streams.  A block leaves ONE partial in the workspace, in fp64 (no overflow of a square, no rounding to speak of);
// each scaling block adds the partials up itself, in the same order: reproducible, no atomics, no launch for the join.  The scaling walks
// its share backwards, so that it begins with what the norm has read last and what may still be in the last-level cache.
// The tensor table travels in the kernel arguments, so that a call can be captured into a graph and needs no staging buffer: in those of
// both kernels where it fits (TENSORS), otherwise in those of small kernels that put it together in the workspace.
// Measured: 73 M fp32 values in 472 tensors 89 (3.3 TB/s) + 97 us (6.0 TB/s, in part from the last-level cache) behind three table launches of
// 2-5 us; 302 M bf16 values in nine tensors 142 (4.2 TB/s) + 215 us (5.6 TB/s).  A large copy: 4.7-5.4 TB/s.  512 or 2048 blocks, 2 or 8
// accesses a thread, and chunks dealt out in turn instead of contiguous shares were all within 5 %.
#include "typed.h"
#include <algorithm>
#include <cmath>
#include <limits>
#include <new>

namespace {

constexpr int TENSORS = 160;          // 24 bytes each: the argument block stays below 4 KB
constexpr int CHUNK = 4096;           // values
constexpr int THREADS = 256;
constexpr int BLOCKS = 1024;          // partial sums of one call
constexpr int U = 4;                  // 16-byte accesses a thread has under way

// Tensor i holds the chunks [first(i), first(i + 1)); the last of them has last(i) & 0xffffff values, their type is last(i) >> 24.
struct InlineTable {
  const void* src_[TENSORS];
  void* dst_[TENSORS];
  uint32_t first_[TENSORS + 1], last_[TENSORS];
  int count;
  __device__ __forceinline__ const void* src(int i) const { return src_[i]; }
  __device__ __forceinline__ void* dst(int i) const { return dst_[i]; }
  __device__ __forceinline__ uint32_t first(int i) const { return first_[i]; }
  __device__ __forceinline__ uint32_t last(int i) const { return last_[i]; }
};
static_assert(sizeof(InlineTable) <= 3968, "kernel arguments");
struct MemoryTable {
  const void** src_;
  void** dst_;
  uint32_t *first_, *last_;
  int count;
  __device__ __forceinline__ const void* src(int i) const { return src_[i]; }
  __device__ __forceinline__ void* dst(int i) const { return dst_[i]; }
  __device__ __forceinline__ uint32_t first(int i) const { return first_[i]; }
  __device__ __forceinline__ uint32_t last(int i) const { return last_[i]; }
};

// Entries [at, at + t.count) of the table in memory, whose chunks begin at `chunk`.
__global__ __launch_bounds__(THREADS) void grad_table_kernel(InlineTable t, MemoryTable m, int at, uint32_t chunk) {
  const int i = threadIdx.x;
  if (i < t.count) {
    m.src_[at + i] = t.src_[i];
    m.dst_[at + i] = t.dst_[i];
    m.last_[at + i] = t.last_[i];
  }
  if (i <= t.count) m.first_[at + i] = chunk + t.first_[i];        // (the last one is the next launch's first, with the same value)
}

// Tensor that chunk c belongs to.
template <typename Table>
__device__ __forceinline__ int tensor_of(const Table& t, uint32_t c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first(mid) <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ uint32_t share_begin(uint32_t chunks, uint32_t block, uint32_t blocks) { return (uint32_t)((uint64_t)chunks * block / blocks); }

// f(tensor, its first value here, values here) for the tensors of the chunks [c0, c1), from the first to the last or the other way.
template <bool BACK, typename Table, typename F>
__device__ __forceinline__ void walk(const Table& t, uint32_t c0, uint32_t c1, F f) {
  if (c0 >= c1) return;
  for (int i = tensor_of(t, BACK ? c1 - 1 : c0); c0 < c1; i += BACK ? -1 : 1) {
    const uint32_t first = t.first(i), behind = t.first(i + 1), from = max(c0, first), to = min(c1, behind);
    const int64_t n = (int64_t)(to - from - 1) * CHUNK + (to == behind ? t.last(i) & 0xffffff : CHUNK);      // (else the share ends inside the tensor)
    f(i, (int64_t)(from - first) * CHUNK, n);
    if (BACK) c1 = from;
    else c0 = to;
  }
}

// One value joined to the running partial: P = 1 and 2 sums, P = 0 the largest magnitude (NaN counts as larger than infinity).
template <int P>
__device__ __forceinline__ void take(double& acc, uint32_t& top, float v) {
  if (P == 0) top = max(top, __float_as_uint(v) & 0x7fffffffu);
  else if (P == 1) acc += (double)fabsf(v);
  else acc = fma((double)v, (double)v, acc);
}

template <int P, typename T>
__device__ __forceinline__ void norm_span(const T* p, int64_t n, double* acc, uint32_t& top) {
  constexpr int N = MbvaeVec<T>::N, STEP = THREADS * N;
  typedef typename MbvaeVec<T>::Aligned V;
  typedef typename MbvaeVec<T>::Any A;
  const T* q = p + threadIdx.x * N;
  int64_t left = n;
  const auto add = [&](const V& v) {
#pragma unroll
    for (int e = 0; e < N; ++e) take<P>(acc[e & 3], top, (float)v[e]);
  };
  if (left >= U * STEP) {
    V next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = *reinterpret_cast<const A*>(q + u * STEP);
    while (true) {
      V v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = next[u];
      left -= U * STEP;
      q += U * STEP;
      const bool more = left >= U * STEP;
      if (more)
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = *reinterpret_cast<const A*>(q + u * STEP);
#pragma unroll
      for (int u = 0; u < U; ++u) add(v[u]);
      if (!more) break;
    }
  }
  const int rest = (int)left - threadIdx.x * N;                     // fewer than U * STEP values are left in the block
  V v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = mbvae_load_raw<T>(q + u * STEP, rest - u * STEP);
#pragma unroll
  for (int u = 0; u < U; ++u) add(v[u]);
}

// Sum (or maximum) over the block of 256 threads, valid in every thread; fixed order.
template <int P>
__device__ __forceinline__ double block_join(double a) {
  __shared__ double red[THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double b = __shfl_xor(a, o, 64);
    a = P == 0 ? (b > a || b != b ? b : a) : a + b;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  double s = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) s = P == 0 ? (red[w] > s || red[w] != red[w] ? red[w] : s) : s + red[w];
  return s;
}

template <int P, typename Table>
__global__ __launch_bounds__(THREADS) void grad_norm_kernel(Table t, uint32_t chunks, double* __restrict__ part) {
  double acc[4] = {0., 0., 0., 0.};
  uint32_t top = 0;
  walk<false>(t, share_begin(chunks, blockIdx.x, gridDim.x), share_begin(chunks, blockIdx.x + 1, gridDim.x), [&](int i, int64_t at, int64_t n) {
    const int dtype = t.last(i) >> 24;
    if (dtype == MBVAE_F32) norm_span<P>(reinterpret_cast<const float*>(t.src(i)) + at, n, acc, top);
    else if (dtype == MBVAE_BF16) norm_span<P>(reinterpret_cast<const mbvae_bf16*>(t.src(i)) + at, n, acc, top);
    else norm_span<P>(reinterpret_cast<const mbvae_f16*>(t.src(i)) + at, n, acc, top);
  });
  const double a = block_join<P>(P == 0 ? (double)__uint_as_float(top) : (acc[0] + acc[1]) + (acc[2] + acc[3]));
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// The norm from the call's partials, in every thread.
template <int P>
__device__ __forceinline__ double join_partials(const double* __restrict__ part, int parts) {
  double p[BLOCKS / THREADS], a = 0.;
#pragma unroll
  for (int k = 0; k < BLOCKS / THREADS; ++k) p[k] = (int)threadIdx.x + k * THREADS < parts ? part[threadIdx.x + k * THREADS] : 0.;
#pragma unroll
  for (int k = 0; k < BLOCKS / THREADS; ++k) a = P == 0 ? (p[k] > a || p[k] != p[k] ? p[k] : a) : a + p[k];
  a = block_join<P>(a);
  return P == 2 ? sqrt(a) : a;
}

template <int P>
__global__ __launch_bounds__(THREADS) void grad_norm_final_kernel(const double* __restrict__ part, int parts, float* __restrict__ norm) {
  const double a = join_partials<P>(part, parts);
  if (threadIdx.x == 0) *norm = (float)a;
}

// q = p * f * 2^e over n values, the last ones first.
template <typename T>
__device__ __forceinline__ void scale_span(const T* p, T* q, int64_t n, float f, int e2) {
  constexpr int N = MbvaeVec<T>::N, STEP = THREADS * N;
  typedef typename MbvaeVec<T>::Aligned V;
  typedef typename MbvaeVec<T>::Any A;
  const auto put = [&](T* to, const V& v, int left) {
    float w[N];
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = __builtin_amdgcn_ldexpf((float)v[e] * f, e2);
    mbvae_store_vec<T>(to, left, w);
  };
  int64_t at = n / (U * STEP) * (U * STEP);                          // what lies behind the last whole group comes first
  V next[U];
  const int mine = threadIdx.x * N, rest = (int)(n - at) - mine;
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = mbvae_load_raw<T>(p + at + mine + u * STEP, rest - u * STEP);
  int64_t was = at;
  bool whole = false;
  while (true) {
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = next[u];
    at -= U * STEP;
    if (at >= 0)                                                     // (asked for before the stores: a load behind a store waits for it)
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = *reinterpret_cast<const A*>(p + at + mine + u * STEP);
#pragma unroll
    for (int u = 0; u < U; ++u) put(q + was + mine + u * STEP, v[u], whole ? N : rest - u * STEP);
    if (at < 0) break;
    was = at;
    whole = true;
  }
}

template <int P, typename Table>
__global__ __launch_bounds__(THREADS) void grad_scale_kernel(Table t, uint32_t chunks, const double* __restrict__ part, int parts, double max_norm,
                                                             int in_place, float* __restrict__ norm) {
  const double a = join_partials<P>(part, parts);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)a;
  const double c = max_norm / (a + 1e-6);
  float f = c > 1. || max_norm == INFINITY ? 1.f : (float)c;              // (a NaN norm makes every gradient NaN)
  int e = 0;
  if (c > 0. && c < 1.17549435e-38) f = (float)frexp(c, &e);              // a factor below fp32's normal range would lose its bits
  if (in_place && f == 1.f) return;                        // nothing to scale: the values stay as they are
  walk<true>(t, share_begin(chunks, blockIdx.x, gridDim.x), share_begin(chunks, blockIdx.x + 1, gridDim.x), [&](int i, int64_t at, int64_t n) {
    const int dtype = t.last(i) >> 24;
    if (dtype == MBVAE_F32) scale_span(reinterpret_cast<const float*>(t.src(i)) + at, reinterpret_cast<float*>(t.dst(i)) + at, n, f, e);
    else if (dtype == MBVAE_BF16) scale_span(reinterpret_cast<const mbvae_bf16*>(t.src(i)) + at, reinterpret_cast<mbvae_bf16*>(t.dst(i)) + at, n, f, e);
    else scale_span(reinterpret_cast<const mbvae_f16*>(t.src(i)) + at, reinterpret_cast<mbvae_f16*>(t.dst(i)) + at, n, f, e);
  });
}

struct Span { uintptr_t at, end; int64_t tensor; bool out; };

// True if some output shares memory with another output, or with an input other than its own exact place.
bool outputs_collide(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int64_t count, bool& failed) {
  Span* s = new (std::nothrow) Span[2 * count];
  failed = s == nullptr;
  if (failed) return false;
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t bytes = (uintptr_t)numel[i] * mbvae_dtype_size(dtype[i]);
    const uintptr_t a = (uintptr_t)src[i], b = (uintptr_t)dst[i];
    if (a != b) s[n++] = {a, a + bytes, i, false};
    s[n++] = {b, b + bytes, i, true};
  }
  std::sort(s, s + n, [](const Span& x, const Span& y) { return x.at < y.at; });
  uintptr_t any = 0, out = 0;               // ends of what has been passed: of everything, of the outputs
  bool hit = false;
  for (int64_t i = 0; i < n && !hit; ++i) {
    hit = s[i].out ? s[i].at < any : s[i].at < out;
    any = std::max(any, s[i].end);
    if (s[i].out) out = std::max(out, s[i].end);
  }
  delete[] s;
  return hit;
}

int pick_p(double p) { return p == 2. ? 2 : p == 1. ? 1 : p == std::numeric_limits<double>::infinity() ? 0 : -1; }

// Calls launch(table, entries before it, chunks before it) for each run of at most TENSORS non-empty tensors.
template <typename F>
int for_tables(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int64_t count, F launch) {
  InlineTable t;
  t.count = 0;
  t.first_[0] = 0;
  int entries = 0;
  uint32_t chunks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    if (t.count && (i == count || t.count == TENSORS)) {
      const int st = launch(t, entries, chunks);
      if (st != MBVAE_OK) return st;
      entries += t.count;
      chunks += t.first_[t.count];
      t.count = 0;
    }
    if (i == count || numel[i] == 0) continue;
    const int64_t c = (numel[i] + CHUNK - 1) / CHUNK;
    t.src_[t.count] = src[i];
    t.dst_[t.count] = dst ? dst[i] : nullptr;
    t.last_[t.count] = (uint32_t)(numel[i] - (c - 1) * CHUNK) | (uint32_t)dtype[i] << 24;
    t.first_[t.count + 1] = t.first_[t.count] + (uint32_t)c;
    ++t.count;
  }
  return MBVAE_OK;
}

struct Call {
  bool write, in_place;
  double max_norm;
  float* norm;
  double* part;
  hipStream_t stream;
};
template <int P, typename Table>
int run(const Table& t, uint32_t chunks, const Call& c) {
  const int blocks = (int)std::min<uint32_t>(chunks, BLOCKS);
  hipLaunchKernelGGL((grad_norm_kernel<P, Table>), dim3(blocks), dim3(THREADS), 0, c.stream, t, chunks, c.part);
  if (c.write)
    hipLaunchKernelGGL((grad_scale_kernel<P, Table>), dim3(blocks), dim3(THREADS), 0, c.stream, t, chunks, c.part, blocks, c.max_norm, c.in_place ? 1 : 0,
                       c.norm);
  else
    hipLaunchKernelGGL((grad_norm_final_kernel<P>), dim3(1), dim3(THREADS), 0, c.stream, c.part, blocks, c.norm);
  return mbvae_launch_status();
}
template <typename Table>
int run(int p, const Table& t, uint32_t chunks, const Call& c) {
  return p == 2 ? run<2>(t, chunks, c) : p == 1 ? run<1>(t, chunks, c) : run<0>(t, chunks, c);
}

}  // namespace

extern "C" {

// The partials and, where it does not fit the kernel arguments, the tensor table.
int64_t mbvae_grad_clip_workspace(int64_t count) { return (int64_t)sizeof(double) * BLOCKS + (count > TENSORS ? 24 * count + 8 : 0); }

// src, dst, numel, dtype: HOST arrays of `count` device pointers, value counts and types, read before the call returns.
// dst == NULL: the norm alone (max_norm is not looked at); dst[i] == src[i] for all i scales in place.
int mbvae_grad_clip(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int64_t count, double p,
                    double max_norm, float* norm, void* ws, int64_t ws_bytes, hipStream_t stream) {
  (void)hipGetLastError();  // drop stale (non-sticky) errors left by other runtime users
  if (count < 0 || !norm || !ws || (count && (!src || !numel || !dtype)) || ((uintptr_t)ws & 7)) return MBVAE_EINVAL;
  if (ws_bytes < mbvae_grad_clip_workspace(count)) return MBVAE_EINVAL;
  const int pick = pick_p(p);
  if (pick < 0) return MBVAE_EUNSUPPORTED;
  if (dst && !(max_norm >= 0.)) return MBVAE_EINVAL;
  Call c = {dst != nullptr, dst != nullptr, max_norm, norm, reinterpret_cast<double*>(ws), stream};
  int64_t chunks = 0, entries = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int size = mbvae_dtype_size(dtype[i]);
    if (size == 0 || numel[i] < 0 || numel[i] > ((int64_t)1 << 40)) return MBVAE_EINVAL;
    if (numel[i] && (!src[i] || (uintptr_t)src[i] % size || (dst && (!dst[i] || (uintptr_t)dst[i] % size)))) return MBVAE_EINVAL;
    if (dst && numel[i] && dst[i] != src[i]) c.in_place = false;
    chunks += (numel[i] + CHUNK - 1) / CHUNK;
    entries += numel[i] != 0;
  }
  if (chunks >= (int64_t)1 << 32 || entries > 0x7fffffff) return MBVAE_EUNSUPPORTED;
  if (dst) {
    bool failed = false;
    if (outputs_collide(src, dst, numel, dtype, count, failed) || failed) return MBVAE_EINVAL;
  }
  if (entries == 0) {                                               // nothing at all: a norm of zero
    hipLaunchKernelGGL((grad_norm_final_kernel<1>), dim3(1), dim3(THREADS), 0, stream, c.part, 0, norm);
    return mbvae_launch_status();
  }
  if (entries <= TENSORS)
    return for_tables(src, dst, numel, dtype, count, [&](const InlineTable& t, int, uint32_t) { return run(pick, t, (uint32_t)chunks, c); });
  MemoryTable m;
  char* w = reinterpret_cast<char*>(c.part + BLOCKS);
  m.src_ = reinterpret_cast<const void**>(w);
  m.dst_ = reinterpret_cast<void**>(w + 8 * entries);
  m.first_ = reinterpret_cast<uint32_t*>(w + 16 * entries);
  m.last_ = m.first_ + entries + 1;
  m.count = (int)entries;
  const int st = for_tables(src, dst, numel, dtype, count, [&](const InlineTable& t, int at, uint32_t chunk) {
    hipLaunchKernelGGL(grad_table_kernel, dim3(1), dim3(THREADS), 0, stream, t, m, at, chunk);
    return mbvae_launch_status();
  });
  return st != MBVAE_OK ? st : run(pick, m, (uint32_t)chunks, c);
}

}  // extern "C"
