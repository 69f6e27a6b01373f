// Global norm of a list of gradient tensors and their scaling to a largest norm.
//   norm = (sum |g|^p)^(1/p) over every value of every tensor (p = 1, 2 or infinity), out = g * min(1, max_norm / (norm + 1e-6)).
// The work is one streaming read for the norm and one read + write for the scaling; nothing is computed per tensor.
// The tensor table travels in the kernel arguments (at most TENSORS entries a launch), so a call can be captured into a graph and
// needs no staging buffer.  Tensors are cut into chunks of CHUNK values that a fixed grid walks over; every block leaves ONE partial
// sum in the workspace, in fp64 (no overflow of a square, no rounding to speak of), and each scaling block adds the partials
// up itself in the same order: reproducible, no atomics, no separate launch for the join.
#include "typed.h"
#include <algorithm>
#include <cmath>
#include <limits>
#include <new>

namespace {

constexpr int TENSORS = 160;          // 24 bytes each: the argument block stays below 4 KB
constexpr int CHUNK = 8192;           // values
constexpr int THREADS = 256;
constexpr int BLOCKS = 1024;          // partial sums of one call (shared out over its launches)

struct TensorTable {
  const void* src[TENSORS];
  void* dst[TENSORS];
  uint32_t first[TENSORS + 1];        // first chunk of tensor i; first[count] = chunks of the launch
  uint32_t last[TENSORS];             // values of the tensor's last chunk, plus its type in the upper bits
  int count;
};
static_assert(sizeof(TensorTable) <= 3968, "kernel arguments");

// Tensor that chunk c belongs to (the table is wave-uniform: scalar loads and branches).
__device__ __forceinline__ int tensor_of(const TensorTable& t, uint32_t c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// One value joined to the running partial: P = 1 and 2 sums, P = 0 the largest magnitude (NaN counts as larger than infinity).
template <int P>
__device__ __forceinline__ void take(double& acc, uint32_t& top, float v) {
  if (P == 0) top = max(top, __float_as_uint(v) & 0x7fffffffu);
  else if (P == 1) acc += (double)fabsf(v);
  else acc = fma((double)v, (double)v, acc);
}

template <int P, typename T>
__device__ __forceinline__ void norm_chunk(const T* p, int n, double* acc, uint32_t& top) {
  constexpr int N = MbvaeVec<T>::N;
  float v[N];
#pragma unroll 4
  for (int i = threadIdx.x * N; i < n; i += THREADS * N) {
    mbvae_load_vec<T>(p + i, n - i, v);
#pragma unroll
    for (int e = 0; e < N; ++e) take<P>(acc[e & 3], top, v[e]);
  }
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

template <int P>
__global__ __launch_bounds__(THREADS) void grad_norm_kernel(TensorTable t, double* __restrict__ part) {
  double acc[4] = {0., 0., 0., 0.};
  uint32_t top = 0;
  for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int i = tensor_of(t, c);
    const uint32_t k = c - t.first[i];
    const int n = c + 1 == t.first[i + 1] ? (int)(t.last[i] & 0xffffff) : CHUNK, dtype = t.last[i] >> 24;
    const int64_t at = (int64_t)k * CHUNK;
    if (dtype == MBVAE_F32) norm_chunk<P>(reinterpret_cast<const float*>(t.src[i]) + at, n, acc, top);
    else if (dtype == MBVAE_BF16) norm_chunk<P>(reinterpret_cast<const mbvae_bf16*>(t.src[i]) + at, n, acc, top);
    else norm_chunk<P>(reinterpret_cast<const mbvae_f16*>(t.src[i]) + at, n, acc, top);
  }
  const double a = block_join<P>(P == 0 ? (double)__uint_as_float(top) : (acc[0] + acc[1]) + (acc[2] + acc[3]));
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// The norm from the call's partials, in every thread.
template <int P>
__device__ __forceinline__ double join_partials(const double* __restrict__ part, int parts) {
  double a = 0.;
  for (int i = threadIdx.x; i < parts; i += THREADS) a = P == 0 ? (part[i] > a || part[i] != part[i] ? part[i] : a) : a + part[i];
  a = block_join<P>(a);
  return P == 2 ? sqrt(a) : a;
}

template <int P>
__global__ __launch_bounds__(THREADS) void grad_norm_final_kernel(const double* __restrict__ part, int parts, float* __restrict__ norm) {
  const double a = join_partials<P>(part, parts);
  if (threadIdx.x == 0) *norm = (float)a;
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* p, T* q, int n, float f) {
  constexpr int N = MbvaeVec<T>::N;
  float v[N];
#pragma unroll 4
  for (int i = threadIdx.x * N; i < n; i += THREADS * N) {
    mbvae_load_vec<T>(p + i, n - i, v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= f;
    mbvae_store_vec<T>(q + i, n - i, v);
  }
}

template <int P>
__global__ __launch_bounds__(THREADS) void grad_scale_kernel(TensorTable t, const double* __restrict__ part, int parts, double max_norm,
                                                             int in_place, float* __restrict__ norm) {
  const double a = join_partials<P>(part, parts);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)a;
  const double c = max_norm / (a + 1e-6);
  const float f = c > 1. ? 1.f : (float)c;                 // (a NaN norm makes every gradient NaN)
  if (in_place && f == 1.f) return;                        // nothing to scale: the values stay as they are
  for (uint32_t ch = blockIdx.x; ch < t.first[t.count]; ch += gridDim.x) {
    const int i = tensor_of(t, ch);
    const uint32_t k = ch - t.first[i];
    const int n = ch + 1 == t.first[i + 1] ? (int)(t.last[i] & 0xffffff) : CHUNK, dtype = t.last[i] >> 24;
    const int64_t at = (int64_t)k * CHUNK;
    if (dtype == MBVAE_F32) scale_chunk(reinterpret_cast<const float*>(t.src[i]) + at, reinterpret_cast<float*>(t.dst[i]) + at, n, f);
    else if (dtype == MBVAE_BF16)
      scale_chunk(reinterpret_cast<const mbvae_bf16*>(t.src[i]) + at, reinterpret_cast<mbvae_bf16*>(t.dst[i]) + at, n, f);
    else scale_chunk(reinterpret_cast<const mbvae_f16*>(t.src[i]) + at, reinterpret_cast<mbvae_f16*>(t.dst[i]) + at, n, f);
  }
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

// Calls launch(table, chunks, chunks before it) for each run of at most TENSORS non-empty tensors.
template <typename F>
int for_tables(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int64_t count, F launch) {
  TensorTable t;
  t.count = 0;
  t.first[0] = 0;
  int64_t before = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t chunks = i < count ? (numel[i] + CHUNK - 1) / CHUNK : 0;
    if (t.count && (i == count || t.count == TENSORS || t.first[t.count] + chunks > 0x7fffffff)) {
      const int st = launch(t, before);
      if (st != MBVAE_OK) return st;
      before += t.first[t.count];
      t.count = 0;
    }
    if (i == count || chunks == 0) continue;
    t.src[t.count] = src[i];
    t.dst[t.count] = dst ? dst[i] : nullptr;
    t.last[t.count] = (uint32_t)(numel[i] - (chunks - 1) * CHUNK) | (uint32_t)dtype[i] << 24;
    t.first[t.count + 1] = t.first[t.count] + (uint32_t)chunks;
    ++t.count;
  }
  return MBVAE_OK;
}

// Blocks of a launch over `chunks` chunks, `before` of the call's `total` already launched: its share of BLOCKS, and at least one.
int share(int64_t chunks, int64_t total) {
  return (int)std::max<int64_t>(1, total <= BLOCKS ? chunks : chunks * BLOCKS / total);
}

template <int P>
int norm_and_scale(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int64_t count, double max_norm,
                   bool in_place, float* norm, double* part, hipStream_t stream) {
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += (numel[i] + CHUNK - 1) / CHUNK;
  int parts = 0;
  int st = for_tables(src, nullptr, numel, dtype, count, [&](const TensorTable& t, int64_t) {
    const int blocks = share(t.first[t.count], total);
    hipLaunchKernelGGL((grad_norm_kernel<P>), dim3(blocks), dim3(THREADS), 0, stream, t, part + parts);
    parts += blocks;
    return mbvae_launch_status();
  });
  if (st != MBVAE_OK) return st;
  if (!dst || total == 0) {
    hipLaunchKernelGGL((grad_norm_final_kernel<P>), dim3(1), dim3(THREADS), 0, stream, part, parts, norm);
    return mbvae_launch_status();
  }
  return for_tables(src, dst, numel, dtype, count, [&](const TensorTable& t, int64_t before) {
    const int blocks = share(t.first[t.count], total);
    hipLaunchKernelGGL((grad_scale_kernel<P>), dim3(blocks), dim3(THREADS), 0, stream, t, part, parts, max_norm, in_place ? 1 : 0,
                       before == 0 ? norm : nullptr);
    return mbvae_launch_status();
  });
}

}  // namespace

extern "C" {

// Partials of one call over `count` tensors: BLOCKS shared out by chunks, and at least one block a launch.
int64_t mbvae_grad_clip_workspace(int64_t count) { return (int64_t)sizeof(double) * (BLOCKS + (count < 0 ? 0 : count) / TENSORS + 2); }

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
  bool in_place = dst != nullptr;
  for (int64_t i = 0; i < count; ++i) {
    const int size = mbvae_dtype_size(dtype[i]);
    if (size == 0 || numel[i] < 0 || numel[i] > ((int64_t)1 << 43)) return MBVAE_EINVAL;
    if (numel[i] && (!src[i] || (uintptr_t)src[i] % size || (dst && (!dst[i] || (uintptr_t)dst[i] % size)))) return MBVAE_EINVAL;
    if (dst && numel[i] && dst[i] != src[i]) in_place = false;
  }
  if (dst) {
    bool failed = false;
    if (outputs_collide(src, dst, numel, dtype, count, failed) || failed) return MBVAE_EINVAL;
  }
  double* part = reinterpret_cast<double*>(ws);
  if (pick == 2) return norm_and_scale<2>(src, dst, numel, dtype, count, max_norm, in_place, norm, part, stream);
  if (pick == 1) return norm_and_scale<1>(src, dst, numel, dtype, count, max_norm, in_place, norm, part, stream);
  return norm_and_scale<0>(src, dst, numel, dtype, count, max_norm, in_place, norm, part, stream);
}

}  // extern "C"
