// Gated residual update between two norms, forward and backward.
//   v = N_post(u),   y = x + a * w * v,   n = N_pre(y),        w = sigmoid(z) * (keep ? keep_scale : 0)
// u is the block's output (or x itself), N_post the norm behind the block, z its gate, a the residual scale (one value a column), keep a
// dropout mask, N_pre the norm in front of the next block; every part but x may be absent.  N is LayerNorm, (t - mean) / sqrt(var + eps)
// * gamma + beta, or the root-mean-square norm t / sqrt(mean t^2 + eps) * gamma (+ beta).
// Backward, with G the gradient of n through N_pre:
//   t = dy + G,  dx = t,  dv = t * a * w,  da = sum_rows t * w * v,  dz = t * a * v * w',  du = dv through N_post,
//   dgamma = sum_rows d * hat,  dbeta = sum_rows d     for both norms.
// All of it is bound by memory: one team of lanes holds a whole row in registers, so each operand is read once and each output
// written once, the row sums of the norms stay inside the team, and y is formed again in the backward from x, u and z (which it
// reads anyway) instead of being read.  The column sums are kept in registers over all rows of a team, joined per block, and the blocks'
// partials are added by a second kernel in a fixed order: reproducible, no atomics.
// All sums, statistics and intermediate values are fp32; outputs are rounded once.
#include "typed.h"
#include <algorithm>

namespace {

struct Norm {
  const void* gamma;      // null: this norm is absent
  const void* beta;       // null: no shift
};
struct Args {
  const void *x, *u, *z;
  const uint8_t* keep;
  const void* scale;
  Norm post, pre;
  int64_t ldx, ldu, ldz, rows;
  int D, ptype, rms;
  float keep_scale, eps;
  float4* stats;          // per row: mean and reciprocal deviation of u, then of y
};
struct FwdArgs : Args {
  void *y, *n;
};
struct BwdArgs : Args {
  const void *dy, *dn;
  int64_t lddy, lddn;
  void *dx, *du, *dz;
  float* part;            // [blocks][SUMS][D]
};
// The column sums, in the order in which the partials are laid out.
enum { SUM_SCALE, SUM_POST_G, SUM_POST_B, SUM_PRE_G, SUM_PRE_B, SUMS };

template <int TPR>
constexpr int block_threads() { return TPR > 256 ? TPR : 256; }

// Sum of two values over a row's team.  Teams wider than a wave meet in LDS; the buffers alternate so that one barrier a sum is enough.
template <int TPR>
struct Team {
  float2* red;            // [2][waves of the block]
  int turn;
  __device__ __forceinline__ float2 sum(float a, float b) {
    if constexpr (TPR <= 64) {
      return make_float2(mbvae_team_sum<TPR>(a), mbvae_team_sum<TPR>(b));
    } else {
      constexpr int WAVES = block_threads<TPR>() / 64, MINE = TPR / 64;
      a = mbvae_team_sum<64>(a);
      b = mbvae_team_sum<64>(b);
      float2* r = red + turn * WAVES;
      turn ^= 1;
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) r[wave] = make_float2(a, b);
      __syncthreads();
      const int first = wave / MINE * MINE;
      float2 s = r[first];
#pragma unroll
      for (int w = 1; w < MINE; ++w) { s.x += r[first + w].x; s.y += r[first + w].y; }
      return s;
    }
  }
};

// sigmoid(z) and its derivative, both accurate at either end.
__device__ __forceinline__ void sigmoid(float z, float& s, float& ds) {
  const float t = expf(-fabsf(z)), r = 1.f / (1.f + t);
  s = z < 0.f ? t * r : r;
  ds = t * r * r;
}

// A row's elements of one lane: EPL of them, in 16-byte pieces TPR pieces apart.
template <typename T, int TPR, int EPL>
struct Row {
  static constexpr int N = MbvaeVec<T>::N, NV = EPL / N;
  static_assert(NV * N == EPL, "whole pieces");
  static __device__ __forceinline__ int col(int lane, int v) { return (v * TPR + lane) * N; }
  static __device__ __forceinline__ void load(const void* p, int64_t at, int D, int lane, float* out) {
#pragma unroll
    for (int v = 0; v < NV; ++v) mbvae_load_vec<T>(reinterpret_cast<const T*>(p) + at + col(lane, v), D - col(lane, v), out + v * N);
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, int D, int lane, const float* val) {
#pragma unroll
    for (int v = 0; v < NV; ++v) mbvae_store_vec<T>(reinterpret_cast<T*>(p) + at + col(lane, v), D - col(lane, v), val + v * N);
  }
  // one value per column, in the parameters' type; `none` where p is null and behind the row's end
  static __device__ __forceinline__ void param(const void* p, int type, int D, int lane, float none, float* out) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int c = col(lane, v) + e;
        out[v * N + e] = p && c < D ? mbvae_load_param(p, type, c) : none;
      }
  }
  static __device__ __forceinline__ void keep(const uint8_t* p, int64_t at, int D, int lane, bool* out) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int c = col(lane, v) + e;
        out[v * N + e] = c < D ? p[at + c] != 0 : false;
      }
  }
  static __device__ __forceinline__ bool inside(int D, int lane, int e) { return col(lane, e / N) + e % N < D; }
};

// Mean and reciprocal deviation of a row (two-pass: the deviations are summed from the mean).
template <typename R, int EPL, typename TeamT>
__device__ __forceinline__ void row_stats(TeamT& team, const float* t, int D, int lane, bool rms, float eps, float& mean, float& r) {
  mean = 0.f;
  if (!rms) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) s += t[e];
    mean = team.sum(s, 0.f).x / D;
  }
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    const float d = R::inside(D, lane, e) ? t[e] - mean : 0.f;
    q += d * d;
  }
  r = 1.f / sqrtf(team.sum(q, 0.f).x / D + eps);
}

template <typename T, int TPR, int EPL>
__global__ __launch_bounds__(block_threads<TPR>()) void gated_norm_fwd_kernel(FwdArgs a) {
  typedef Row<T, TPR, EPL> R;
  constexpr int TEAMS = block_threads<TPR>() / TPR;
  __shared__ float2 red[2 * (block_threads<TPR>() / 64)];
  Team<TPR> team{red, 0};
  const int lane = threadIdx.x % TPR, D = a.D;
  float pg[EPL], pb[EPL], ng[EPL], nb[EPL], sc[EPL];
  R::param(a.post.gamma, a.ptype, D, lane, 0.f, pg);
  R::param(a.post.beta, a.ptype, D, lane, 0.f, pb);
  R::param(a.pre.gamma, a.ptype, D, lane, 0.f, ng);
  R::param(a.pre.beta, a.ptype, D, lane, 0.f, nb);
  R::param(a.scale, a.ptype, D, lane, 1.f, sc);
  for (int64_t base = (int64_t)blockIdx.x * TEAMS; base < a.rows; base += (int64_t)gridDim.x * TEAMS) {
    const bool active = base + threadIdx.x / TPR < a.rows;          // (idle teams repeat the last row and store nothing)
    const int64_t row = active ? base + threadIdx.x / TPR : a.rows - 1;
    float y[EPL], v[EPL];
    R::load(a.x, row * a.ldx, D, lane, y);
    if (a.u) R::load(a.u, row * a.ldu, D, lane, v);
    else
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = y[e];
    float w[EPL];
    if (a.z) {
      R::load(a.z, row * a.ldz, D, lane, w);
#pragma unroll
      for (int e = 0; e < EPL; ++e) { float ds; sigmoid(w[e], w[e], ds); }
    } else
#pragma unroll
      for (int e = 0; e < EPL; ++e) w[e] = 1.f;
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.post.gamma) {
      row_stats<R, EPL>(team, v, D, lane, a.rms, a.eps, st.x, st.y);
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = (v[e] - st.x) * st.y * pg[e] + pb[e];
    }
    bool kept[EPL];
    if (a.keep) R::keep(a.keep, row * D, D, lane, kept);
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      float t = v[e] * (a.keep ? w[e] * a.keep_scale : w[e]) * sc[e];
      if (a.keep && !kept[e]) t = 0.f;                              // a dropped value adds nothing, whatever it is
      y[e] += t;
    }
    if (active) R::store(a.y, row * D, D, lane, y);
    if (a.pre.gamma) {
      row_stats<R, EPL>(team, y, D, lane, a.rms, a.eps, st.z, st.w);
#pragma unroll
      for (int e = 0; e < EPL; ++e) y[e] = (y[e] - st.z) * st.w * ng[e] + nb[e];
      if (active) R::store(a.n, row * D, D, lane, y);
    }
    if (a.stats && active && lane == 0) a.stats[row] = st;
  }
}

template <typename T, int TPR, int EPL>
__global__ __launch_bounds__(block_threads<TPR>()) void gated_norm_bwd_kernel(BwdArgs a) {
  typedef Row<T, TPR, EPL> R;
  constexpr int THREADS = block_threads<TPR>(), TEAMS = THREADS / TPR;
  __shared__ float2 red[2 * (THREADS / 64)];
  __shared__ float join[THREADS * EPL];
  Team<TPR> team{red, 0};
  const int lane = threadIdx.x % TPR, D = a.D;
  const bool post = a.post.gamma != nullptr, pre = a.pre.gamma != nullptr && a.dn != nullptr;
  float pg[EPL], pb[EPL], ng[EPL], sc[EPL];
  R::param(a.post.gamma, a.ptype, D, lane, 0.f, pg);
  R::param(a.post.beta, a.ptype, D, lane, 0.f, pb);
  R::param(a.pre.gamma, a.ptype, D, lane, 0.f, ng);
  R::param(a.scale, a.ptype, D, lane, 1.f, sc);
  float sums[SUMS][EPL];
#pragma unroll
  for (int s = 0; s < SUMS; ++s)
#pragma unroll
    for (int e = 0; e < EPL; ++e) sums[s][e] = 0.f;
  for (int64_t base = (int64_t)blockIdx.x * TEAMS; base < a.rows; base += (int64_t)gridDim.x * TEAMS) {
    const bool active = base + threadIdx.x / TPR < a.rows;
    const int64_t row = active ? base + threadIdx.x / TPR : a.rows - 1;
    const float4 st = a.stats ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    float x[EPL], v[EPL], w[EPL], dw[EPL], t[EPL], d[EPL];
    R::load(a.x, row * a.ldx, D, lane, x);
    if (a.u) R::load(a.u, row * a.ldu, D, lane, v);
    else
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = x[e];
    if (a.z) R::load(a.z, row * a.ldz, D, lane, w);
    if (a.dy) R::load(a.dy, row * a.lddy, D, lane, t);
    else
#pragma unroll
      for (int e = 0; e < EPL; ++e) t[e] = 0.f;
    if (pre) R::load(a.dn, row * a.lddn, D, lane, d);
    bool kept[EPL];
    if (a.keep) R::keep(a.keep, row * D, D, lane, kept);
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      if (a.z) sigmoid(w[e], w[e], dw[e]);
      else { w[e] = 1.f; dw[e] = 0.f; }
      if (a.keep) {
        w[e] = kept[e] ? w[e] * a.keep_scale : 0.f;
        dw[e] = kept[e] ? dw[e] * a.keep_scale : 0.f;
      }
      if (post) v[e] = (v[e] - st.x) * st.y;                       // normalised
    }
    if (pre) {
      float g[EPL], hat[EPL], s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const bool in = R::inside(D, lane, e);
        const float vv = post ? v[e] * pg[e] + pb[e] : v[e];
        const float y = x[e] + (!a.keep || kept[e] ? vv * w[e] * sc[e] : 0.f);
        hat[e] = in ? (y - st.z) * st.w : 0.f;
        g[e] = d[e] * ng[e];
        s1 += g[e];
        s2 += g[e] * hat[e];
        if (active) { sums[SUM_PRE_G][e] += d[e] * hat[e]; sums[SUM_PRE_B][e] += d[e]; }
      }
      const float2 m = team.sum(s1, s2);
      const float m1 = a.rms ? 0.f : m.x / D, m2 = m.y / D;
#pragma unroll
      for (int e = 0; e < EPL; ++e) t[e] += st.w * (g[e] - m1 - hat[e] * m2);
    }
    // t is the whole gradient of y
    float dv[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const float vv = post ? v[e] * pg[e] + pb[e] : v[e];
      const bool on = !a.keep || kept[e];
      dv[e] = on ? t[e] * sc[e] * w[e] : 0.f;
      dw[e] = on ? t[e] * sc[e] * vv * dw[e] : 0.f;
      if (active) {
        sums[SUM_SCALE][e] += on ? t[e] * w[e] * vv : 0.f;
        if (post) { sums[SUM_POST_G][e] += dv[e] * v[e]; sums[SUM_POST_B][e] += dv[e]; }
      }
    }
    if (a.dz && active) R::store(a.dz, row * D, D, lane, dw);
    if (post) {
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const bool in = R::inside(D, lane, e);
        if (!in) v[e] = 0.f;
        dv[e] = dv[e] * pg[e];
        s1 += dv[e];
        s2 += dv[e] * v[e];
      }
      const float2 m = team.sum(s1, s2);
      const float m1 = a.rms ? 0.f : m.x / D, m2 = m.y / D;
#pragma unroll
      for (int e = 0; e < EPL; ++e) dv[e] = st.y * (dv[e] - m1 - v[e] * m2);
    }
    if (a.u) {
      if (a.du && active) R::store(a.du, row * D, D, lane, dv);
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) t[e] += dv[e];
    }
    if (a.dx && active) R::store(a.dx, row * D, D, lane, t);
  }
  // column sums of the block: its teams in order
#pragma unroll
  for (int s = 0; s < SUMS; ++s) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EPL; ++e) join[e * THREADS + threadIdx.x] = sums[s][e];
    __syncthreads();
    if (threadIdx.x < TPR) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const int c = R::col(lane, e / R::N) + e % R::N;
        float total = 0.f;
        for (int k = 0; k < TEAMS; ++k) total += join[e * THREADS + k * TPR + threadIdx.x];
        if (c < D) a.part[((int64_t)blockIdx.x * SUMS + s) * D + c] = total;
      }
    }
  }
}

// out[s][c] = sum over the blocks of part[block][s][c], in the parameters' type.  32 columns x 8 groups of blocks.
struct Outs { void* p[SUMS]; };
__global__ __launch_bounds__(256) void gated_norm_sums_kernel(const float* __restrict__ part, Outs outs, int blocks, int D, int ptype) {
  __shared__ float red[8][33];
  const int cx = threadIdx.x & 31, g = threadIdx.x >> 5, s = blockIdx.y;
  const int c = blockIdx.x * 32 + cx;
  if (!outs.p[s]) return;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < D) {
    const float* p = part + (int64_t)s * D + c;
    const int64_t step = (int64_t)SUMS * D;
    int b = g;
    for (; b + 24 < blocks; b += 32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) a[q] += p[(b + 8 * q) * step];
    }
    for (; b < blocks; b += 8) a[0] += p[b * step];
  }
  red[g][cx] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (g == 0 && c < D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[k][cx];
    mbvae_store_param(outs.p[s], ptype, c, t);
  }
}

constexpr int MAX_D = 8192;
constexpr int64_t MAX_BLOCKS_BWD = 1024;

// Lanes a row and elements a lane: as few idle lanes as the width allows up to one wave of two pieces, then 16 elements a lane.
// f(lanes, elements) with both as constants.
template <typename T, typename F>
void for_width(int D, F f) {
  constexpr int N = MbvaeVec<T>::N;
#define GN_CASE(lanes, elements) f(std::integral_constant<int, lanes>(), std::integral_constant<int, elements>())
  if (D <= 16 * N) GN_CASE(16, N);
  else if (D <= 32 * N) GN_CASE(32, N);
  else if (D <= 64 * N) GN_CASE(64, N);
  else if (D <= 512) GN_CASE(64, 8);
  else if (D <= 1024) GN_CASE(64, 16);
  else if (D <= 2048) GN_CASE(128, 16);
  else if (D <= 4096) GN_CASE(256, 16);
  else GN_CASE(512, 16);
#undef GN_CASE
}

int64_t teams_for(int dtype, int64_t D) {
  const int N = dtype == MBVAE_F32 ? 4 : 8;
  const int lanes = D <= 16 * N ? 16 : D <= 32 * N ? 32 : D <= 1024 ? 64 : D <= 2048 ? 128 : D <= 4096 ? 256 : 512;
  return std::max(256, lanes) / lanes;
}
int64_t bwd_blocks(int dtype, int64_t rows, int64_t D) {
  const int64_t teams = teams_for(dtype, D);
  return std::max<int64_t>(1, std::min<int64_t>((rows + teams - 1) / teams, MAX_BLOCKS_BWD));
}

int check(const Args& a, int dtype, int64_t rows, int64_t D, int ptype) {
  if (rows < 0 || D <= 0 || mbvae_dtype_size(dtype) == 0 || mbvae_dtype_size(ptype) == 0) return MBVAE_EINVAL;
  if (a.ldx < 0 || a.ldu < 0 || a.ldz < 0) return MBVAE_EINVAL;
  if (rows && !a.x) return MBVAE_EINVAL;
  if ((a.post.beta && !a.post.gamma) || (a.pre.beta && !a.pre.gamma)) return MBVAE_EINVAL;
  if (((uintptr_t)a.stats & 15) || !(a.eps >= 0.f)) return MBVAE_EINVAL;
  if (D > MAX_D || rows >= (int64_t)1 << 31) return MBVAE_EUNSUPPORTED;
  return MBVAE_OK;
}

template <typename T>
void launch_fwd(const FwdArgs& a, hipStream_t stream) {
  for_width<T>(a.D, [&](auto lanes, auto elements) {
    constexpr int TPR = decltype(lanes)::value, EPL = decltype(elements)::value, TEAMS = block_threads<TPR>() / TPR;
    const int64_t blocks = std::min<int64_t>((a.rows + TEAMS - 1) / TEAMS, 4096);
    hipLaunchKernelGGL((gated_norm_fwd_kernel<T, TPR, EPL>), dim3((unsigned)blocks), dim3(block_threads<TPR>()), 0, stream, a);
  });
}
template <typename T>
void launch_bwd(const BwdArgs& a, int64_t blocks, hipStream_t stream) {
  for_width<T>(a.D, [&](auto lanes, auto elements) {
    constexpr int TPR = decltype(lanes)::value, EPL = decltype(elements)::value;
    hipLaunchKernelGGL((gated_norm_bwd_kernel<T, TPR, EPL>), dim3((unsigned)blocks), dim3(block_threads<TPR>()), 0, stream, a);
  });
}

}  // namespace

extern "C" {

int mbvae_gated_norm_fwd(const void* x, int64_t ldx, const void* u, int64_t ldu, const void* z, int64_t ldz, const uint8_t* keep, float keep_scale,
                         const void* post_gamma, const void* post_beta, const void* scale, const void* pre_gamma, const void* pre_beta, void* y, void* n,
                         float* stats, int64_t rows, int64_t D, int rms, float eps, int dtype, int ptype, hipStream_t stream) {
  (void)hipGetLastError();  // drop stale (non-sticky) errors left by other runtime users
  FwdArgs a;
  a.x = x; a.u = u; a.z = z; a.keep = keep; a.scale = scale;
  a.post = {post_gamma, post_beta}; a.pre = {pre_gamma, pre_beta};
  a.ldx = ldx; a.ldu = ldu; a.ldz = ldz; a.rows = rows; a.D = (int)std::min<int64_t>(D, MAX_D); a.ptype = ptype; a.rms = rms;
  a.keep_scale = keep_scale; a.eps = eps; a.stats = reinterpret_cast<float4*>(stats);
  a.y = y; a.n = n;
  const int st = check(a, dtype, rows, D, ptype);
  if (st != MBVAE_OK) return st;
  if (rows == 0) return MBVAE_OK;
  if (!y || (pre_gamma && !n)) return MBVAE_EINVAL;
  if (dtype == MBVAE_F32) launch_fwd<float>(a, stream);
  else if (dtype == MBVAE_BF16) launch_fwd<mbvae_bf16>(a, stream);
  else launch_fwd<mbvae_f16>(a, stream);
  return mbvae_launch_status();
}

int64_t mbvae_gated_norm_bwd_workspace(int64_t rows, int64_t D, int dtype) {
  if (rows < 0 || D <= 0 || D > MAX_D || mbvae_dtype_size(dtype) == 0) return 0;
  return (int64_t)sizeof(float) * bwd_blocks(dtype, rows, D) * SUMS * D;
}

int mbvae_gated_norm_bwd(const void* x, int64_t ldx, const void* u, int64_t ldu, const void* z, int64_t ldz, const uint8_t* keep, float keep_scale,
                         const void* post_gamma, const void* post_beta, const void* scale, const void* pre_gamma, const float* stats, const void* dy,
                         int64_t lddy, const void* dn, int64_t lddn, void* dx, void* du, void* dz, void* dscale, void* dpost_gamma, void* dpost_beta,
                         void* dpre_gamma, void* dpre_beta, int64_t rows, int64_t D, int rms, float eps, int dtype, int ptype, void* ws, int64_t ws_bytes,
                         hipStream_t stream) {
  (void)hipGetLastError();  // drop stale (non-sticky) errors left by other runtime users
  BwdArgs a;
  a.x = x; a.u = u; a.z = z; a.keep = keep; a.scale = scale;
  a.post = {post_gamma, post_beta}; a.pre = {pre_gamma, nullptr};
  a.ldx = ldx; a.ldu = ldu; a.ldz = ldz; a.rows = rows; a.D = (int)std::min<int64_t>(D, MAX_D); a.ptype = ptype; a.rms = rms;
  a.keep_scale = keep_scale; a.eps = eps; a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  a.dy = dy; a.dn = dn; a.lddy = lddy; a.lddn = lddn; a.dx = dx; a.du = du; a.dz = dz; a.part = reinterpret_cast<float*>(ws);
  const int st = check(a, dtype, rows, D, ptype);
  if (st != MBVAE_OK) return st;
  if (lddy < 0 || lddn < 0 || (dn && !pre_gamma) || (rows && !stats) || !ws || ((uintptr_t)ws & 15)) return MBVAE_EINVAL;
  if ((dpost_gamma || dpost_beta) && !post_gamma) return MBVAE_EINVAL;
  if ((dpre_gamma || dpre_beta) && !pre_gamma) return MBVAE_EINVAL;
  if ((du && !u) || (dz && !z)) return MBVAE_EINVAL;
  if (ws_bytes < mbvae_gated_norm_bwd_workspace(rows, D, dtype)) return MBVAE_EINVAL;
  const int64_t blocks = bwd_blocks(dtype, rows, D);
  if (dtype == MBVAE_F32) launch_bwd<float>(a, blocks, stream);
  else if (dtype == MBVAE_BF16) launch_bwd<mbvae_bf16>(a, blocks, stream);
  else launch_bwd<mbvae_f16>(a, blocks, stream);
  const Outs outs = {{dscale, dpost_gamma, dpost_beta, dpre_gamma, dpre_beta}};
  if (dscale || dpost_gamma || dpost_beta || dpre_gamma || dpre_beta)
    hipLaunchKernelGGL(gated_norm_sums_kernel, dim3((unsigned)((D + 31) / 32), SUMS), dim3(256), 0, stream, a.part, outs, (int)blocks, (int)D, ptype);
  return mbvae_launch_status();
}

}  // extern "C"
