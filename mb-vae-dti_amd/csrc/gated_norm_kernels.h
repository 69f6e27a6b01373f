// Kernels of the gated residual update (see gated_norm.hip for the mathematics) for one activation type.
#pragma once
#include "gated_norm.h"
#include <type_traits>

namespace {

// 1 / a to within a rounding: the hardware's reciprocal and one Newton step.
__device__ __forceinline__ float reciprocal(float a) {
  const float r = __builtin_amdgcn_rcpf(a);
  return fmaf(fmaf(-a, r, 1.f), r, r);
}

// ------------------------------------------------------------------------------------------------ sums over a row
// TPR lanes of a wave own a row (4 to 64), or, with TPR == 0, a whole block does: its waves meet in LDS, in buffers that alternate so
// that one barrier a sum is enough.
template <int TPR>
struct Team {
  float2* red;            // [2][16], used by whole blocks
  int turn;
  __device__ __forceinline__ float2 sum(float a, float b) {
    if constexpr (TPR > 0) {
      return make_float2(mbvae_team_sum<TPR>(a), mbvae_team_sum<TPR>(b));
    } else {
      a = mbvae_team_sum<64>(a);
      b = mbvae_team_sum<64>(b);
      float2* r = red + turn * 16;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = make_float2(a, b);
      __syncthreads();
      float2 s = r[0];
      for (unsigned w = 1; w < blockDim.x / 64; ++w) { s.x += r[w].x; s.y += r[w].y; }
      return s;
    }
  }
  __device__ __forceinline__ float sum(float a) {
    if constexpr (TPR > 0) return mbvae_team_sum<TPR>(a);
    else return sum(a, 0.f).x;
  }
  // Mean of the D values that the team's threads hold (t, where own) and the sum of their squared deviations from it, each summed from
  // the values themselves.  A block needs one barrier for both: its waves exchange the mean and the deviations of what each holds.
  template <int EPL, typename R>
  __device__ __forceinline__ void moments(const R& row, const float* t, float inv_D, float& mean, float& squares) {
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) s += row.counted(e, t[e]);
    const auto deviations = [&](float m) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float d = row.own(e) ? t[e] - m : 0.f;
        q = fmaf(d, d, q);
      }
    };
    if constexpr (TPR > 0) {
      mean = sum(s) * inv_D;
      deviations(mean);
      squares = sum(q);
    } else {
      const unsigned wave = threadIdx.x >> 6, waves = blockDim.x / 64;
      const float m = mbvae_team_sum<64>(s) * reciprocal(row.held(wave));
      deviations(m);
      q = mbvae_team_sum<64>(q);
      float2* r = red + turn * 16;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) r[wave] = make_float2(m, q);
      __syncthreads();
      float total = 0.f, within = 0.f, between = 0.f;
      for (unsigned w = 0; w < waves; ++w) total = fmaf(row.held(w), r[w].x, total);
      mean = total * inv_D;
      for (unsigned w = 0; w < waves; ++w) {
        const float d = r[w].x - mean;
        within += r[w].y;
        between = fmaf(row.held(w) * d, d, between);
      }
      squares = within + between;
    }
  }
};

// sigmoid(z) and its derivative, accurate at both ends: with t = exp(-|z|) they are 1 / (1 + t) or t / (1 + t), and t / (1 + t)^2.
// t = 2^-(h + l) where h + l is |z| log2(e) to 48 bits: the hardware's 2^h, corrected by l to first order.
__device__ __forceinline__ void sigmoid(float z, float& s, float& ds) {
  const float a = fabsf(z), h = a * 1.44269502f, l = fmaf(a, 1.44269502f, -h) + a * 1.92596299e-8f;
  const float t0 = __builtin_amdgcn_exp2f(-h), t = a < 128.f ? fmaf(t0 * -0.693147181f, l, t0) : t0;      // (from 128 on l may not be finite)
  const float r = reciprocal(1.f + t);
  s = z < 0.f ? t * r : r;
  ds = t * r * r;
}

// ------------------------------------------------------------------------------------------------ one thread's elements of a row
// EPL of them in 16-byte pieces; piece v of thread l is the row's (v * width + l)-th.  WHOLE: the row is a whole number of pieces.
// MOVED: it is not, and its last piece is moved back to end where the row ends: it repeats columns of the piece before, which both
// threads compute alike and store alike, and which `own` leaves out of the sums.  (Taking the last piece element by element instead made a
// row of 38 bf16 values 2.4 times as slow.)  SHORT: the row is shorter than one piece and goes element by element.
enum { WHOLE, MOVED, SHORT };
template <typename T, int TPR, int EPL, int KIND>
struct Row {
  static constexpr int N = MbvaeVec<T>::N, NV = EPL / N;
  static constexpr bool ALIGNED = KIND == WHOLE;
  static_assert(NV * N == EPL, "whole pieces");
  typedef typename MbvaeVec<T>::Aligned Piece;
  int lane, D, first[NV], start[NV];              // piece v: the column it is there for, and the one it begins at
  bool there[NV];
  __device__ __forceinline__ Row(int columns) : lane(TPR ? threadIdx.x % (TPR ? TPR : 1) : threadIdx.x), D(columns) {
    const int width = TPR ? TPR : blockDim.x;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      first[v] = (v * width + lane) * N;
      there[v] = first[v] < D;
      start[v] = ALIGNED || first[v] + N <= D ? first[v] : KIND == MOVED ? D - N : 0;
    }
  }
  __device__ __forceinline__ int col(int e) const { return start[e / N] + e % N; }
  // whether element e is one of the row's, and this thread's to count
  __device__ __forceinline__ bool own(int e) const { return there[e / N] && (ALIGNED || (col(e) >= first[e / N] && col(e) < D)); }
  __device__ __forceinline__ float counted(int e, float t) const { return ALIGNED || own(e) ? t : 0.f; }

  // how many of the row's values wave w of a block holds
  __device__ __forceinline__ float held(int w) const {
    int n = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) n += min(max(D - (v * (int)blockDim.x + 64 * w) * N, 0), 64 * N);
    return (float)n;
  }

  // p: the row.  `on`: whether the row is there at all (a team behind the last row has zeros for all it loads)
  __device__ __forceinline__ void load(const T* p, bool on, Piece* out) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Piece t = {};
      if constexpr (KIND != SHORT) {
        if (on && there[v]) t = *reinterpret_cast<const typename MbvaeVec<T>::Any*>(p + start[v]);
      } else {
        t = mbvae_load_raw<T>(p, on && there[v] ? D : 0);
      }
      out[v] = t;
    }
  }
  static __device__ __forceinline__ void widen(const Piece* in, float* out) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) out[e] = (float)in[e / N][e % N];
  }
  __device__ __forceinline__ void store(T* p, bool on, const float* val) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if constexpr (KIND != SHORT) {
        if (on && there[v]) mbvae_store_vec<T>(p + start[v], N, val + v * N);
      } else {
        mbvae_store_vec<T>(p, on && there[v] ? D : 0, val);
      }
    }
  }
  // a vector over the columns in the parameters' type; `none` where p is null
  template <typename P>
  __device__ __forceinline__ void param_of(const P* p, float* out) const {
    constexpr int M = MbvaeVec<P>::N, STEP = N < M ? N : M;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int q = 0; q < N; q += STEP) {
        const int left = there[v] ? D - start[v] - q : 0;
        float t[M];
        mbvae_load_vec<P>(p + start[v] + q, M > N && left > N ? N : left, t);            // (N of a longer piece)
#pragma unroll
        for (int e = 0; e < STEP; ++e) out[v * N + q + e] = t[e];
      }
  }
  __device__ __forceinline__ void param(const void* p, int type, float none, float* out) const {
    if (!p) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) out[e] = none;
    } else if (type == MBVAE_F32) param_of(reinterpret_cast<const float*>(p), out);
    else if (type == MBVAE_BF16) param_of(reinterpret_cast<const mbvae_bf16*>(p), out);
    else param_of(reinterpret_cast<const mbvae_f16*>(p), out);
  }
  typedef uint8_t Bytes __attribute__((ext_vector_type(MbvaeVec<T>::N)));
  typedef Bytes AnyBytes __attribute__((aligned(1)));
  __device__ __forceinline__ void keep(const uint8_t* p, bool on, Bytes* out) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      Bytes b = {};
      if constexpr (KIND != SHORT) {
        if (on && there[v]) b = *reinterpret_cast<const AnyBytes*>(p + start[v]);
      } else if (on && there[v]) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (e < D) b[e] = p[e];
      }
      out[v] = b;
    }
  }
};

// Mean and reciprocal deviation of a row.
template <int EPL, typename R, typename TeamT>
__device__ __forceinline__ void row_stats(const R& row, TeamT& team, const float* t, float inv_D, bool rms, float eps, float& mean, float& r) {
  float squares;
  mean = 0.f;
  if (rms) {
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const float d = row.counted(e, t[e]);
      q = fmaf(d, d, q);
    }
    squares = team.sum(q);
  } else {
    team.template moments<EPL>(row, t, inv_D, mean, squares);
  }
  // 1 / sqrt(a) to within a rounding: the hardware's and one Newton step.  Not where that leaves the range: eps = 0 and a row of zeros; a sum of
  // squares beyond fp32, which is infinite here - r is 0, and what is finite of such a row becomes 0 (and not NaN).
  const float a = fmaf(squares, inv_D, eps), r0 = __builtin_amdgcn_rsqf(a), step = fmaf(r0 * -a, r0, 1.f);
  r = a > 1e-37f && a < INFINITY ? fmaf(0.5f * r0, step, r0) : 1.f / sqrtf(a);
}

// Both kernels walk over the rows with a fixed grid and ask for the next row's operands before the current row's results are stored: a
// load behind a store would wait for it (one counter, in order).
// Blocks of 16-bit rows are held to 128 registers, which lets 16 waves share a compute unit: their rows are short next to the exchanges
// that a block waits for.  (fp32 would spill: 1024 values 133 -> 213 us.)
template <typename T, int TPR, int EPL, int THREADS, int KIND>
__global__ __launch_bounds__(THREADS, TPR == 0 && sizeof(T) == 2 ? 4 : 1) void gated_norm_fwd_kernel(GatedNormArgs a) {
  typedef Row<T, TPR, EPL, KIND> R;
  constexpr int TEAMS = TPR ? THREADS / (TPR ? TPR : 1) : 1, NV = R::NV;
  __shared__ float2 red[32];
  Team<TPR> team{red, 0};
  const R row(a.D);
  const float inv_D = 1.f / a.D;
  float pg[EPL], pb[EPL], ng[EPL], nb[EPL], sc[EPL];
  row.param(a.post_g, a.ptype, 0.f, pg);
  row.param(a.post_b, a.ptype, 0.f, pb);
  row.param(a.pre_g, a.ptype, 0.f, ng);
  row.param(a.pre_b, a.ptype, 0.f, nb);
  row.param(a.scale, a.ptype, 1.f, sc);
  const int64_t stride = (int64_t)gridDim.x * TEAMS;
  int64_t base = (int64_t)blockIdx.x * TEAMS, r = base + (TPR ? threadIdx.x / (TPR ? TPR : 1) : 0);
  const T *px = reinterpret_cast<const T*>(a.x) + r * a.ldx, *pu = reinterpret_cast<const T*>(a.u) + r * a.ldu,
          *pz = reinterpret_cast<const T*>(a.z) + r * a.ldz;
  const uint8_t* pk = a.keep + r * a.D;
  T *py = reinterpret_cast<T*>(a.y) + r * a.D, *pn = reinterpret_cast<T*>(a.n) + r * a.D;
  typename R::Piece xn[NV], un[NV], zn[NV];
  typename R::Bytes kn[NV];
  const auto ask = [&]() {
    const bool on = r < a.rows;
    row.load(px, on, xn);
    if (a.u) row.load(pu, on, un);
    if (a.z) row.load(pz, on, zn);
    if (a.keep) row.keep(pk, on, kn);
    px += stride * a.ldx; pu += stride * a.ldu; pz += stride * a.ldz; pk += stride * a.D;
  };
  ask();
  for (; base < a.rows; base += stride) {
    const bool on = r < a.rows;
    const int64_t mine = r;
    float y[EPL], v[EPL], w[EPL];
    R::widen(xn, y);
    if (a.u) R::widen(un, v);
    else
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = y[e];
    if (a.z) {
      R::widen(zn, w);
#pragma unroll
      for (int e = 0; e < EPL; ++e) { float ds; sigmoid(w[e], w[e], ds); }
    } else
#pragma unroll
      for (int e = 0; e < EPL; ++e) w[e] = 1.f;
    typename R::Bytes kept[NV];
    if (a.keep)
#pragma unroll
      for (int q = 0; q < NV; ++q) kept[q] = kn[q];
    r += stride;
    if (base + stride < a.rows) ask();
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.post_g) {
      row_stats<EPL>(row, team, v, inv_D, a.rms, a.eps, st.x, st.y);
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = fmaf((v[e] - st.x) * st.y, pg[e], pb[e]);
    }
    if (a.keep) {
#pragma unroll
      for (int e = 0; e < EPL; ++e)                                 // a dropped value adds nothing, whatever it is
        y[e] = kept[e / R::N][e % R::N] ? fmaf(v[e] * (w[e] * a.keep_scale), sc[e], y[e]) : y[e];
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) y[e] = fmaf(v[e] * w[e], sc[e], y[e]);
    }
    row.store(py, on, y);
    py += stride * a.D;
    if (a.pre_g) {
      row_stats<EPL>(row, team, y, inv_D, a.rms, a.eps, st.z, st.w);
#pragma unroll
      for (int e = 0; e < EPL; ++e) y[e] = fmaf((y[e] - st.z) * st.w, ng[e], nb[e]);
      row.store(pn, on, y);
      pn += stride * a.D;
    }
    if (a.stats && on && row.lane == 0) a.stats[mine] = st;
  }
}

template <typename T, int TPR, int EPL, int THREADS, int KIND>
__global__ __launch_bounds__(THREADS) void gated_norm_bwd_kernel(GatedNormArgs a) {
  typedef Row<T, TPR, EPL, KIND> R;
  constexpr int TEAMS = TPR ? THREADS / (TPR ? TPR : 1) : 1, NV = R::NV;
  __shared__ float2 red[32];
  __shared__ float join[TEAMS > 1 ? THREADS * EPL : 1];
  Team<TPR> team{red, 0};
  const R row(a.D);
  const float inv_D = 1.f / a.D, mean_weight = a.rms ? 0.f : inv_D;
  const bool post = a.post_g != nullptr, pre = a.pre_g != nullptr && a.dn != nullptr;
  float pg[EPL], pb[EPL], ng[EPL], sc[EPL];
  row.param(a.post_g, a.ptype, 0.f, pg);
  row.param(a.post_b, a.ptype, 0.f, pb);
  row.param(a.pre_g, a.ptype, 0.f, ng);
  row.param(a.scale, a.ptype, 1.f, sc);
  float sums[GATED_SUMS][EPL];
#pragma unroll
  for (int s = 0; s < GATED_SUMS; ++s)
#pragma unroll
    for (int e = 0; e < EPL; ++e) sums[s][e] = 0.f;
  const int64_t stride = (int64_t)gridDim.x * TEAMS;
  int64_t base = (int64_t)blockIdx.x * TEAMS, r = base + (TPR ? threadIdx.x / (TPR ? TPR : 1) : 0);
  typename R::Piece xn[NV], un[NV], zn[NV], tn[NV], dn[NV];
  typename R::Bytes kn[NV];
  float4 sn = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto ask = [&]() {
    const bool on = r < a.rows;
    sn = on ? a.stats[r] : make_float4(0.f, 0.f, 0.f, 0.f);
    row.load(reinterpret_cast<const T*>(a.x) + r * a.ldx, on, xn);
    if (a.u) row.load(reinterpret_cast<const T*>(a.u) + r * a.ldu, on, un);
    if (a.z) row.load(reinterpret_cast<const T*>(a.z) + r * a.ldz, on, zn);
    if (a.dy) row.load(reinterpret_cast<const T*>(a.dy) + r * a.lddy, on, tn);
    if (pre) row.load(reinterpret_cast<const T*>(a.dn) + r * a.lddn, on, dn);
    if (a.keep) row.keep(a.keep + r * a.D, on, kn);
  };
  if (base < a.rows) ask();
  for (; base < a.rows; base += stride) {
    const bool on = r < a.rows;
    const int64_t mine = r;
    const float4 st = sn;
    float x[EPL], v[EPL], w[EPL], dw[EPL], t[EPL], d[EPL];
    R::widen(xn, x);
    if (a.u) R::widen(un, v);
    else
#pragma unroll
      for (int e = 0; e < EPL; ++e) v[e] = x[e];
    if (a.z) R::widen(zn, w);
    if (a.dy) R::widen(tn, t);
    else
#pragma unroll
      for (int e = 0; e < EPL; ++e) t[e] = 0.f;
    if (pre) R::widen(dn, d);
    bool kept[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) kept[e] = !a.keep || kn[e / R::N][e % R::N] != 0;
    r += stride;
    if (base + stride < a.rows) ask();
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      if (a.z) sigmoid(w[e], w[e], dw[e]);
      else { w[e] = 1.f; dw[e] = 0.f; }
      if (a.keep) {
        w[e] = kept[e] ? w[e] * a.keep_scale : 0.f;
        dw[e] = kept[e] ? dw[e] * a.keep_scale : 0.f;
      }
      if (post) v[e] = (v[e] - st.x) * st.y;          // normalised (behind the row's end it meets a gradient of zero)
    }
    if (pre) {
      float g[EPL], hat[EPL], s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float vv = post ? fmaf(v[e], pg[e], pb[e]) : v[e];
        const float y = kept[e] ? fmaf(vv * w[e], sc[e], x[e]) : x[e];
        hat[e] = (y - st.z) * st.w;
        g[e] = d[e] * ng[e];
        const float gc = row.counted(e, g[e]);
        s1 += gc;
        s2 = fmaf(gc, hat[e], s2);
        sums[GATED_SUM_PRE_G][e] = fmaf(d[e], hat[e], sums[GATED_SUM_PRE_G][e]);
        sums[GATED_SUM_PRE_B][e] += d[e];
      }
      const float2 m = team.sum(s1, s2);
      const float m1 = m.x * mean_weight, m2 = m.y * inv_D;
#pragma unroll
      for (int e = 0; e < EPL; ++e) t[e] = fmaf(st.w, g[e] - fmaf(hat[e], m2, m1), t[e]);
    }
    // t is the whole gradient of y
    float dv[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const float vv = post ? fmaf(v[e], pg[e], pb[e]) : v[e];
      dv[e] = kept[e] ? t[e] * sc[e] * w[e] : 0.f;
      dw[e] = kept[e] ? t[e] * sc[e] * vv * dw[e] : 0.f;
      sums[GATED_SUM_SCALE][e] += kept[e] ? t[e] * w[e] * vv : 0.f;
      if (post) {
        sums[GATED_SUM_POST_G][e] = fmaf(dv[e], v[e], sums[GATED_SUM_POST_G][e]);
        sums[GATED_SUM_POST_B][e] += dv[e];
      }
    }
    if (a.dz) row.store(reinterpret_cast<T*>(a.dz) + mine * a.D, on, dw);
    if (post) {
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        dv[e] *= pg[e];
        const float gc = row.counted(e, dv[e]);
        s1 += gc;
        s2 = fmaf(gc, v[e], s2);
      }
      const float2 m = team.sum(s1, s2);
      const float m1 = m.x * mean_weight, m2 = m.y * inv_D;
#pragma unroll
      for (int e = 0; e < EPL; ++e) dv[e] = st.y * (dv[e] - fmaf(v[e], m2, m1));
    }
    if (a.u) {
      if (a.du) row.store(reinterpret_cast<T*>(a.du) + mine * a.D, on, dv);
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) t[e] += dv[e];
    }
    if (a.dx) row.store(reinterpret_cast<T*>(a.dx) + mine * a.D, on, t);
  }
  // column sums of the block: its teams in order
  float* part = a.part + (int64_t)blockIdx.x * GATED_SUMS * a.D;
#pragma unroll
  for (int s = 0; s < GATED_SUMS; ++s) {
    if (s == GATED_SUM_SCALE ? !a.scale : s <= GATED_SUM_POST_B ? !post : !pre) {
      if (s < GATED_SUM_PRE_G || a.pre_g == nullptr) continue;        // (a norm in front without a gradient behind it: its sums are zero)
    }
    if constexpr (TEAMS > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EPL; ++e) join[e * THREADS + threadIdx.x] = sums[s][e];
      __syncthreads();
      if (threadIdx.x < TPR) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          float total = 0.f;
#pragma unroll
          for (int k = 0; k < TEAMS; ++k) total += join[e * THREADS + k * TPR + threadIdx.x];
          sums[s][e] = total;
        }
      }
    }
    if (TEAMS == 1 || threadIdx.x < TPR)
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (row.own(e)) part[(int64_t)s * a.D + row.col(e)] = sums[s][e];
  }
}

// f(threads a row within a wave or 0, elements, the block's most threads, kind of row), all constants.
template <typename T, typename F>
void for_shape(int dtype, int D, F f) {
  constexpr int N = MbvaeVec<T>::N;
  const GatedNormShape s = gated_norm_shape(dtype, D);
#define GN_INT(i) std::integral_constant<int, i>()
#define GN_CASE(lanes, elements, threads)                                                              \
  do {                                                                                                 \
    if (D % N == 0) f(GN_INT(lanes), GN_INT(elements), GN_INT(threads), GN_INT(WHOLE));                \
    else f(GN_INT(lanes), GN_INT(elements), GN_INT(threads), GN_INT(MOVED));                           \
  } while (0)
  if (D < N) f(GN_INT(4), GN_INT(N), GN_INT(256), GN_INT(SHORT));
  else if (s.threads_a_row == 4) GN_CASE(4, N, 256);
  else if (s.threads_a_row == 8) GN_CASE(8, N, 256);
  else if (s.threads_a_row == 16) GN_CASE(16, N, 256);
  else if (s.threads_a_row == 32) GN_CASE(32, N, 256);
  else if (s.threads_a_row == 64 && s.elements == N) GN_CASE(64, N, 256);
  else if (s.threads_a_row == 64) GN_CASE(64, 8, 256);
  else if (s.block <= 256) GN_CASE(0, 8, 256);
  else if (s.block <= 512) GN_CASE(0, 8, 512);
  else GN_CASE(0, 8, 1024);
#undef GN_CASE
#undef GN_INT
}

template <typename T>
void gated_norm_launch(int dtype, bool forward, const GatedNormArgs& a, unsigned blocks, hipStream_t stream) {
  const unsigned threads = (unsigned)gated_norm_shape(dtype, a.D).block;
  for_shape<T>(dtype, a.D, [&](auto lanes, auto elements, auto most, auto kind) {
    constexpr int TPR = decltype(lanes)::value, EPL = decltype(elements)::value, MOST = decltype(most)::value, KIND = decltype(kind)::value;
    if (forward) hipLaunchKernelGGL((gated_norm_fwd_kernel<T, TPR, EPL, MOST, KIND>), dim3(blocks), dim3(threads), 0, stream, a);
    else hipLaunchKernelGGL((gated_norm_bwd_kernel<T, TPR, EPL, MOST, KIND>), dim3(blocks), dim3(threads), 0, stream, a);
  });
}

}  // namespace
