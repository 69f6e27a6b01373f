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
// Measured (us; rate over what each kernel reads and writes): 1 M rows of 64 fp32 values with a gate, forward 247 (5.4 TB/s), backward 388
// (5.5 TB/s); 16 384 rows of 256 bf16 values with both norms, gate and scale 13.4 and 21.2 (3.1 and 3.2 TB/s); 4095 rows of 1037 fp16
// values, root-mean-square norms, 17.6 and 35 (1.9 and 1.5 TB/s); 4096 rows of 8192 fp32 values with everything 252 and 925 (2.7 and 1.2 TB/s:
// 1024 threads leave 128 registers, and both spill); 256 rows of 512 fp32 values 5.0 and 6.6 (a launch); the column sums' join 3-6.
#include "gated_norm.h"
#include <algorithm>

namespace {

constexpr int SUMS = GATED_SUMS;

// out[s][c] = sum over the blocks of part[block][s][c], in the parameters' type.  8 columns x 32 groups of blocks, joined in order.
struct Outs { void* p[SUMS]; };
__global__ __launch_bounds__(256) void gated_norm_sums_kernel(const float* __restrict__ part, Outs outs, int blocks, int D, int ptype) {
  __shared__ float red[32][9];
  const int cx = threadIdx.x & 7, g = threadIdx.x >> 3, s = blockIdx.y;
  const int c = blockIdx.x * 8 + cx;
  if (!outs.p[s]) return;
  float a[8] = {};
  if (c < D) {
    const float* p = part + (int64_t)s * D + c;
    const int64_t step = (int64_t)SUMS * D;
    int b = g;
    for (; b + 7 * 32 < blocks; b += 8 * 32) {
#pragma unroll
      for (int q = 0; q < 8; ++q) a[q] += p[(b + 32 * q) * step];
    }
    for (; b < blocks; b += 32) a[0] += p[b * step];
  }
  red[g][cx] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  __syncthreads();
  if (g == 0 && c < D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][cx];
    mbvae_store_param(outs.p[s], ptype, c, t);
  }
}

constexpr int MAX_D = 8192;

// Blocks: as many as keep `waves` waves on every compute unit, at least one.  More of them have more places of memory open at once and
// were slower: forward over 1 M rows of 64 fp32 values 282 us with 4096 blocks of four waves, 262 with 2048, 246-252 with 768 (12 waves a
// unit), 287 with 512; backward 452 with 1024, 428 with 768, 410 with 512 (8 waves), 384 with 256 (4 waves) - which in turn is slower
// where a block has few rows (16 384 rows of 256 bf16 values: 26.3 / 26.0 / 21.5 / 25.2 us).
int64_t blocks_for(int dtype, int64_t rows, int64_t D, int waves) {
  const GatedNormShape s = gated_norm_shape(dtype, (int)D);
  const int64_t teams = s.block / s.threads_a_row, most = (int64_t)mbvae_num_cus() * std::max(1, waves / (s.block / 64));
  return std::max<int64_t>(1, std::min<int64_t>((rows + teams - 1) / teams, most));
}
// Forward of 16-bit rows that take a block: 16 waves a unit, which exchange more than they stream (65 536 rows of 520 bf16 values 177 us
// with 12, 145 with 16).
int64_t fwd_blocks(int dtype, int64_t rows, int64_t D) {
  return blocks_for(dtype, rows, D, dtype != MBVAE_F32 && gated_norm_shape(dtype, (int)D).threads_a_row > 64 ? 16 : 12);
}
int64_t bwd_blocks(int dtype, int64_t rows, int64_t D) {
  const GatedNormShape s = gated_norm_shape(dtype, (int)D);
  const int64_t walk = rows / (s.block / s.threads_a_row) / mbvae_num_cus();      // rows a team would walk over with one block a unit
  return blocks_for(dtype, rows, D, walk >= 128 && s.threads_a_row <= 64 ? 4 : 8);
}

int check(const GatedNormArgs& a, int dtype, int64_t rows, int64_t D, int ptype) {
  if (rows < 0 || D <= 0 || mbvae_dtype_size(dtype) == 0 || mbvae_dtype_size(ptype) == 0) return MBVAE_EINVAL;
  if (a.ldx < 0 || a.ldu < 0 || a.ldz < 0) return MBVAE_EINVAL;
  if (rows && !a.x) return MBVAE_EINVAL;
  if ((a.post_b && !a.post_g) || (a.pre_b && !a.pre_g)) return MBVAE_EINVAL;
  if (((uintptr_t)a.stats & 15) || !(a.eps >= 0.f)) return MBVAE_EINVAL;
  if (D > MAX_D || rows >= (int64_t)1 << 31) return MBVAE_EUNSUPPORTED;
  return MBVAE_OK;
}

int launch(bool forward, int dtype, const GatedNormArgs& a, int64_t blocks, hipStream_t stream) {
  const auto f = dtype == MBVAE_F32 ? gated_norm_launch_f32 : dtype == MBVAE_BF16 ? gated_norm_launch_bf16 : gated_norm_launch_f16;
  f(forward, a, (unsigned)blocks, stream);
  return mbvae_launch_status();
}

}  // namespace

extern "C" {

int mbvae_gated_norm_fwd(const void* x, int64_t ldx, const void* u, int64_t ldu, const void* z, int64_t ldz, const uint8_t* keep, float keep_scale,
                         const void* post_gamma, const void* post_beta, const void* scale, const void* pre_gamma, const void* pre_beta, void* y, void* n,
                         float* stats, int64_t rows, int64_t D, int rms, float eps, int dtype, int ptype, hipStream_t stream) {
  (void)hipGetLastError();  // drop stale (non-sticky) errors left by other runtime users
  GatedNormArgs a = {};
  a.x = x; a.u = u; a.z = z; a.keep = keep; a.scale = scale;
  a.post_g = post_gamma; a.post_b = post_beta; a.pre_g = pre_gamma; a.pre_b = pre_beta;
  a.ldx = ldx; a.ldu = ldu; a.ldz = ldz; a.rows = rows; a.D = (int)std::min<int64_t>(D, MAX_D); a.ptype = ptype; a.rms = rms;
  a.keep_scale = keep_scale; a.eps = eps; a.stats = reinterpret_cast<float4*>(stats);
  a.y = y; a.n = n;
  const int st = check(a, dtype, rows, D, ptype);
  if (st != MBVAE_OK) return st;
  if (rows == 0) return MBVAE_OK;
  if (!y || (pre_gamma && !n)) return MBVAE_EINVAL;
  return launch(true, dtype, a, fwd_blocks(dtype, rows, D), stream);
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
  GatedNormArgs a = {};
  a.x = x; a.u = u; a.z = z; a.keep = keep; a.scale = scale;
  a.post_g = post_gamma; a.post_b = post_beta; a.pre_g = pre_gamma;
  a.ldx = ldx; a.ldu = ldu; a.ldz = ldz; a.rows = rows; a.D = (int)std::min<int64_t>(D, MAX_D); a.ptype = ptype; a.rms = rms;
  a.keep_scale = keep_scale; a.eps = eps; a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  a.dy = dy; a.dn = dn; a.lddy = lddy; a.lddn = lddn; a.dx = dx; a.du = du; a.dz = dz; a.part = reinterpret_cast<float*>(ws);
  const int st = check(a, dtype, rows, D, ptype);
  if (st != MBVAE_OK) return st;
  if (lddy < 0 || lddn < 0 || (dn && !pre_gamma) || (rows && !stats) || !ws || ((uintptr_t)ws & 15)) return MBVAE_EINVAL;
  if (dscale && !scale) return MBVAE_EINVAL;
  if ((dpost_gamma || dpost_beta) && !post_gamma) return MBVAE_EINVAL;
  if ((dpre_gamma || dpre_beta) && !pre_gamma) return MBVAE_EINVAL;
  if ((du && !u) || (dz && !z)) return MBVAE_EINVAL;
  if (ws_bytes < mbvae_gated_norm_bwd_workspace(rows, D, dtype)) return MBVAE_EINVAL;
  const int64_t blocks = bwd_blocks(dtype, rows, D);
  const int launched = launch(false, dtype, a, blocks, stream);
  if (launched != MBVAE_OK) return launched;
  const Outs outs = {{dscale, dpost_gamma, dpost_beta, dpre_gamma, dpre_beta}};
  if (dscale || dpost_gamma || dpost_beta || dpre_gamma || dpre_beta)
    hipLaunchKernelGGL(gated_norm_sums_kernel, dim3((unsigned)((D + 7) / 8), SUMS), dim3(256), 0, stream, a.part, outs, (int)blocks, (int)D, ptype);
  return mbvae_launch_status();
}

}  // extern "C"
