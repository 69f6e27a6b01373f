// Gated residual update between two norms, forward and backward: what the entry points (gated_norm.hip) and the three sources that hold
// the kernels of one activation type each (gated_norm_f32.hip, _bf16, _f16) share.
#pragma once
#include "typed.h"

enum { GATED_SUM_SCALE, GATED_SUM_POST_G, GATED_SUM_POST_B, GATED_SUM_PRE_G, GATED_SUM_PRE_B, GATED_SUMS };      // column sums, as the partials lie

struct GatedNormArgs {
  const void *x, *u, *z;              // u null: x; z null: no gate
  const uint8_t* keep;
  const void *post_g, *post_b, *scale, *pre_g, *pre_b;
  int64_t ldx, ldu, ldz, rows;
  int D, ptype, rms;
  float keep_scale, eps;
  float4* stats;                      // per row: mean and reciprocal deviation of u, then of y
  void *y, *n;                        // forward
  const void *dy, *dn;                // backward
  int64_t lddy, lddn;
  void *dx, *du, *dz;
  float* part;                        // [blocks][GATED_SUMS][D]
};

// Threads a row and elements a thread.  Up to 64 pieces of 16 bytes (fp32: up to 512 values) a row belongs to 4 to 64 lanes of a
// wave; wider rows to a block of their own with 8 elements a thread, as few waves as hold the row.
struct GatedNormShape {
  int threads_a_row, elements, block;
};
inline GatedNormShape gated_norm_shape(int dtype, int D) {
  const int N = dtype == MBVAE_F32 ? 4 : 8;
  if (D <= 4 * N) return {4, N, 256};
  if (D <= 8 * N) return {8, N, 256};
  if (D <= 16 * N) return {16, N, 256};
  if (D <= 32 * N) return {32, N, 256};
  if (D <= 64 * N) return {64, N, 256};
  if (D <= 512) return {64, 8, 256};
  const int threads = (D + 511) / 512 * 64;
  return {threads, 8, threads};
}

void gated_norm_launch_f32(bool forward, const GatedNormArgs& a, unsigned blocks, hipStream_t stream);
void gated_norm_launch_bf16(bool forward, const GatedNormArgs& a, unsigned blocks, hipStream_t stream);
void gated_norm_launch_f16(bool forward, const GatedNormArgs& a, unsigned blocks, hipStream_t stream);
