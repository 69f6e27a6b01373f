// Gated residual update: the kernels of bf16 activations.
#include "gated_norm_kernels.h"

void gated_norm_launch_bf16(bool forward, const GatedNormArgs& a, unsigned blocks, hipStream_t stream) {
  gated_norm_launch<mbvae_bf16>(MBVAE_BF16, forward, a, blocks, stream);
}
