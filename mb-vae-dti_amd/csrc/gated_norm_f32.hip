// Gated residual update: the kernels of fp32 activations.
#include "gated_norm_kernels.h"

void gated_norm_launch_f32(bool forward, const GatedNormArgs& a, unsigned blocks, hipStream_t stream) {
  gated_norm_launch<float>(MBVAE_F32, forward, a, blocks, stream);
}
