// Gated residual update: the kernels of fp16 activations.
#include "gated_norm_kernels.h"

void gated_norm_launch_f16(bool forward, const GatedNormArgs& a, unsigned blocks, hipStream_t stream) {
  gated_norm_launch<mbvae_f16>(MBVAE_F16, forward, a, blocks, stream);
}
