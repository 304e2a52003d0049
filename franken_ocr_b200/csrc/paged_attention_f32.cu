// Attention over a paged cache of f32.
#include "paged_attention_simt.cuh"

namespace focr {

int launch_attention_f32(AttnArgs &a, cudaStream_t st) { return launch_simt_dim<float>(a, st); }

}  // namespace focr
