// Attention over a paged cache of f16.
#include "paged_attention_mma.cuh"
#include "paged_attention_simt.cuh"

namespace focr {

int launch_attention_f16(AttnArgs &a, cudaStream_t st) {
    if (a.q_type == FOCR_F16 && a.group >= MMA_HEADS) return launch_mma_dim<__half>(a, st);
    return launch_simt_dim<__half>(a, st);
}

}  // namespace focr
