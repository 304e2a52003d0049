// Attention over a paged cache of bf16.
#include "paged_attention_mma.cuh"
#include "paged_attention_simt.cuh"

namespace focr {

int launch_attention_bf16(AttnArgs &a, cudaStream_t st) {
    if (a.q_type == FOCR_BF16 && a.group >= MMA_HEADS) return launch_mma_dim<__nv_bfloat16>(a, st);
    return launch_simt_dim<__nv_bfloat16>(a, st);
}

}  // namespace focr
